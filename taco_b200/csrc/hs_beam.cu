// The selection of a beam search over beams and vocabulary (hs_op_beam_select, hs_batch_beam_step).
//
// A row of logits is read as the LM head leaves it: u16 distances from the tile maxima. A symbol's
// distance D from the row maximum is the whole number of table units that its log weight lies below
// the largest, so D is its cost up to the row's normaliser: cost = base + N + D with N = #{j :
// table[j] W > table[0]^2}, the least j at which table[j] / table[0] is not above table[0] / W. A
// symbol's key is D << 16 | symbol: keys are distinct, their order is the order of the candidates of a
// row (the lower symbol first among equal distances), and they fit in 30 bits.
#include <cuda_runtime.h>

#include <cstdint>

#include "hs_common.cuh"
#include "hs_draft.hpp"

namespace hs {

namespace {

constexpr int BEAM_THREADS = 512;
constexpr int BEAM_LIST = 1024;  // candidates that pass the first threshold
constexpr uint32_t NO_KEY = 0xFFFFFFFFu;
constexpr int64_t BASE_LIMIT = 1LL << 62;

__global__ void __launch_bounds__(BEAM_THREADS) k_beam_select(const BeamArgs a) {
    __shared__ uint32_t s_min[BEAM_THREADS], s_list[BEAM_LIST];
    __shared__ uint32_t s_best[MAX_BEAMS][MAX_KEEP];  // the cheapest keys of each row, in order
    __shared__ int s_len[MAX_BEAMS];
    __shared__ int64_t s_row[MAX_BEAMS];              // base + N
    __shared__ uint8_t s_fin[MAX_BEAMS];
    __shared__ int64_t s_max;
    __shared__ unsigned long long s_sum;
    __shared__ uint32_t s_cut, s_count, s_norm;
    const int tid = threadIdx.x, lane = tid & 31;
    const int last = a.tlen - 1, tiles = (a.vocab + (1 << a.tsh) - 1) >> a.tsh;
    const uint32_t keep = (uint32_t)a.keep;
    for (int b = 0; b < a.beams; b++) {
        const size_t row = (size_t)blockIdx.x * a.beams + b;
        const int64_t base = a.base[row];
        const bool dead = base < 0 || base >= BASE_LIMIT, fin = a.finished && a.finished[row] != 0;
        if (tid == 0) {
            s_fin[b] = fin;
            s_row[b] = base;
            s_len[b] = dead ? 0 : fin ? 1 : 0;
            s_best[b][0] = 0;
        }
        if (dead || fin) continue;
        const size_t lrow = a.row_of ? a.row_of[row] : row;
        const uint16_t* dist = a.dist + lrow * a.dist_stride;
        const int64_t* tops = a.tops + lrow * a.tops_stride;
        __syncthreads();
        if (tid == 0) {
            s_max = INT64_MIN;
            s_sum = 0;
            s_cut = NO_KEY - 1;
            s_count = 0;
            s_norm = 0;
        }
        __syncthreads();
        int64_t mx = INT64_MIN;
        for (int t = tid; t < tiles; t += BEAM_THREADS) mx = tops[t] > mx ? tops[t] : mx;
        for (int o = 16; o > 0; o >>= 1) {
            const int64_t w = __shfl_xor_sync(0xffffffffu, mx, o);
            mx = w > mx ? w : mx;
        }
        if (lane == 0) atomicMax((long long*)&s_max, (long long)mx);
        __syncthreads();
        mx = s_max;
        auto key_of = [&](int v) -> uint32_t {
            // The offset as an unsigned difference: right for any maxima, and never below 0.
            const uint64_t off = (uint64_t)mx - (uint64_t)tops[v >> a.tsh];
            const uint32_t d = off < (uint64_t)last ? (uint32_t)off + dist[v] : (uint32_t)last;
            return (d < (uint32_t)last ? d : (uint32_t)last) << 16 | (uint32_t)v;
        };
        uint64_t sum = 0;
        uint32_t mine = NO_KEY;
        for (int v = tid; v < a.vocab; v += BEAM_THREADS) {
            const uint32_t key = key_of(v);
            sum += a.table[key >> 16];
            if ((int)(key >> 16) <= a.last_weight) mine = key < mine ? key : mine;
        }
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) atomicAdd(&s_sum, (unsigned long long)sum);
        // The keep-th smallest of the threads' smallest keys: at least `keep` keys are not above it.
        s_min[tid] = mine;
        __syncthreads();
        uint32_t rank = 0;
        for (int i = 0; i < BEAM_THREADS; i++) rank += s_min[i] < mine;
        if (mine != NO_KEY && rank == keep - 1) s_cut = mine;
        const uint64_t W = s_sum;
        const u128 one = (u128)a.table[0] * a.table[0];
        uint32_t norm = 0;
        for (int j = tid; j < a.tlen; j += BEAM_THREADS) norm += (u128)a.table[j] * W > one;
        norm = __reduce_add_sync(0xffffffffu, norm);
        if (lane == 0) atomicAdd(&s_norm, norm);
        __syncthreads();
        uint32_t cut = s_cut;
        auto good = [&](uint32_t key) { return (int)(key >> 16) <= a.last_weight; };
        auto collect = [&](uint32_t upto) {
            for (int v = tid; v < a.vocab; v += BEAM_THREADS) {
                const uint32_t key = key_of(v);
                if (key <= upto && good(key)) {
                    const uint32_t at = atomicAdd(&s_count, 1u);
                    if (at < BEAM_LIST) s_list[at] = key;
                }
            }
            __syncthreads();
        };
        collect(cut);
        if (s_count > BEAM_LIST) {
            // Too many keys pass (they cluster in a few threads' symbols): the least key that `keep`
            // keys are not above, by bisection over key values, each step a pass over the row.
            uint32_t lo = 0, hi = cut;
            while (lo < hi) {
                const uint32_t mid = lo + (hi - lo) / 2;
                __syncthreads();
                if (tid == 0) s_count = 0;
                __syncthreads();
                uint32_t n = 0;
                for (int v = tid; v < a.vocab; v += BEAM_THREADS) {
                    const uint32_t key = key_of(v);
                    n += key <= mid && good(key);
                }
                n = __reduce_add_sync(0xffffffffu, n);
                if (lane == 0) atomicAdd(&s_count, n);
                __syncthreads();
                if (s_count >= keep) hi = mid;
                else lo = mid + 1;
            }
            __syncthreads();
            if (tid == 0) s_count = 0;
            __syncthreads();
            collect(lo);
        }
        const uint32_t n = s_count;
        for (uint32_t i = tid; i < n; i += BEAM_THREADS) {
            const uint32_t key = s_list[i];
            uint32_t at = 0;
            for (uint32_t k = 0; k < n; k++) at += s_list[k] < key;
            if (at < keep) s_best[b][at] = key;
        }
        if (tid == 0) {
            s_len[b] = (int)(n < keep ? n : keep);
            s_row[b] = base + s_norm;
        }
    }
    __syncthreads();
    // The merge of the rows' lists: a candidate's place is the number of candidates before it (cost,
    // then beam, then symbol), by bisection in every list.
    uint32_t total = 0;
    for (int b = 0; b < a.beams; b++) total += (uint32_t)s_len[b];
    const size_t out = (size_t)blockIdx.x * keep;
    for (uint32_t i = tid; i < (uint32_t)a.beams * keep; i += BEAM_THREADS) {
        const int b = (int)(i / keep), k = (int)(i % keep);
        if (k >= s_len[b]) continue;
        const uint32_t key = s_best[b][k];
        const int64_t cost = s_row[b] + (key >> 16);
        uint32_t at = (uint32_t)k;
        for (int o = 0; o < a.beams && at < keep; o++) {
            if (o == b) continue;
            int lo = 0, hi = s_len[o];
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                const int64_t c = s_row[o] + (s_best[o][mid] >> 16);
                if (c < cost || (c == cost && o < b)) lo = mid + 1;
                else hi = mid;
            }
            at += (uint32_t)lo;
        }
        if (at < keep) {
            a.parent[out + at] = (uint32_t)b;
            a.token[out + at] = s_fin[b] ? NO_KEY : key & 0xFFFFu;
            a.cost[out + at] = cost;
        }
    }
    for (uint32_t i = total + tid; i < keep; i += BEAM_THREADS) {
        a.parent[out + i] = NO_KEY;
        a.token[out + i] = NO_KEY;
        a.cost[out + i] = -1;
    }
}

}  // namespace

cudaError_t launch_beam_select(const BeamArgs& a, int num_sms, cudaStream_t st) {
    (void)num_sms;
    if (a.groups == 0) return cudaSuccess;
    k_beam_select<<<(unsigned)a.groups, BEAM_THREADS, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace hs
