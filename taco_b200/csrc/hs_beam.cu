// The selection of a beam search over beams and vocabulary (hs_op_beam_select, hs_batch_beam_step).
//
// A row of logits is read as the LM head leaves it: u16 distances from the tile maxima. A symbol's
// distance D from the row maximum is the whole number of table units that its log weight lies below
// the largest, so D is its cost up to the row's normaliser: cost = base + N + D with N = #{j :
// table[j] W > table[0]^2}, the least j at which table[j] / table[0] is not above table[0] / W. A
// symbol's key is D << 16 | symbol: keys are distinct, their order is the order of the candidates of a
// row (the lower symbol first among equal distances), and they fit in 30 bits.
//
// A cluster of blocks takes a group; its items are the rows' segments (1 to 8 a row), dealt round-robin
// to the blocks. A block reads a segment once, sums its weights and takes each thread's smallest distance.
// The keep-th smallest of the minima of 64 groups of four threads is a distance that at least `keep`
// symbols are not above: only symbols up to it are candidates (about `keep` of them, unless distances
// tie). The few groups of 8 symbols that hold one are read again (from L2), and each candidate finds its
// place by counting. The lists and sums go to the first block's shared memory, which adds the normalisers
// and merges the lists.
//
// The sums are one table look-up per symbol, in shared memory at random banks: this bounds the kernel. The
// look-ups take 32 bits, floor(table[j] / 2^s), so the sum is known to lie in [L 2^s, L 2^s + vocab (2^s -
// 1)]. N does not decrease with W, so where both ends give one N it is exact; where they differ (W next to
// a border) the row is summed again with the whole 64-bit weights.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "hs_common.cuh"
#include "hs_draft.hpp"

namespace cg = cooperative_groups;

namespace hs {

namespace {

constexpr int BEAM_THREADS = 256;
constexpr int BEAM_WARPS = BEAM_THREADS / 32;
constexpr int BEAM_BLOCKS = 4;   // blocks of an SM (registers)
constexpr int BEAM_UNROLL = 4;   // loads of 8 symbols that a thread has in flight
constexpr int BEAM_GROUPS = 64;  // the minima that give the first threshold (four threads each)
constexpr int BEAM_LIST = 512;   // symbols up to the threshold that are held, and groups of 8 of them
constexpr int BEAM_LISTS = 2 * MAX_BEAMS;
constexpr uint32_t NO_KEY = 0xFFFFFFFFu;
constexpr int64_t BASE_LIMIT = 1LL << 62;
static_assert(4 * BEAM_GROUPS == BEAM_THREADS && BEAM_WARPS == 8, "the reductions");
static_assert(MAX_KEEP <= BEAM_GROUPS, "the threshold needs as many minima as places");

// sum + e by the multiply-add pipe: the integer adds of the distances keep the other one.
__device__ __forceinline__ uint64_t add_wide(uint64_t sum, uint32_t e) {
    uint64_t r;
    asm("mad.wide.u32 %0, %1, 1, %2;" : "=l"(r) : "r"(e), "l"(sum));
    return r;
}

struct BeamSmem {
    // The segment in work.
    int64_t red[BEAM_WARPS];
    uint64_t redu[BEAM_WARPS];
    uint16_t off[MAX_CODER_VOCAB / 64];  // the tiles' distances from the row maximum, cut at the table
    __align__(16) uint32_t least[BEAM_GROUPS];
    uint32_t list[BEAM_LIST], keys[BEAM_LIST];
    uint32_t cut, held, count;
    // The group's lists (in the cluster's first block): their lengths here, their keys [lists][keep] and
    // the keys' places behind this struct.
    int len[BEAM_LISTS];
    uint64_t sum[BEAM_LISTS];
    int64_t top[MAX_BEAMS];        // the row maxima
    int64_t row[MAX_BEAMS];        // base + N
    uint8_t fin[MAX_BEAMS], border[MAX_BEAMS];
};

__global__ void __launch_bounds__(BEAM_THREADS, BEAM_BLOCKS) k_beam_select(const __grid_constant__ BeamArgs a, int segs, int vec,
                                                                 int cut_bits) {
    extern __shared__ __align__(16) uint8_t s_beam[];
    uint32_t* sT = reinterpret_cast<uint32_t*>(s_beam);  // tlen weights / 2^cut_bits, then 0 for no symbol
    BeamSmem& sm = *reinterpret_cast<BeamSmem*>(s_beam + 16 * (((size_t)a.tlen + 4) / 4));
    uint32_t* s_best = reinterpret_cast<uint32_t*>(&sm + 1);
    uint32_t* s_place = s_best + a.beams * segs * a.keep;
    uint16_t* s_near = reinterpret_cast<uint16_t*>(s_place + a.beams * segs * a.keep);  // the vectors' smallest D
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    const int last = a.tlen - 1, tiles = (a.vocab + (1 << a.tsh) - 1) >> a.tsh;
    const uint32_t keep = (uint32_t)a.keep, no_symbol = (uint32_t)a.tlen;
    const int vecs = (a.vocab + 7) / 8, seg_vecs = (vecs + segs - 1) / segs;
    for (int i = tid; i <= a.tlen; i += BEAM_THREADS) sT[i] = i < a.tlen ? (uint32_t)(a.table[i] >> cut_bits) : 0;
    __syncthreads();

    for (int group = blockIdx.x / C; group < a.groups; group += gridDim.x / C) {
        if (rank == 0)
            for (int b = tid; b < a.beams; b += BEAM_THREADS) {
                const size_t r = (size_t)group * a.beams + b;
                sm.row[b] = a.base[r];
                sm.fin[b] = a.finished && a.finished[r] != 0;
            }
        // The first block's lists of the group before are merged before they are written again (the
        // cluster barrier at the end of a group).
        for (int item = rank; item < a.beams * segs; item += C) {
            const int b = item / segs, seg = item % segs;
            const size_t row = (size_t)group * a.beams + b;
            const int64_t base = a.base[row];
            uint32_t* best = cl.map_shared_rank(s_best + item * a.keep, 0);
            if (base < 0 || base >= BASE_LIMIT || (a.finished && a.finished[row] != 0)) {
                // A dead beam has no candidates; one that has ended is a candidate itself.
                if (tid == 0) {
                    const bool one = base >= 0 && base < BASE_LIMIT && seg == 0;
                    *cl.map_shared_rank(&sm.len[item], 0) = one ? 1 : 0;
                    *cl.map_shared_rank(&sm.sum[item], 0) = 0;
                    if (one) best[0] = 0;
                }
                continue;
            }
            const size_t lrow = a.row_of ? a.row_of[row] : row;
            const uint16_t* dist = a.dist + lrow * a.dist_stride;
            const int64_t* tops = a.tops + lrow * a.tops_stride;
            const int v0 = seg * seg_vecs, v1 = v0 + seg_vecs < vecs ? v0 + seg_vecs : vecs;
            // The segment's whole groups of 8 symbols are read as vectors; what the vocabulary's end leaves,
            // or everything if the rows are not aligned, symbol by symbol.
            const int vw = vec ? min(v1, a.vocab / 8) : v0;
            uint4 raw[BEAM_UNROLL];
            auto load_all = [&](int v) {
#pragma unroll
                for (int k = 0; k < BEAM_UNROLL; k++)
                    if (v + k * BEAM_THREADS < vw)
                        raw[k] = __ldg(reinterpret_cast<const uint4*>(dist) + v + k * BEAM_THREADS);
            };
            load_all(v0 + tid);  // on their way while the row maximum is found
            int64_t mx = INT64_MIN;
            for (int t = tid; t < tiles; t += BEAM_THREADS) mx = tops[t] > mx ? tops[t] : mx;
            for (int o = 16; o > 0; o >>= 1) {
                const int64_t x = __shfl_xor_sync(0xffffffffu, mx, o);
                mx = x > mx ? x : mx;
            }
            if (lane == 0) sm.red[w] = mx;
            __syncthreads();
            mx = sm.red[lane % (BEAM_WARPS)];
            for (int o = 4; o > 0; o >>= 1) {
                const int64_t x = __shfl_xor_sync(0xffffffffu, mx, o);
                mx = x > mx ? x : mx;
            }
            // The offset as an unsigned difference: right for any maxima, and never below 0.
            for (int t = tid; t < tiles; t += BEAM_THREADS) {
                const uint64_t o = (uint64_t)mx - (uint64_t)tops[t];
                sm.off[t] = (uint16_t)(o < (uint64_t)last ? o : (uint64_t)last);
            }
            if (tid == 0) sm.count = sm.held = 0;
            __syncthreads();
            // The next segment on its way into L2.
            if (vec && tid == 0 && item + C < a.beams * segs) {
                const int b2 = (item + C) / segs, s2 = (item + C) % segs;
                const size_t r2 = (size_t)group * a.beams + b2;
                const int f0 = s2 * seg_vecs, f1 = f0 + seg_vecs < a.vocab / 8 ? f0 + seg_vecs : a.vocab / 8;
                // (bases and strides of 16 bytes: `vec`)
                if (f1 > f0)
                    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(
                                     a.dist + (a.row_of ? a.row_of[r2] : r2) * a.dist_stride + 8 * (size_t)f0),
                                 "r"(16 * (f1 - f0)));
            }
            uint64_t sum = 0;
            uint32_t nearest = no_symbol;
            auto far_of = [&](int v) -> uint32_t {
                const uint32_t o = sm.off[v >> a.tsh];
                return o + min((uint32_t)dist[v], (uint32_t)last - o);
            };
            // D = min(offset + distance, last) = offset + min(distance, last - offset), two symbols at a
            // time: no half carries into the other.
            auto add = [&](int v, uint4 d) {
                const uint32_t off2 = (uint32_t)sm.off[(8 * v) >> a.tsh] * 0x10001u;
                const uint32_t most2 = (uint32_t)last * 0x10001u - off2;
                const uint32_t x[4] = {__vminu2(d.x, most2) + off2, __vminu2(d.y, most2) + off2,
                                       __vminu2(d.z, most2) + off2, __vminu2(d.w, most2) + off2};
                uint32_t e[8];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    e[2 * j] = sT[x[j] & 0xFFFFu];
                    e[2 * j + 1] = sT[x[j] >> 16];
                }
#pragma unroll
                for (int j = 0; j < 8; j++) sum = add_wide(sum, e[j]);
                const uint32_t m2 = __vminu2(__vminu2(x[0], x[1]), __vminu2(x[2], x[3]));
                const uint32_t m = min(m2 & 0xFFFFu, m2 >> 16);
                s_near[v - v0] = (uint16_t)m;
                nearest = min(nearest, m);
            };
            for (int v = v0 + tid; v < vw; v += BEAM_UNROLL * BEAM_THREADS) {
                uint4 cur[BEAM_UNROLL];
#pragma unroll
                for (int k = 0; k < BEAM_UNROLL; k++) cur[k] = raw[k];
                load_all(v + BEAM_UNROLL * BEAM_THREADS);
#pragma unroll
                for (int k = 0; k < BEAM_UNROLL; k++)
                    if (v + k * BEAM_THREADS < vw) add(v + k * BEAM_THREADS, cur[k]);
            }
            // (a thread's groups are v0 + tid + k BEAM_THREADS, these too)
            for (int v = v0 + tid + max(0, (vw - v0 - tid + BEAM_THREADS - 1) / BEAM_THREADS) * BEAM_THREADS; v < v1;
                 v += BEAM_THREADS) {
                uint32_t m = no_symbol;
                for (int i = 8 * v; i < 8 * v + 8 && i < a.vocab; i++) {
                    const uint32_t D = far_of(i);
                    sum += sT[D];
                    m = min(m, D);
                }
                s_near[v - v0] = (uint16_t)m;
                nearest = min(nearest, m);
            }
            uint32_t least = nearest;
            least = min(least, __shfl_xor_sync(0xffffffffu, least, 1));
            least = min(least, __shfl_xor_sync(0xffffffffu, least, 2));
            if ((lane & 3) == 0) sm.least[tid >> 2] = least;
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) sm.redu[w] = sum;
            __syncthreads();
            {
                // The place of a minimum among the minima (equal ones by their index): four threads a
                // minimum, each against a quarter of them.
                const int i = tid >> 2, o0 = (tid & 3) * (BEAM_GROUPS / 4);
                const uint32_t mine = sm.least[i];
                uint32_t at = 0;
#pragma unroll
                for (int k = 0; k < BEAM_GROUPS / 4; k += 4) {
                    const uint4 o = *reinterpret_cast<const uint4*>(&sm.least[o0 + k]);
                    const int j = o0 + k;
                    at += (o.x < mine + (j < i)) + (o.y < mine + (j + 1 < i)) + (o.z < mine + (j + 2 < i)) +
                          (o.w < mine + (j + 3 < i));
                }
                at += __shfl_xor_sync(0xffffffffu, at, 1);
                at += __shfl_xor_sync(0xffffffffu, at, 2);
                if ((tid & 3) == 0 && at == keep - 1) sm.cut = mine;
            }
            if (w == BEAM_WARPS - 1) {
                uint64_t all = lane < BEAM_WARPS ? sm.redu[lane] : 0;
                for (int o = 4; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
                if (lane == 0) {
                    *cl.map_shared_rank(&sm.sum[item], 0) = all;
                    if (seg == 0) *cl.map_shared_rank(&sm.top[b], 0) = mx;
                }
            }
            __syncthreads();
            const uint32_t cut = min(sm.cut, (uint32_t)a.last_weight);
            // The groups of 8 symbols that hold a candidate, then a thread for each of their symbols.
            if (nearest <= cut)
                for (int v = v0 + tid; v < v1; v += BEAM_THREADS)
                    if (s_near[v - v0] <= cut) {
                        const uint32_t at = atomicAdd(&sm.held, 1u);
                        if (at < BEAM_LIST) sm.list[at] = (uint32_t)v;
                    }
            __syncthreads();
            const uint32_t held = sm.held;
            if (held <= BEAM_LIST)
                for (uint32_t i = tid; i < 8 * held; i += BEAM_THREADS) {
                    const uint32_t v = 8 * sm.list[i >> 3] + (i & 7);
                    const uint32_t D = v < (uint32_t)a.vocab ? far_of((int)v) : no_symbol;
                    if (D > cut) continue;
                    const uint32_t at = atomicAdd(&sm.count, 1u);
                    if (at < BEAM_LIST) sm.keys[at] = D << 16 | v;
                }
            __syncthreads();
            if (held > BEAM_LIST || sm.count > BEAM_LIST) {
                // Distances tie: the least key that `keep` keys are not above, by bisection over keys.
                auto each = [&](uint32_t upto, auto f) {
                    if (nearest > upto >> 16) return;
                    for (int v = v0 + tid; v < v1; v += BEAM_THREADS) {
                        if (s_near[v - v0] > upto >> 16) continue;
                        for (int i = 8 * v; i < 8 * v + 8 && i < a.vocab; i++) {
                            const uint32_t key = far_of(i) << 16 | (uint32_t)i;
                            if (key <= upto) f(key);
                        }
                    }
                };
                uint32_t lo = 0, hi = cut << 16 | 0xFFFFu;
                while (lo < hi) {
                    const uint32_t mid = lo + (hi - lo) / 2;
                    __syncthreads();
                    if (tid == 0) sm.count = 0;
                    __syncthreads();
                    uint32_t n = 0;
                    each(mid, [&](uint32_t) { n++; });
                    n = __reduce_add_sync(0xffffffffu, n);
                    if (lane == 0) atomicAdd(&sm.count, n);
                    __syncthreads();
                    if (sm.count >= keep) hi = mid;
                    else lo = mid + 1;
                }
                __syncthreads();
                if (tid == 0) sm.count = 0;
                __syncthreads();
                each(lo, [&](uint32_t key) { sm.keys[atomicAdd(&sm.count, 1u)] = key; });
                __syncthreads();
            }
            const uint32_t n = sm.count;
            for (uint32_t i = tid; i < n; i += BEAM_THREADS) {
                const uint32_t key = sm.keys[i];
                uint32_t at = 0;
                for (uint32_t k = 0; k < n; k++) at += sm.keys[k] < key;
                if (at < keep) best[at] = key;
            }
            if (tid == 0) *cl.map_shared_rank(&sm.len[item], 0) = (int)(n < keep ? n : keep);
            __syncthreads();  // the list and the count are read
        }
        cl.sync();
        if (rank == 0) {
            // N of a sum: a warp cuts the range in 32 parts at a time.
            auto norm_of = [&](uint64_t W) {
                const u128 one = (u128)a.table[0] * a.table[0];
                int lo = 0, hi = W ? a.tlen : 0;  // the entries below lo pass, those from hi on do not
                while (lo < hi) {
                    const int step = (hi - lo + 31) / 32, j = lo + step * lane;
                    const int pass = __popc(__ballot_sync(0xffffffffu, j < hi && (u128)a.table[j] * W > one));
                    // The first `pass` probes pass: N lies after the last of them, up to the next.
                    if (pass == 0) hi = lo;
                    else {
                        const int next = lo + step * pass;
                        lo = next - step + 1;
                        hi = next < hi ? next : hi;
                    }
                }
                return lo;
            };
            const int lists = a.beams * segs;
            for (uint32_t i = tid; i < (uint32_t)lists * keep; i += BEAM_THREADS) s_place[i] = i % keep;
            if (tid == 0) sm.count = 0;
            __syncthreads();
            for (int b = w; b < a.beams; b += BEAM_WARPS) {
                uint64_t W = 0;
                for (int i = 0; i < segs; i++) W += sm.sum[b * segs + i];
                W <<= cut_bits;
                sm.border[b] = 0;
                if (sm.fin[b] || sm.row[b] < 0 || sm.row[b] >= BASE_LIMIT) continue;
                const uint64_t out = (uint64_t)a.vocab * ((1ull << cut_bits) - 1);  // at most left out
                const int lo = norm_of(W);
                // The upper end gives more if the first entry that does not pass would.
                const uint64_t up = W + out < W ? UINT64_MAX : W + out;
                const bool border = lo < a.tlen && (u128)a.table[lo] * up > (u128)a.table[0] * a.table[0];
                if (lane == 0) {
                    sm.row[b] += lo;
                    sm.border[b] = border;
                    if (border) sm.count = 1;
                }
            }
            __syncthreads();
            if (sm.count) {
                // Sums next to a border of N: the low bits of the weights too, with the table replaced by
                // them for the moment.
                const uint32_t low = (uint32_t)((1ull << cut_bits) - 1);
                for (int i = tid; i < a.tlen; i += BEAM_THREADS) sT[i] = (uint32_t)a.table[i] & low;
                __syncthreads();
                for (int b = 0; b < a.beams; b++) {
                    if (!sm.border[b]) continue;
                    const size_t r = (size_t)group * a.beams + b, lrow = a.row_of ? a.row_of[r] : r;
                    uint64_t W = 0;
#pragma unroll 8
                    for (int v = tid; v < a.vocab; v += BEAM_THREADS) {
                        const uint64_t o = (uint64_t)sm.top[b] - (uint64_t)a.tops[lrow * a.tops_stride + (v >> a.tsh)];
                        const uint32_t D = o < (uint64_t)last ? (uint32_t)o + a.dist[lrow * a.dist_stride + v] : (uint32_t)last;
                        W += sT[D < (uint32_t)last ? D : (uint32_t)last];
                    }
                    for (int o = 16; o > 0; o >>= 1) W += __shfl_xor_sync(0xffffffffu, W, o);
                    if (lane == 0) sm.redu[w] = W;
                    __syncthreads();
                    if (w == 0) {
                        W = 0;
                        for (int i = 0; i < segs; i++) W += sm.sum[b * segs + i];
                        W <<= cut_bits;
                        for (int i = 0; i < BEAM_WARPS; i++) W += sm.redu[i];
                        const int N = norm_of(W);
                        if (lane == 0) sm.row[b] = a.base[r] + N;
                    }
                    __syncthreads();
                }
                for (int i = tid; i < a.tlen; i += BEAM_THREADS) sT[i] = (uint32_t)(a.table[i] >> cut_bits);
                __syncthreads();
            }
            // The merge of the lists: a candidate's place is the number of candidates before it (by cost,
            // then beam, then symbol). Each (candidate, list) pair is a bisection of its own.
            const uint32_t pairs = (uint32_t)lists * keep * (uint32_t)lists;
            for (uint32_t i = tid; i < pairs; i += BEAM_THREADS) {
                const uint32_t cand = i / lists;
                const int o = (int)(i % lists), l = (int)(cand / keep), k = (int)(cand % keep);
                if (o == l || k >= sm.len[l]) continue;
                const int b = l / segs, ob = o / segs;
                const uint32_t key = s_best[l * keep + k];
                const int64_t cost = sm.row[b] + (key >> 16), obase = sm.row[ob];
                int lo = 0, hi = sm.len[o];
                while (lo < hi) {
                    const int mid = (lo + hi) / 2;
                    const uint32_t k2 = s_best[o * keep + mid];
                    const int64_t c = obase + (k2 >> 16);
                    const bool before = ob == b ? k2 < key : c < cost || (c == cost && ob < b);
                    if (before) lo = mid + 1;
                    else hi = mid;
                }
                if (lo) atomicAdd(&s_place[cand], (uint32_t)lo);
            }
            __syncthreads();
            uint32_t total = 0;
            for (int l = 0; l < lists; l++) total += (uint32_t)sm.len[l];
            const size_t out = (size_t)group * keep;
            for (uint32_t i = tid; i < (uint32_t)lists * keep; i += BEAM_THREADS) {
                const int l = (int)(i / keep), k = (int)(i % keep), b = l / segs;
                const uint32_t at = s_place[i];
                if (k >= sm.len[l] || at >= keep) continue;
                const uint32_t key = s_best[l * keep + k];
                a.parent[out + at] = (uint32_t)b;
                a.token[out + at] = sm.fin[b] ? NO_KEY : key & 0xFFFFu;
                a.cost[out + at] = sm.row[b] + (key >> 16);
            }
            for (uint32_t i = total + tid; i < keep; i += BEAM_THREADS) {
                a.parent[out + i] = NO_KEY;
                a.token[out + i] = NO_KEY;
                a.cost[out + i] = -1;
            }
        }
        cl.sync();  // the lists are merged
    }
}

size_t beam_smem(int tlen, int beams, int segs, int keep, int vocab) {
    return 16 * (((size_t)tlen + 4) / 4) + sizeof(BeamSmem) + 8 * (size_t)beams * segs * keep +
           2 * (size_t)(((vocab + 7) / 8 + segs - 1) / segs);
}

}  // namespace

cudaError_t configure_beam() {
    return cudaFuncSetAttribute((const void*)k_beam_select, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)beam_smem(MAX_LOGIT_TABLE, BEAM_LISTS, 1, MAX_KEEP, MAX_CODER_VOCAB));
}

cudaError_t launch_beam_select(const BeamArgs& a, int num_sms, cudaStream_t st) {
    if (a.groups == 0) return cudaSuccess;
    const int vec = reinterpret_cast<uintptr_t>(a.dist) % 16 == 0 && a.dist_stride % 8 == 0;
    // The split: `segs` segments a row and clusters of C blocks, by the time that a wave of clusters
    // takes: the segments of its busiest block (a fixed part each, and one that grows with their symbols)
    // and a merge.
    const int slots = BEAM_BLOCKS * num_sms;
    int segs = 1, C = 1;
    double best = 1e300;
    for (int s = 1; s <= 8; s *= 2) {
        if (s > 1 && (a.beams * s > BEAM_LISTS || a.vocab / s < 4 * BEAM_THREADS)) break;
        for (int c = 1; c <= 8; c *= 2) {
            const double waves = (double)((a.groups + slots / c - 1) / (slots / c));
            const double time = waves * ((a.beams * s + c - 1) / c * (2.0 + 2e-4 * a.vocab / s) + 3.0 + 0.05 * a.beams * s);
            if (time < best) {
                best = time;
                segs = s;
                C = c;
            }
        }
    }
    cudaLaunchConfig_t cfg{};
    const int clusters = slots / C;
    cfg.gridDim = dim3((unsigned)((a.groups < clusters ? a.groups : clusters) * C));
    cfg.blockDim = dim3(BEAM_THREADS);
    cfg.dynamicSmemBytes = beam_smem(a.tlen, a.beams, segs, a.keep, a.vocab);
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)C;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_beam_select, a, segs, vec, a.cut_bits);
}

}  // namespace hs
