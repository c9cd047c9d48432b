// The selection of a beam search over beams and vocabulary (hs_op_beam_select, hs_batch_beam_step).
//
// A row of logits is read as the LM head leaves it: u16 distances from the tile maxima. A symbol's
// distance D from the row maximum is the whole number of table units that its log weight lies below
// the largest, so D is its cost up to the row's normaliser: cost = base + N + D with N = #{j :
// table[j] W > table[0]^2}, the least j at which table[j] / table[0] is not above table[0] / W. A
// symbol's key is D << 16 | symbol: keys are distinct, their order is the order of the candidates of a
// row (the lower symbol first among equal distances), and they fit in 30 bits.
//
// A cluster of blocks takes a group; its items are the rows' segments (2 to 8 a row), dealt round-robin
// to the blocks. A block reads a segment once and holds its distances in registers, two in a word. It sums
// the weights (one table look-up per symbol, the table in shared memory: this bounds the kernel) and finds
// the segment's `keep` smallest keys: the keep-th smallest of 128 threads-of-four minima is a distance that
// at least `keep` symbols are not above, so only symbols up to it are candidates (about `keep` of them,
// unless distances tie), and each finds its place by counting. The lists and sums go to the first block's
// shared memory, which adds the normalisers and merges the lists.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "hs_common.cuh"
#include "hs_draft.hpp"

namespace cg = cooperative_groups;

namespace hs {

namespace {

constexpr int BEAM_THREADS = 512;
constexpr int BEAM_VECS = 8;     // groups of 8 symbols of a thread: a segment of up to 32,768 symbols
constexpr int BEAM_GROUPS = 128; // the minima that give the first threshold (four threads each)
constexpr int BEAM_LIST = 1024;  // symbols up to the threshold that are held
constexpr int BEAM_LISTS = 2 * MAX_BEAMS;
constexpr uint32_t NO_KEY = 0xFFFFFFFFu;
constexpr int64_t BASE_LIMIT = 1LL << 62;
static_assert(MAX_KEEP <= BEAM_GROUPS, "the threshold needs as many minima as places");
static_assert(2 * BEAM_VECS * BEAM_THREADS * 8 >= MAX_CODER_VOCAB, "two segments hold every vocabulary");

struct BeamSmem {
    // The segment in work.
    int64_t red[BEAM_THREADS / 32];
    uint64_t redu[BEAM_THREADS / 32];
    uint16_t off[MAX_CODER_VOCAB / 64];  // the tiles' distances from the row maximum, cut at the table
    __align__(16) uint32_t least[BEAM_GROUPS];
    uint32_t list[BEAM_LIST];
    uint32_t cut, count;
    // The group's lists (in the cluster's first block).
    uint32_t best[BEAM_LISTS][MAX_KEEP];
    int len[BEAM_LISTS];
    uint64_t sum[BEAM_LISTS];
    int64_t row[MAX_BEAMS];  // base + N
    uint8_t fin[MAX_BEAMS];
};

__global__ void __launch_bounds__(BEAM_THREADS, 2) k_beam_select(const __grid_constant__ BeamArgs a, int segs, int vec) {
    extern __shared__ __align__(16) uint8_t s_beam[];
    uint64_t* sT = reinterpret_cast<uint64_t*>(s_beam);  // tlen weights, then 0 for no symbol
    BeamSmem& sm = *reinterpret_cast<BeamSmem*>(s_beam + 8 * (((size_t)a.tlen + 2) & ~(size_t)1));
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    const int last = a.tlen - 1, tiles = (a.vocab + (1 << a.tsh) - 1) >> a.tsh;
    const uint32_t keep = (uint32_t)a.keep, last2 = (uint32_t)last * 0x10001u, no_symbol = (uint32_t)a.tlen;
    const int vecs = (a.vocab + 7) / 8, seg_vecs = (vecs + segs - 1) / segs;
    for (int i = tid; i <= a.tlen; i += BEAM_THREADS) sT[i] = i < a.tlen ? a.table[i] : 0;
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
            uint32_t* best = cl.map_shared_rank(sm.best[item], 0);
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
            // The segment's distances from the tile maxima, 8 symbols a vector.
            uint32_t d[BEAM_VECS][4];
#pragma unroll
            for (int k = 0; k < BEAM_VECS; k++) {
                const int v = v0 + tid + k * BEAM_THREADS;
                d[k][0] = d[k][1] = d[k][2] = d[k][3] = 0;
                if (v >= v1) continue;
                if (vec && 8 * v + 8 <= a.vocab) {
                    const uint4 x = __ldg(reinterpret_cast<const uint4*>(dist + 8 * (size_t)v));
                    d[k][0] = x.x;
                    d[k][1] = x.y;
                    d[k][2] = x.z;
                    d[k][3] = x.w;
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if (8 * v + j < a.vocab) d[k][j >> 1] |= (uint32_t)dist[8 * (size_t)v + j] << (16 * (j & 1));
                }
            }
            int64_t mx = INT64_MIN;
            for (int t = tid; t < tiles; t += BEAM_THREADS) mx = tops[t] > mx ? tops[t] : mx;
            for (int o = 16; o > 0; o >>= 1) {
                const int64_t x = __shfl_xor_sync(0xffffffffu, mx, o);
                mx = x > mx ? x : mx;
            }
            if (lane == 0) sm.red[w] = mx;
            __syncthreads();
            for (int i = 0; i < BEAM_THREADS / 32; i++) mx = sm.red[i] > mx ? sm.red[i] : mx;
            // The offset as an unsigned difference: right for any maxima, and never below 0.
            for (int t = tid; t < tiles; t += BEAM_THREADS) {
                const uint64_t o = (uint64_t)mx - (uint64_t)tops[t];
                sm.off[t] = (uint16_t)(o < (uint64_t)last ? o : (uint64_t)last);
            }
            if (tid == 0) sm.count = 0;
            __syncthreads();
            // D = min(offset + distance, last) of two symbols at a time (the sum saturates above last).
            uint64_t sum = 0;
            uint32_t least2 = no_symbol * 0x10001u;
#pragma unroll
            for (int k = 0; k < BEAM_VECS; k++) {
                const int v = v0 + tid + k * BEAM_THREADS;
                uint32_t(&x)[4] = d[k];
                if (v >= v1) {
                    x[0] = x[1] = x[2] = x[3] = no_symbol * 0x10001u;
                    continue;
                }
                const uint32_t off2 = (uint32_t)sm.off[(8 * v) >> a.tsh] * 0x10001u;
#pragma unroll
                for (int j = 0; j < 4; j++) x[j] = __vminu2(__vaddus2(x[j], off2), last2);
                if (8 * v + 8 > a.vocab) {
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if (8 * v + j >= a.vocab)
                            x[j >> 1] = __byte_perm(x[j >> 1], no_symbol, j & 1 ? 0x5410 : 0x3254);
                }
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    sum += sT[x[j] & 0xFFFFu] + sT[x[j] >> 16];
                    least2 = __vminu2(least2, x[j]);
                }
            }
            uint32_t least = min(least2 & 0xFFFFu, least2 >> 16);
            least = min(least, __shfl_xor_sync(0xffffffffu, least, 1));
            least = min(least, __shfl_xor_sync(0xffffffffu, least, 2));
            if ((lane & 3) == 0) sm.least[tid >> 2] = least;
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) sm.redu[w] = sum;
            __syncthreads();
            if (tid < BEAM_GROUPS) {
                // The place of a minimum among the minima (equal ones by their index).
                const uint32_t mine = sm.least[tid];
                uint32_t at = 0;
#pragma unroll 8
                for (int i = 0; i < BEAM_GROUPS; i += 4) {
                    const uint4 o = *reinterpret_cast<const uint4*>(&sm.least[i]);
                    at += (o.x < mine || (o.x == mine && i < tid)) + (o.y < mine || (o.y == mine && i + 1 < tid)) +
                          (o.z < mine || (o.z == mine && i + 2 < tid)) + (o.w < mine || (o.w == mine && i + 3 < tid));
                }
                if (at == keep - 1) sm.cut = mine;
            } else if (tid == BEAM_GROUPS) {
                uint64_t all = 0;
                for (int i = 0; i < BEAM_THREADS / 32; i++) all += sm.redu[i];
                *cl.map_shared_rank(&sm.sum[item], 0) = all;
            }
            __syncthreads();
            const uint32_t cut = min(sm.cut, (uint32_t)a.last_weight);
            // f(key) for every symbol with D <= cut.
            auto near = [&](uint32_t cut, auto f) {
                const uint32_t cut2 = cut * 0x10001u;
#pragma unroll
                for (int k = 0; k < BEAM_VECS; k++) {
                    const uint32_t(&x)[4] = d[k];
                    const uint32_t least = __vminu2(__vminu2(x[0], x[1]), __vminu2(x[2], x[3]));
                    if (__vcmpleu2(least, cut2) == 0) continue;
                    const uint32_t sym = 8u * (uint32_t)(v0 + tid + k * BEAM_THREADS);
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const uint32_t D = j & 1 ? x[j >> 1] >> 16 : x[j >> 1] & 0xFFFFu;
                        if (D <= cut) f(D << 16 | (sym + j));
                    }
                }
            };
            auto collect = [&](uint32_t upto) {
                near(upto >> 16, [&](uint32_t key) {
                    if (key > upto) return;
                    const uint32_t at = atomicAdd(&sm.count, 1u);
                    if (at < BEAM_LIST) sm.list[at] = key;
                });
                __syncthreads();
            };
            collect(cut << 16 | 0xFFFFu);
            if (sm.count > BEAM_LIST) {
                // Distances tie: the least key that `keep` keys are not above, by bisection over keys.
                uint32_t lo = 0, hi = cut << 16 | 0xFFFFu;
                while (lo < hi) {
                    const uint32_t mid = lo + (hi - lo) / 2;
                    __syncthreads();
                    if (tid == 0) sm.count = 0;
                    __syncthreads();
                    uint32_t n = 0;
                    near(mid >> 16, [&](uint32_t key) { n += key <= mid; });
                    n = __reduce_add_sync(0xffffffffu, n);
                    if (lane == 0) atomicAdd(&sm.count, n);
                    __syncthreads();
                    if (sm.count >= keep) hi = mid;
                    else lo = mid + 1;
                }
                __syncthreads();
                if (tid == 0) sm.count = 0;
                __syncthreads();
                collect(lo);
            }
            const uint32_t n = sm.count;
            for (uint32_t i = tid; i < n; i += BEAM_THREADS) {
                const uint32_t key = sm.list[i];
                uint32_t at = 0;
                for (uint32_t k = 0; k < n; k++) at += sm.list[k] < key;
                if (at < keep) best[at] = key;
            }
            if (tid == 0) *cl.map_shared_rank(&sm.len[item], 0) = (int)(n < keep ? n : keep);
            __syncthreads();  // the list and the count are read
        }
        cl.sync();
        if (rank == 0) {
            // The normalisers: a warp takes a row and cuts the range of N in 32 parts at a time.
            for (int b = w; b < a.beams; b += BEAM_THREADS / 32) {
                uint64_t W = 0;
                for (int i = 0; i < segs; i++) W += sm.sum[b * segs + i];
                const u128 one = (u128)sT[0] * sT[0];
                int lo = 0, hi = W ? a.tlen : 0;  // the entries below lo pass, those from hi on do not
                while (lo < hi) {
                    const int step = (hi - lo + 31) / 32, j = lo + step * lane;
                    const int pass = __popc(__ballot_sync(0xffffffffu, j < hi && (u128)sT[j] * W > one));
                    // The first `pass` probes pass: N lies after the last of them, up to the next.
                    if (pass == 0) hi = lo;
                    else {
                        const int next = lo + step * pass;
                        lo = next - step + 1;
                        hi = next < hi ? next : hi;
                    }
                }
                __syncwarp();
                if (lane == 0) sm.row[b] += lo;
            }
            __syncthreads();
            // The merge of the lists: a candidate's place is the number of candidates before it (by cost,
            // then beam, then symbol), by bisection in every list.
            const int lists = a.beams * segs;
            uint32_t total = 0;
            for (int l = 0; l < lists; l++) total += (uint32_t)sm.len[l];
            const size_t out = (size_t)group * keep;
            for (uint32_t i = tid; i < (uint32_t)lists * keep; i += BEAM_THREADS) {
                const int l = (int)(i / keep), k = (int)(i % keep), b = l / segs;
                if (k >= sm.len[l]) continue;
                const uint32_t key = sm.best[l][k];
                const int64_t cost = sm.row[b] + (key >> 16);
                uint32_t at = (uint32_t)k;
                for (int o = 0; o < lists && at < keep; o++) {
                    if (o == l) continue;
                    const int ob = o / segs;
                    const int64_t obase = sm.row[ob];
                    int lo = 0, hi = sm.len[o];
                    while (lo < hi) {
                        const int mid = (lo + hi) / 2;
                        const uint32_t k2 = sm.best[o][mid];
                        const int64_t c = obase + (k2 >> 16);
                        const bool before = ob == b ? k2 < key : c < cost || (c == cost && ob < b);
                        if (before) lo = mid + 1;
                        else hi = mid;
                    }
                    at += (uint32_t)lo;
                }
                if (at < keep) {
                    a.parent[out + at] = (uint32_t)b;
                    a.token[out + at] = sm.fin[b] ? NO_KEY : key & 0xFFFFu;
                    a.cost[out + at] = cost;
                }
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

size_t beam_smem(int tlen) { return 8 * (((size_t)tlen + 2) & ~(size_t)1) + sizeof(BeamSmem); }

}  // namespace

cudaError_t configure_beam() {
    return cudaFuncSetAttribute((const void*)k_beam_select, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)beam_smem(MAX_LOGIT_TABLE));
}

cudaError_t launch_beam_select(const BeamArgs& a, int num_sms, cudaStream_t st) {
    if (a.groups == 0) return cudaSuccess;
    const int vec = reinterpret_cast<uintptr_t>(a.dist) % 16 == 0 && a.dist_stride % 8 == 0;
    // Two segments a row hold every vocabulary; more where the rows are too few to fill the GPU and a
    // segment keeps a full round of vectors.
    int segs = 2;
    while (segs < 8 && a.beams * segs * 2 <= BEAM_LISTS && a.groups * a.beams * segs * 2 <= 2 * num_sms &&
           a.vocab / (segs * 2) >= 8 * BEAM_THREADS)
        segs *= 2;
    const int C = a.beams * segs < 8 ? a.beams * segs : 8;
    cudaLaunchConfig_t cfg{};
    const int clusters = 2 * num_sms / C;
    cfg.gridDim = dim3((unsigned)((a.groups < clusters ? a.groups : clusters) * C));
    cfg.blockDim = dim3(BEAM_THREADS);
    cfg.dynamicSmemBytes = beam_smem(a.tlen);
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)C;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_beam_select, a, segs, vec);
}

}  // namespace hs
