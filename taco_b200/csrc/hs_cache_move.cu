// The moves of KV-cache rows: the reordering of the beams' states after a selection and the commit of
// an accepted path of a draft tree. Both are in place: a thread owns the same bytes of every slot (or
// row) that takes part, reads all of them before it writes any, so no order of threads matters.
// Bytes in and out are the only cost (times: B200, 144 planes of 1,024 rows of 64, calls repeated on the same
// caches; in a reorder every beam takes another one's rows, so all of them are read and written).
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "hs_common.cuh"
#include "hs_draft.hpp"

namespace hs {

namespace {

// Threads of a block of the kernel for B beams: 32 loads of 16 bytes a thread want more registers than 256
// threads have (8 groups of 16 beams of 700 rows by the kernel for 32: 1.17 ms, 0.66 with 128 threads; the
// kernel for 16 0.59, and with 128 threads 0.60, that for 4 0.58 against 0.56).
__host__ __device__ constexpr int move_threads(int B) { return B > 16 ? 128 : 256; }

// The first n bytes (1 to 15) of a unit, in a store for each bit of n.
__device__ __forceinline__ void put_head(int8_t* to, uint4 v, uint32_t n) {
    uint32_t a = v.x, b = v.y;
    if (n & 8) {
        *reinterpret_cast<uint2*>(to) = make_uint2(v.x, v.y);
        to += 8;
        a = v.z;
        b = v.w;
    }
    if (n & 4) {
        *reinterpret_cast<uint32_t*>(to) = a;
        to += 4;
        a = b;
    }
    if (n & 2) {
        *reinterpret_cast<uint16_t*>(to) = (uint16_t)a;
        to += 2;
        a >>= 16;
    }
    if (n & 1) *to = (int8_t)a;
}

// T: the unit of a move (16 bytes where n_ctx and head_dim are multiples of 16, else a byte). B: the
// most beams of a group. blockIdx.y is the group, blockIdx.x a plane's keys (rows * hd bytes from row 0)
// or values (the first `rows` bytes of each channel's row): a unit of values may pass the last row, and
// then goes by parts (byte by byte one group of 8 beams of 300 rows took 30 us cold, by parts 20). Caches whose
// sizes or addresses are no multiples of 16 go by bytes: 32 groups of 4 of 700 rows, n_ctx 1,000, half of the beams
// living on, 1.64 ms, a group of 8 of 300 rows 55 us.
//
// Bound by HBM: 32 groups of 4 beams of 700 rows take 0.56 ms (5.9 TB/s in and out, 90 % of a copy's rate; 0.37 to
// 0.40 where about half of the beams live on), 16 of 8 0.57, 8 of 16 0.61. The loads of beams that a group does not have cost: the kernel for 32 takes 1.2 ms with
// groups of 4, so there is one for 4, 8, 16 and 32.
template <typename T, int B>
__global__ void __launch_bounds__(move_threads(B)) k_cache_reorder(const CacheView c, const uint32_t* slots,
                                                                const uint32_t* parents, const uint32_t* rows,
                                                                uint32_t groups, uint32_t beams, int* err) {
    __shared__ uint32_t s_dst[B], s_src[B], s_rows[B];  // the moves of the group: slots, and the rows moved
    __shared__ uint32_t s_n, s_most, s_bad;
    constexpr int W = (int)sizeof(T), MOVE_THREADS = move_threads(B);
    for (uint32_t g = blockIdx.y; g < groups; g += gridDim.y) {
        __syncthreads();
        if (threadIdx.x < 32) {
            // Lane j looks at beam j; the moves keep their order.
            const uint32_t j = threadIdx.x, at = g * beams + j;
            const uint32_t p = j < beams ? parents[at] : 0xFFFFFFFFu;
            bool move = p != j && p != 0xFFFFFFFFu, bad = move && p >= beams;
            uint32_t dst = 0, src = 0, r = 0;
            if (move && !bad) {
                dst = slots ? slots[at] : at;
                src = slots ? slots[g * beams + p] : g * beams + p;
                r = rows[g * beams + p];
                bad = dst >= c.slots || src >= c.slots || r > (uint32_t)c.n_ctx;
            }
            move = move && !bad;
            const uint32_t all = __ballot_sync(0xffffffffu, move), any_bad = __ballot_sync(0xffffffffu, bad);
            if (move) {
                const int n = __popc(all & ((1u << j) - 1u));
                s_dst[n] = dst;
                s_src[n] = src;
                s_rows[n] = r;
            }
            const uint32_t most = __reduce_max_sync(0xffffffffu, move ? r : 0u);
            if (j == 0) {
                s_n = (uint32_t)__popc(all);
                s_most = most;
                s_bad = any_bad;
            }
        }
        __syncthreads();
        const int n = (int)s_n;
        if (s_bad && threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.z == 0) atomicCAS(err, 0, ERR_DRAFT_PARENT);
        if (n == 0) continue;
        const size_t plane = (size_t)(blockIdx.x >> 1) * c.n_ctx * c.hd;  // (blockIdx.z: a part of its units)
        const bool values = blockIdx.x & 1;
        int8_t* base = (values ? c.v : c.k) + plane;
        // Units of a channel's values, and of the plane's keys or values in all (at most 8192 * 1024).
        const uint32_t vu = (s_most + W - 1) / W, total = values ? vu * c.hd : s_most * c.hd / W;
#pragma unroll 1
        for (uint32_t u = blockIdx.z * MOVE_THREADS + threadIdx.x; u < total; u += gridDim.z * MOVE_THREADS) {
            const uint32_t ch = values ? u / vu : 0, x = (values ? u - ch * vu : u) * W;  // the unit's first byte
            int8_t* at = base + (size_t)ch * c.n_ctx + x;
            const uint32_t row = values ? 1 : c.hd;  // bytes of a row in this run of bytes
            T val[B];
#pragma unroll
            for (int j = 0; j < B; j++)
                if (j < n && x < s_rows[j] * row) val[j] = *reinterpret_cast<const T*>(at + s_src[j] * c.slot_stride);
#pragma unroll
            for (int j = 0; j < B; j++) {
                if (j >= n || x >= s_rows[j] * row) continue;
                int8_t* to = at + s_dst[j] * c.slot_stride;
                if (W == 1 || x + W <= s_rows[j] * row) {
                    *reinterpret_cast<T*>(to) = val[j];
                } else {
                    // The last rows of a channel's values end inside the unit.
                    if constexpr (W == 16) put_head(to, val[j], s_rows[j] - x);
                }
            }
        }
    }
}

// A warp moves parts of planes of one tree: a plane's keys (part 0) or some channels of its values.
// path is strictly increasing, so path[j] >= j: taken in ascending runs, all of a run's rows read before
// any is written, no row is written before it is read. The bytes of a path lie in a few 32-byte sectors of
// each channel's row of values: that traffic is the cost. A lane takes a path's byte of COMMIT_DEEP channels,
// all in flight: 64 trees with a path of 8, their sectors in L2, take 28 us with 32 channels and three blocks an
// SM, 32 with 16 channels and 36 with 64 (paths of 24 of 128 nodes 54, 58, 55 us); from HBM 39 (and 50) us, where the
// sectors alone would be 17 (25). A byte a lane is what is left: with a path of 8 a quarter of the lanes have one. A
// warp shared by several channels of short paths is no faster (35 us).
constexpr int COMMIT_DEEP = 32, COMMIT_WARPS = 8, COMMIT_BLOCKS = 3;

template <bool VEC>
__global__ void __launch_bounds__(32 * COMMIT_WARPS, COMMIT_BLOCKS) k_cache_commit(const CacheView c, const TreeSeq* seqs,
                                                                   const uint32_t* path, const uint32_t* lengths,
                                                                   uint32_t path_stride, int parts, uint32_t units,
                                                                   int* err) {
    const int lane = threadIdx.x & 31;
    const uint32_t first = blockIdx.y * (uint32_t)COMMIT_WARPS + (threadIdx.x >> 5);  // unit of the tree
    const uint32_t i = blockIdx.x;
    const TreeSeq s = seqs[i];
    const uint32_t m = lengths[i];
    bool bad = m > path_stride || m > s.count || s.count > (uint32_t)MAX_TREE || s.slot >= c.slots ||
               s.prefix > (uint32_t)c.n_ctx || s.count > (uint32_t)c.n_ctx - s.prefix;
    // Lane l holds the path's entries l, l + 32, ...; the ones past its end are not read, and stay where they are.
    uint32_t p[MAX_TREE / 32];
    uint32_t before = 0;  // the last entry of the run before, plus one
    if (!bad) {
#pragma unroll
        for (int k = 0; k < MAX_TREE / 32; k++) {
            const uint32_t j = 32 * k + lane;
            p[k] = j < m ? path[(size_t)i * path_stride + j] : j;
        }
#pragma unroll
        for (int k = 0; k < MAX_TREE / 32; k++) {
            const uint32_t j = 32 * k + lane;
            uint32_t up = __shfl_up_sync(0xffffffffu, p[k], 1);
            if (lane == 0) up = before - 1;
            bad = bad || (j < m && (p[k] >= s.count || (j > 0 && p[k] <= up)));
            before = __shfl_sync(0xffffffffu, p[k], 31) + 1;
        }
    }
    if (__any_sync(0xffffffffu, bad)) {
        if (lane == 0 && first == 0) atomicCAS(err, 0, ERR_DRAFT_PATH);
        return;
    }
    for (uint32_t unit = first; unit < units; unit += gridDim.y * COMMIT_WARPS) {
        const uint32_t plane = unit / (uint32_t)parts, part = unit % (uint32_t)parts;
        const size_t base = s.slot * c.slot_stride + (size_t)plane * ((size_t)c.n_ctx * c.hd);
        if (part == 0) {
            int8_t* K = c.k + base + (size_t)s.prefix * c.hd;
            using T = typename std::conditional<VEC, uint4, uint8_t>::type;
            const uint32_t pieces = c.hd / (uint32_t)sizeof(T);  // of a row
            for (uint32_t k0 = 0; k0 * 32 < m; k0++) {
                // Runs of 8 rows (an entry of the path from the lane that holds it).
                for (uint32_t j0 = 32 * k0; j0 < 32 * k0 + 32 && j0 < m; j0 += 8) {
                    for (uint32_t x0 = 0; x0 < pieces; x0 += 4) {
                        const uint32_t j = j0 + (lane >> 2), x = x0 + (lane & 3);
                        const uint32_t from = __shfl_sync(0xffffffffu, k0 == 0 ? p[0] : k0 == 1 ? p[1] : k0 == 2 ? p[2] : p[3],
                                                          (int)(j & 31));
                        const bool move = j < m && x < pieces && from != j;
                        T val;
                        if (move) val = reinterpret_cast<const T*>(K + (size_t)from * c.hd)[x];
                        __syncwarp();
                        if (move) reinterpret_cast<T*>(K + (size_t)j * c.hd)[x] = val;
                        __syncwarp();
                    }
                }
            }
            continue;
        }
        const int ch0 = (int)(part - 1) * COMMIT_DEEP, n = min(COMMIT_DEEP, c.hd - ch0);
        int8_t* V = c.v + base + (size_t)ch0 * c.n_ctx + s.prefix;
        for (uint32_t k0 = 0; k0 * 32 < m; k0++) {
            const uint32_t j = 32 * k0 + lane, from = k0 == 0 ? p[0] : k0 == 1 ? p[1] : k0 == 2 ? p[2] : p[3];
            const int mine = j < m && from != j ? n : 0;
            const int8_t* of = V + from;
            int8_t* to = V + j;
            int8_t val[COMMIT_DEEP];
#pragma unroll
            for (int q = 0; q < COMMIT_DEEP; q++, of += c.n_ctx)
                if (q < mine) val[q] = *of;
            __syncwarp();
#pragma unroll
            for (int q = 0; q < COMMIT_DEEP; q++, to += c.n_ctx)
                if (q < mine) *to = val[q];
            __syncwarp();
        }
    }
}

template <typename T, int B>
void reorder(const CacheView& c, const uint32_t* slots, const uint32_t* parents, const uint32_t* rows, uint32_t groups,
             uint32_t beams, int num_sms, int* err, cudaStream_t st) {
    // Blocks beyond one for each group and plane's keys or values: up to 6 for an SM, so that few groups have
    // many loads in flight, each with at least two units a thread at a full context. One group of 4 beams of 300
    // rows in L2: 9.1 us; 10.2 without the parts, 10.5 with up to 16 for an SM (8: 14.8, 14.7, 16.7).
    const uint64_t blocks = 2ull * c.planes * groups, full = (uint64_t)c.n_ctx * c.hd / sizeof(T);
    const uint64_t most = (full + 2 * move_threads(B) - 1) / (2 * move_threads(B));
    const uint64_t parts = std::min<uint64_t>({(6ull * num_sms + blocks - 1) / blocks, most, 64});
    const dim3 grid(2 * c.planes, groups < 65535u ? groups : 65535u, (unsigned)parts);
    k_cache_reorder<T, B><<<grid, move_threads(B), 0, st>>>(c, slots, parents, rows, groups, beams, err);
}

template <typename T>
void reorder_any(const CacheView& c, const uint32_t* slots, const uint32_t* parents, const uint32_t* rows, uint32_t groups,
                 uint32_t beams, int num_sms, int* err, cudaStream_t st) {
    if (beams <= 4) reorder<T, 4>(c, slots, parents, rows, groups, beams, num_sms, err, st);
    else if (beams <= 8) reorder<T, 8>(c, slots, parents, rows, groups, beams, num_sms, err, st);
    else if (beams <= 16) reorder<T, 16>(c, slots, parents, rows, groups, beams, num_sms, err, st);
    else reorder<T, 32>(c, slots, parents, rows, groups, beams, num_sms, err, st);
}

}  // namespace

cudaError_t launch_cache_reorder(const CacheView& c, const uint32_t* slots, const uint32_t* parents,
                                 const uint32_t* rows, uint32_t groups, uint32_t beams, int num_sms, int* err,
                                 cudaStream_t st) {
    if (groups == 0 || beams == 0) return cudaSuccess;  // (one beam: nothing moves, but its parent is checked)
    if (c.vec) reorder_any<uint4>(c, slots, parents, rows, groups, beams, num_sms, err, st);
    else reorder_any<uint8_t>(c, slots, parents, rows, groups, beams, num_sms, err, st);
    return cudaGetLastError();
}

cudaError_t launch_cache_commit(const CacheView& c, const TreeSeq* seqs, const uint32_t* path, const uint32_t* lengths,
                                uint32_t n_seq, uint32_t path_stride, int* err, cudaStream_t st) {
    if (n_seq == 0) return cudaSuccess;
    const int parts = 1 + (c.hd + COMMIT_DEEP - 1) / COMMIT_DEEP;
    const uint32_t units = c.planes * (uint32_t)parts;
    const uint32_t blocks = (units + COMMIT_WARPS - 1) / COMMIT_WARPS;
    const dim3 grid(n_seq, blocks < 65535u ? blocks : 65535u);
    if (c.vec)
        k_cache_commit<true><<<grid, 32 * COMMIT_WARPS, 0, st>>>(c, seqs, path, lengths, path_stride, parts, units, err);
    else
        k_cache_commit<false><<<grid, 32 * COMMIT_WARPS, 0, st>>>(c, seqs, path, lengths, path_stride, parts, units, err);
    return cudaGetLastError();
}

}  // namespace hs
