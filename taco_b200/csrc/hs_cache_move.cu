// The moves of KV-cache rows: the reordering of the beams' states after a selection and the commit of
// an accepted path of a draft tree. Both are in place: a thread owns the same bytes of every slot (or
// row) that takes part, reads all of them before it writes any, so no order of threads matters.
// Bytes in and out are the only cost.
#include <cuda_runtime.h>

#include <cstdint>

#include "hs_common.cuh"
#include "hs_draft.hpp"

namespace hs {

namespace {

constexpr int MOVE_THREADS = 256;

// T: the unit of a move (16 bytes where n_ctx and head_dim are multiples of 16, else a byte). B: the
// most beams of a group. blockIdx.y is the group. The units of a plane are its keys (rows * hd bytes
// from row 0), then its values (the first `rows` bytes of each channel's row): a unit of values may
// pass the last row, and then goes byte by byte.
template <typename T, int B>
__global__ void __launch_bounds__(MOVE_THREADS) k_cache_reorder(const CacheView c, const uint32_t* slots,
                                                                const uint32_t* parents, const uint32_t* rows,
                                                                uint32_t groups, uint32_t beams, int* err) {
    __shared__ uint32_t s_dst[B], s_src[B], s_rows[B];  // the moves of the group: slots, and the rows moved
    __shared__ uint32_t s_n, s_most, s_bad;
    constexpr int W = (int)sizeof(T);
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
        if (s_bad && threadIdx.x == 0 && blockIdx.x == 0) atomicCAS(err, 0, ERR_DRAFT_PARENT);
        if (n == 0) continue;
        const uint32_t most = s_most;
        const size_t ku = (size_t)most * c.hd / W;          // units of a plane's keys
        const size_t vu = ((size_t)most + W - 1) / W;       // units of a channel's values
        const size_t per_plane = ku + vu * c.hd, total = per_plane * c.planes;
        const size_t plane_bytes = (size_t)c.n_ctx * c.hd;
        for (size_t u = (size_t)blockIdx.x * MOVE_THREADS + threadIdx.x; u < total;
             u += (size_t)gridDim.x * MOVE_THREADS) {
            const size_t plane = u / per_plane, r = u % per_plane;
            T val[B];
            if (r < ku) {
                const size_t off = plane * plane_bytes + r * W;
#pragma unroll
                for (int j = 0; j < B; j++)
                    if (j < n && r * W < (size_t)s_rows[j] * c.hd)
                        val[j] = *reinterpret_cast<const T*>(c.k + s_src[j] * c.slot_stride + off);
#pragma unroll
                for (int j = 0; j < B; j++)
                    if (j < n && r * W < (size_t)s_rows[j] * c.hd)
                        *reinterpret_cast<T*>(c.k + s_dst[j] * c.slot_stride + off) = val[j];
            } else {
                const size_t ch = (r - ku) / vu, x = (r - ku) % vu * W;
                const size_t off = plane * plane_bytes + ch * c.n_ctx + x;
#pragma unroll
                for (int j = 0; j < B; j++)
                    if (j < n && x < s_rows[j])
                        val[j] = *reinterpret_cast<const T*>(c.v + s_src[j] * c.slot_stride + off);
#pragma unroll
                for (int j = 0; j < B; j++) {
                    if (j >= n || x >= s_rows[j]) continue;
                    int8_t* to = c.v + s_dst[j] * c.slot_stride + off;
                    if (x + W <= s_rows[j]) {
                        *reinterpret_cast<T*>(to) = val[j];
                    } else {
                        const int8_t* b = reinterpret_cast<const int8_t*>(&val[j]);
                        for (int i = 0; i < (int)(s_rows[j] - x); i++) to[i] = b[i];
                    }
                }
            }
        }
    }
}

// One block per (tree, plane). Row prefix + path[j] -> prefix + j with path strictly increasing, so
// path[j] >= j and a source not yet read is above every row written: a thread moves its bytes in
// ascending order of j.
__global__ void __launch_bounds__(128) k_cache_commit(const CacheView c, const TreeSeq* seqs, const uint32_t* path,
                                                      const uint32_t* lengths, uint32_t n_seq, uint32_t path_stride,
                                                      int* err) {
    __shared__ uint32_t s_path[MAX_TREE];
    __shared__ int s_bad;
    const uint32_t i = blockIdx.x;
    const TreeSeq s = seqs[i];
    const uint32_t m = lengths[i];
    if (threadIdx.x == 0) s_bad = 0;
    __syncthreads();
    bool bad = m > path_stride || m > s.count || s.count > MAX_TREE || s.slot >= c.slots ||
               s.prefix > (uint32_t)c.n_ctx || s.count > (uint32_t)c.n_ctx - s.prefix;
    if (!bad && threadIdx.x < m) {
        const uint32_t p = path[(size_t)i * path_stride + threadIdx.x];
        s_path[threadIdx.x] = p;
        bad = p >= s.count || (threadIdx.x > 0 && p <= path[(size_t)i * path_stride + threadIdx.x - 1]);
    }
    if (bad) s_bad = 1;
    __syncthreads();
    if (s_bad) {
        if (threadIdx.x == 0) atomicCAS(err, 0, ERR_DRAFT_PATH);
        return;
    }
    const size_t base = s.slot * c.slot_stride + (size_t)blockIdx.y * ((size_t)c.n_ctx * c.hd);
    int8_t* K = c.k + base + (size_t)s.prefix * c.hd;
    int8_t* V = c.v + base + s.prefix;
    for (int b = threadIdx.x; b < c.hd; b += 128) {
        for (uint32_t j = 0; j < m; j++) {
            K[(size_t)j * c.hd + b] = K[(size_t)s_path[j] * c.hd + b];
            V[(size_t)b * c.n_ctx + j] = V[(size_t)b * c.n_ctx + s_path[j]];
        }
    }
}

template <typename T>
void reorder(const CacheView& c, const uint32_t* slots, const uint32_t* parents, const uint32_t* rows, uint32_t groups,
             uint32_t beams, dim3 grid, int* err, cudaStream_t st) {
    if (beams <= 4) k_cache_reorder<T, 4><<<grid, MOVE_THREADS, 0, st>>>(c, slots, parents, rows, groups, beams, err);
    else if (beams <= 8) k_cache_reorder<T, 8><<<grid, MOVE_THREADS, 0, st>>>(c, slots, parents, rows, groups, beams, err);
    else if (beams <= 16) k_cache_reorder<T, 16><<<grid, MOVE_THREADS, 0, st>>>(c, slots, parents, rows, groups, beams, err);
    else k_cache_reorder<T, 32><<<grid, MOVE_THREADS, 0, st>>>(c, slots, parents, rows, groups, beams, err);
}

}  // namespace

cudaError_t launch_cache_reorder(const CacheView& c, const uint32_t* slots, const uint32_t* parents,
                                 const uint32_t* rows, uint32_t groups, uint32_t beams, int num_sms, int* err,
                                 cudaStream_t st) {
    if (groups == 0 || beams < 2) return cudaSuccess;
    const uint32_t gy = groups < 65535u ? groups : 65535u;
    const uint32_t gx = (uint32_t)(num_sms * 8 + (int)gy - 1) / gy;
    const dim3 grid(gx < 1 ? 1 : gx, gy);
    if (c.vec) reorder<uint4>(c, slots, parents, rows, groups, beams, grid, err, st);
    else reorder<uint8_t>(c, slots, parents, rows, groups, beams, grid, err, st);
    return cudaGetLastError();
}

cudaError_t launch_cache_commit(const CacheView& c, const TreeSeq* seqs, const uint32_t* path, const uint32_t* lengths,
                                uint32_t n_seq, uint32_t path_stride, int num_sms, int* err, cudaStream_t st) {
    (void)num_sms;
    if (n_seq == 0) return cudaSuccess;
    k_cache_commit<<<dim3(n_seq, c.planes), 128, 0, st>>>(c, seqs, path, lengths, n_seq, path_stride, err);
    return cudaGetLastError();
}

}  // namespace hs
