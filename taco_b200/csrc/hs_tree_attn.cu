// Attention of trees of drafted tokens over the KV cache (hs_op_tree_attention, hs_batch_run_tree).
//
// A tree's nodes are query rows; node j's keys and values are in cache row prefix + j of its slot.
// A row attends to the slot's context (cache rows 0 .. prefix - 1) and to the nodes in its mask. The
// softmax is HardShell's (crates/hardshell/src/softmax.rs:78-104): the exact row maximum before any
// weight and the exact row sum before any probability, p = floor(e 2^P / sum), then
// clamp(rescale(sum p v)). Sums of whole numbers do not depend on their order, so every split of the
// keys gives the same result, bit for bit.
#include <cuda_runtime.h>

#include <cstdint>

#include "hs_common.cuh"
#include "hs_draft.hpp"

namespace hs {

namespace {

// score() of crates/hardshell/src/gpt2/reference.rs:252: |dot| <= 1024 * 2^14 = 2^24, so the product
// fits in 64 bits.
__device__ __forceinline__ int64_t tree_score(int32_t dot, int32_t sm, int ss) {
    return clamp64(rescale64(dot, sm, (uint32_t)ss), -SCORE_LIMIT, SCORE_LIMIT);
}

// Whether a sequence record lies inside the call's bounds (the caller's are the host's).
__device__ __forceinline__ bool tree_seq_ok(const TreeSeq& s, uint32_t n_rows, uint32_t slots, uint32_t max_count,
                                            uint32_t max_keys) {
    return s.count <= max_count && s.first_row <= n_rows && s.count <= n_rows - s.first_row && s.slot < slots &&
           s.prefix <= max_keys && s.count <= max_keys - s.prefix;
}

constexpr int ANY_THREADS = 128;

// The kernel of every head width and alignment: one block per (row, head). Thread j takes the keys
// j, j + 128, ... for the dots and the weights (kept in shared memory), then a warp takes a channel at
// a time for the sum over the keys (V^T rows are contiguous).
__global__ void __launch_bounds__(ANY_THREADS) k_tree_attention_any(const TreeArgs a, int* err) {
    extern __shared__ __align__(16) uint32_t s_any[];  // [max_keys] dots, then e, then p; then q
    __shared__ int64_t red[ANY_THREADS / 32];
    const int hd = a.cache.hd, n_ctx = a.cache.n_ctx;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t seq_i = blockIdx.x / a.max_count;
    const int node = blockIdx.x % a.max_count, h = blockIdx.y;
    const TreeSeq s = a.seqs[seq_i];
    if (!tree_seq_ok(s, a.n_rows, a.cache.slots, a.max_count, a.max_keys)) {
        if (threadIdx.x == 0) atomicCAS(err, 0, ERR_DRAFT_SEQ);
        return;
    }
    if (node >= (int)s.count) return;
    const size_t row = (size_t)s.first_row + node;
    int8_t* sq = reinterpret_cast<int8_t*>(s_any + a.max_keys);
    const int8_t* q = a.q + row * a.q_stride + (size_t)h * hd;
    for (int i = threadIdx.x; i < hd; i += ANY_THREADS) sq[i] = q[i];
    const size_t plane = a.plane0 + h / (a.n_head / a.n_kv);
    const int8_t* K = a.cache.k + s.slot * a.cache.slot_stride + plane * ((size_t)n_ctx * hd);
    const int8_t* V = a.cache.v + s.slot * a.cache.slot_stride + plane * ((size_t)n_ctx * hd);
    const uint32_t* mask = a.mask + row * a.mask_words;
    const int n = (int)(s.prefix + s.count);
    auto seen = [&](int j) {
        const int t = j - (int)s.prefix;
        return t < 0 || ((mask[t >> 5] >> (t & 31)) & 1) != 0;
    };
    __syncthreads();
    int64_t mx = INT64_MIN;
    for (int j = threadIdx.x; j < n; j += ANY_THREADS) {
        if (!seen(j)) continue;
        int32_t dot = 0;
        const int8_t* kr = K + (size_t)j * hd;
        for (int i = 0; i < hd; i++) dot += (int32_t)sq[i] * (int32_t)kr[i];
        s_any[j] = (uint32_t)dot;
        const int64_t y = tree_score(dot, a.rule.sm, a.rule.ss);
        mx = y > mx ? y : mx;
    }
    for (int o = 16; o > 0; o >>= 1) {
        const int64_t w = __shfl_xor_sync(0xffffffffu, mx, o);
        mx = w > mx ? w : mx;
    }
    if (lane == 0) red[warp] = mx;
    __syncthreads();
    for (int w = 0; w < ANY_THREADS / 32; w++) mx = red[w] > mx ? red[w] : mx;
    __syncthreads();
    uint64_t sum = 0;
    for (int j = threadIdx.x; j < n; j += ANY_THREADS) {
        uint32_t e = 0;
        if (seen(j)) {
            const int64_t d = mx - tree_score((int32_t)s_any[j], a.rule.sm, a.rule.ss);
            e = (uint32_t)a.rule.table[d < a.rule.tlen - 1 ? d : a.rule.tlen - 1];
        }
        s_any[j] = e;
        sum += e;
    }
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) red[warp] = (int64_t)sum;
    __syncthreads();
    sum = 0;
    for (int w = 0; w < ANY_THREADS / 32; w++) sum += (uint64_t)red[w];
    if (sum == 0) sum = 1;
    for (int j = threadIdx.x; j < n; j += ANY_THREADS)
        s_any[j] = (uint32_t)(((uint64_t)s_any[j] << a.rule.P) / sum);
    __syncthreads();
    for (int c = warp; c < hd; c += ANY_THREADS / 32) {
        const int8_t* vr = V + (size_t)c * n_ctx;
        int64_t acc = 0;
        for (int j = lane; j < n; j += 32) acc += (int64_t)s_any[j] * (int64_t)vr[j];
        for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
        if (lane == 0)
            a.out[row * a.out_stride + (size_t)h * hd + c] =
                (int8_t)rescale_clamp127(acc, a.rule.om, a.rule.os, (double)a.rule.om * exp2_neg(a.rule.os));
    }
}

}  // namespace

cudaError_t launch_tree_attention(const TreeArgs& a, int num_sms, int* err, cudaStream_t st) {
    (void)num_sms;
    if (a.n_seq == 0 || a.max_count == 0) return cudaSuccess;
    const size_t smem = 4 * (size_t)a.max_keys + (size_t)a.cache.hd;
    const dim3 grid(a.n_seq * (uint32_t)a.max_count, (uint32_t)a.n_head);
    k_tree_attention_any<<<grid, ANY_THREADS, smem, st>>>(a, err);
    return cudaGetLastError();
}

cudaError_t configure_draft_kernels() {
    return cudaFuncSetAttribute((const void*)k_tree_attention_any, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                4 * MAX_ATTN_CTX + 1024);
}

}  // namespace hs
