// Attention of trees of drafted tokens over the KV cache (hs_op_tree_attention, hs_batch_run_tree).
//
// A tree's nodes are query rows; node j's keys and values are in cache row prefix + j of its slot.
// A row attends to the slot's context (cache rows 0 .. prefix - 1) and to the nodes in its mask. The
// softmax is HardShell's (crates/hardshell/src/softmax.rs:78-104): the exact row maximum before any
// weight and the exact row sum before any probability, p = floor(e 2^P / sum), then
// clamp(rescale(sum p v)). Sums of whole numbers do not depend on their order, so every split of the
// keys gives the same result, bit for bit.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <type_traits>

#include "hs_common.cuh"
#include "hs_draft.hpp"

namespace cg = cooperative_groups;

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
// a time for the sum over the keys (V^T rows are contiguous). Each row reads its keys again (from L2) and
// multiplies byte by byte: it is bounded by that, not by HBM (64 trees of 16 nodes at 1,024 keys, 12 heads of 80:
// 610 us, where 64-wide heads take 51).
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

// ---- head widths 64 and 128, 16-byte aligned caches: int8 matrix instructions ----
//
// The unit of work is an item: 16 query rows (nodes, times the query heads of a kv head) of one tree and
// kv head. A cluster of C thread blocks of 8 warps takes an item; its keys are cut into slices of 8 NT
// keys, one for each warp, dealt round-robin to the blocks. A warp holds its 16 x 8 NT scores, then
// weights, then probabilities in registers from the first product to the second:
//   S = Q K^T (mma m16n8k32, s8 x s8), the row maxima over the cluster, e and the row sums over the
//   cluster, p = floor(e 2^P / sum) by an exact multiply-shift, p cut into four unsigned bytes, O += P V
//   (u8 x s8) for each byte plane, the planes joined in 64 bits, O summed over warps and blocks.
// Whole-number sums in any order: the split changes nothing. O is summed over a block's warps by additions in
// shared memory (one word a lane and bank; parts of each warp, added up behind two more barriers, took 466 us
// where this took 405), and over a cluster's blocks when it is written, while the next item is under way.
//
// Bound: not HBM (23 % of it at 64 trees of 16 nodes and 1,024 keys, 51 us), nor the issue of the integer work of a
// score (about 25 instructions from the product to the probability's planes, one of them a table look-up in shared
// memory at random banks; two thirds of the issue slots are empty) but the latencies of an item, which its warps meet
// at three times and two items an SM do not hide. 16 warps an SM are what 64 scores a
// thread leave room for; 32 warps of 64 registers took 785 us where 16 of 128 took 560.
//
// Operands come straight from global memory in the layout of the fragments. The order of the channels in
// a dot product is free, so thread t of a quad takes bytes 16 t .. 16 t + 15 of a key's row (and of the
// query's) as its fragment words: one 16-byte load per key. The order of the keys in O is free as long
// as P and V agree: column c of key tile i is key (c / 2) 2 NT + 2 i + c % 2 of the slice, so that the
// accumulators of thread t hold its 2 NT consecutive keys, which are the bytes of V^T rows it loads.

constexpr int TMAXC = 8;           // blocks of a cluster

__device__ __forceinline__ void mma_s8s8(int32_t (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The first product of a sum: C is 0.
__device__ __forceinline__ void mma_s8s8_first(int32_t (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ void mma_u8s8_first(int32_t (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ void mma_u8s8(int32_t (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ceil_pow2_div (hs_common.cuh) without a 64-bit division. The residual R = 2^sh - x s of the first estimate
// x is at most 2^11 s in magnitude, so the double quotient R / s is within 2^-40 of the exact one, and with
// its whole part taken off |R| is at most s + 12 (s < 2^44). Up to two unit steps then make x the least
// value with x s >= 2^sh, which has -s < R <= 0.
__device__ __forceinline__ uint64_t ceil_pow2_div_near(int sh, uint64_t s) {
    const double inv = 1.0 / (double)s;
    uint64_t x = (uint64_t)(inv * pow2_double(sh));
    int64_t R = (int64_t)((1ull << (sh & 63)) * (sh < 64 ? 1ull : 0ull) - x * s);  // mod 2^64: |R| < 2^63
    const int64_t d = (int64_t)((double)R * inv);
    x += (uint64_t)d;
    R -= d * (int64_t)s;
    if (R > 0) {
        x += 1;
        R -= (int64_t)s;
    }
    if (R > 0) x += 1;
    if (R <= -(int64_t)s) x -= 1;
    return x;
}

// The node and the head of row x of a tree and kv head with G query heads (a division only if they are shared).
__device__ __forceinline__ int node_of(int x, int G) { return G == 1 ? x : x / G; }
__device__ __forceinline__ int head_of(int x, int G) { return G == 1 ? 0 : x % G; }

// The bits of the keys first .. first + 31 that a row sees: the context (below `prefix`) and the tree's
// nodes in the mask words (bits from `count` on are none).
__device__ __forceinline__ uint32_t seen_word(const uint32_t* mask, int first, int prefix, int count) {
    const int t = first - prefix;  // the node of bit 0
    if (t <= -32) return 0xFFFFFFFFu;
    auto word = [&](int w) -> uint32_t {
        const int left = count - 32 * w;
        if (w < 0 || left <= 0) return 0;
        return left >= 32 ? mask[w] : mask[w] & ((1u << left) - 1u);
    };
    if (t < 0) return (word(0) << -t) | ((1u << -t) - 1u);
    return __funnelshift_r(word(t >> 5), word((t >> 5) + 1), t & 31);
}

// clamp(rescale(256 x + y, om, os), -127, 127) for |y| <= 2^28, in single precision where `fast`: os <= 95 and
// |om 2^-os| <= 2^-19. The estimate z of the value plus 1/2 takes the two parts, their sum, the factor and
// the product with a rounding each: an error of at most 2^-22 |z| + 32 |om 2^-os|, below 2^-13 for |z| <
// 256. Values nearer than that to a whole number take the exact rule.
__device__ __forceinline__ int32_t output_of(int2 o, int32_t om, int os, float fsc, double omsc, bool fast) {
    const float z = fmaf(fmaf((float)o.x, 256.0f, (float)o.y), fsc, 0.5f);
    const float fl = floorf(z), fr = z - fl;
    if (fast) {
        if (fabsf(z) >= 256.0f) return z > 0 ? 127 : -127;
        if (fr > 1.220703125e-4f && fr < 1.0f - 1.220703125e-4f) return min(max((int32_t)fl, -127), 127);
    }
    return rescale_clamp127((int64_t)o.x * 256 + o.y, om, os, omsc);
}

// The row extremes of a warp's dots, for rows g and g + 8 of lane (g, t): score() rises with the dot, or falls
// if the multiplier is negative. No key seen: INT32_MIN, or INT32_MAX.
template <int NT>
__device__ __forceinline__ void tree_extremes(const int32_t (&c)[NT][4], bool whole, const uint32_t (&seen)[2], int32_t m,
                                              int32_t (&ext)[2]) {
    auto scan = [&](auto better, int32_t none) {
        ext[0] = ext[1] = none;
        if (whole) {
#pragma unroll
            for (int i = 0; i < NT; i++) {
                ext[0] = better(ext[0], better(c[i][0], c[i][1]));
                ext[1] = better(ext[1], better(c[i][2], c[i][3]));
            }
        } else {
#pragma unroll
            for (int i = 0; i < NT; i++)
#pragma unroll
                for (int x = 0; x < 4; x++)
                    if ((seen[x >> 1] >> (2 * i + (x & 1))) & 1) ext[x >> 1] = better(ext[x >> 1], c[i][x]);
        }
#pragma unroll
        for (int o = 1; o <= 2; o <<= 1)
#pragma unroll
            for (int r = 0; r < 2; r++) ext[r] = better(ext[r], __shfl_xor_sync(0xffffffffu, ext[r], o));
    };
    if (m >= 0) scan([](int32_t x, int32_t y) { return max(x, y); }, INT32_MIN);
    else scan([](int32_t x, int32_t y) { return min(x, y); }, INT32_MAX);
}

// The dots become weights e = table[min(M - score, last)] (0 for keys not seen), summed over the quad's keys.
// ext: the extremes of the whole rows (lane l has row l % 16). The narrow rules take the distance in one
// multiply-add: M - floor((dot m + h) / 2^ss) = floor((M 2^ss + 2^ss - 1 - h - dot m) / 2^ss). With M the score of
// the dot x and h = 2^(ss - 1), M 2^ss + 2^ss - 1 - h lies in x m .. x m + 2^ss - 1, and |x m|, |dot m| are below 2^52
// (heads of at most 128): the sum is below 2^53 + 2^ss < 2^63 in magnitude for the shifts up to 62 of these rules. A
// distance is never negative for a key that is seen, and the unsigned minimum keeps the index inside the table for
// the others.
template <int NT, bool NARROW, bool SSHI>
__device__ __forceinline__ void tree_weigh(int32_t (&c)[NT][4], bool whole, const uint32_t (&seen)[2], int32_t ext,
                                           int32_t m, int ss, const int32_t* table, int last, uint64_t (&sum)[2]) {
    const int g = (threadIdx.x & 31) >> 2;
    const bool none = ext == (m >= 0 ? INT32_MIN : INT32_MAX);
    int64_t mine;
    if constexpr (NARROW) {
        const int64_t half = 1LL << (ss - 1), top = none ? 0 : ((int64_t)ext * m + half) >> ss;
        mine = top * (1LL << ss) + ((1LL << ss) - 1 - half);
    } else {
        mine = none ? 0 : tree_score(ext, m, ss);
    }
    const int64_t top[2] = {__shfl_sync(0xffffffffu, mine, g), __shfl_sync(0xffffffffu, mine, g + 8)};
    sum[0] = sum[1] = 0;
    auto weigh = [&](auto all) {
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int x = 0; x < 4; x++) {
                uint32_t d;
                if constexpr (NARROW) {
                    const int64_t p = (int64_t)c[i][x] * (int64_t)(-m) + top[x >> 1];
                    int32_t y;
                    if constexpr (SSHI) y = (int32_t)(p >> 32) >> (ss - 32);
                    else y = (int32_t)__funnelshift_r((uint32_t)p, (uint32_t)((uint64_t)p >> 32), ss);
                    d = min((uint32_t)y, (uint32_t)last);
                } else {
                    const int64_t dd = top[x >> 1] - tree_score(c[i][x], m, ss);
                    d = (uint64_t)dd < (uint64_t)last ? (uint32_t)dd : (uint32_t)last;
                }
                uint32_t e = (uint32_t)table[d];
                if constexpr (!decltype(all)::value)
                    if (((seen[x >> 1] >> (2 * i + (x & 1))) & 1) == 0) e = 0;
                c[i][x] = (int32_t)e;
                // (weights are below 2^31: two fit in 32 bits)
                if (x & 1) sum[x >> 1] = add_wide(sum[x >> 1], (uint32_t)c[i][x - 1] + e);
            }
    };
    if (whole) weigh(std::true_type{});
    else weigh(std::false_type{});
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1)
#pragma unroll
        for (int r = 0; r < 2; r++) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], o);
}

// The weights become probabilities p = floor(e 2^P / z) (an exact multiply-shift), as byte planes in the
// fragments of the second product: c[4 s + plane] the four A words of plane `plane` for the 32 keys of step s.
// z: the sums of the whole rows (lane l has row l % 16).
template <int NT>
__device__ __forceinline__ void tree_planes(int32_t (&c)[NT][4], uint64_t z, int P) {
    const int g = (threadIdx.x & 31) >> 2;
    if (z == 0) z = 1;
    int l = 64 - __clzll((long long)(z - 1));  // z <= 2^l
    if (l < 1) l = 1;
    const uint64_t mg = ceil_pow2_div_near(31 + P + l, z);
    uint32_t mh[2], ml[2];
    int shift[2];
#pragma unroll
    for (int r = 0; r < 2; r++) {
        mh[r] = __shfl_sync(0xffffffffu, (uint32_t)(mg >> 32), g + 8 * r);
        ml[r] = __shfl_sync(0xffffffffu, (uint32_t)mg, g + 8 * r);
        shift[r] = __shfl_sync(0xffffffffu, l - 1, g + 8 * r);
    }
#pragma unroll
    for (int i = 0; i < NT; i += 4) {
        uint32_t pl[4][4];
#pragma unroll
        for (int r = 0; r < 2; r++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint32_t p[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t e = (uint32_t)c[i + 2 * h + (k >> 1)][2 * r + (k & 1)];
                    const uint64_t u = (uint64_t)e * mh[r] + __umulhi(e, ml[r]);
                    p[k] = (uint32_t)(u >> shift[r]);
                }
                const uint32_t x0 = __byte_perm(p[0], p[1], 0x5140), x1 = __byte_perm(p[0], p[1], 0x7362);
                const uint32_t y0 = __byte_perm(p[2], p[3], 0x5140), y1 = __byte_perm(p[2], p[3], 0x7362);
                pl[0][2 * h + r] = __byte_perm(x0, y0, 0x5410);
                pl[1][2 * h + r] = __byte_perm(x0, y0, 0x7632);
                pl[2][2 * h + r] = __byte_perm(x1, y1, 0x5410);
                pl[3][2 * h + r] = __byte_perm(x1, y1, 0x7632);
            }
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int x = 0; x < 4; x++) c[i + k][x] = (int32_t)pl[k][x];
    }
}

// O of 8 channels and this warp's keys: the planes times the values v (this thread's keys of channel g), joined
// to sum (p >> 8) v and sum (p & 255) v: x.x, x.y of channel 2 t and x.z, x.w of 2 t + 1, rows g and g + 8.
template <int NT>
__device__ __forceinline__ void tree_multiply(const int32_t (&c)[NT][4], const uint32_t (&v)[NT / 2], int4 (&x)[2]) {
    int32_t o[4][4];
#pragma unroll
    for (int st = 0; st < NT / 4; st++)
#pragma unroll
        for (int pl = 0; pl < 4; pl++) {
            const uint32_t A[4] = {(uint32_t)c[4 * st + pl][0], (uint32_t)c[4 * st + pl][1], (uint32_t)c[4 * st + pl][2],
                                   (uint32_t)c[4 * st + pl][3]};
            if (st == 0) mma_u8s8_first(o[pl], A, v[0], v[1]);
            else mma_u8s8(o[pl], A, v[2 * st], v[2 * st + 1]);
        }
#pragma unroll
    for (int r = 0; r < 2; r++) {
        x[r].x = o[1][2 * r] + (o[2][2 * r] + o[3][2 * r] * 256) * 256;
        x[r].y = o[0][2 * r];
        x[r].z = o[1][2 * r + 1] + (o[2][2 * r + 1] + o[3][2 * r + 1] * 256) * 256;
        x[r].w = o[0][2 * r + 1];
    }
}

// O of a tile and 16 HD channels in shared memory: two whole numbers a row and channel, sum (p >> 8) v and
// sum (p & 255) v. With sum p <= 2^30 and |v| <= 128 the first is at most 2^29 in magnitude over all keys, the
// second at most 8192 * 2^15 = 2^28. The word of lane l's number x (of tree_multiply) for row g + 8 r and the 8
// channels j: each of a warp's additions takes all the banks, and so do the reads of the 16 quads of a row.
__device__ __forceinline__ int o_at(int j, int r, int x, int l) { return ((j * 2 + r) * 4 + x) * 32 + ((l + 4 * j) & 31); }

__device__ __forceinline__ void o_add(int32_t* o, int j, const int4 (&x)[2]) {
    const int l = threadIdx.x & 31;
#pragma unroll
    for (int r = 0; r < 2; r++) {
        atomicAdd(o + o_at(j, r, 0, l), x[r].x);
        atomicAdd(o + o_at(j, r, 1, l), x[r].y);
        atomicAdd(o + o_at(j, r, 2, l), x[r].z);
        atomicAdd(o + o_at(j, r, 3, l), x[r].w);
    }
}

// The numbers of four channels, 4 quad .. 4 quad + 3, of a row.
__device__ __forceinline__ void o_get(const int32_t* o, int row, int quad, int2 (&y)[4]) {
    const int l = 4 * (row & 7) + 2 * (quad & 1);
    int2 c[4];
#pragma unroll
    for (int x = 0; x < 4; x++) c[x] = *reinterpret_cast<const int2*>(o + o_at(quad >> 1, row >> 3, x, l));
    y[0] = make_int2(c[0].x, c[1].x);
    y[1] = make_int2(c[2].x, c[3].x);
    y[2] = make_int2(c[0].y, c[1].y);
    y[3] = make_int2(c[2].y, c[3].y);
}
__device__ __forceinline__ void o_clear(int32_t* o, int row, int quad) {
#pragma unroll
    for (int x = 0; x < 4; x++)
        *reinterpret_cast<int2*>(o + o_at(quad >> 1, row >> 3, x, 4 * (row & 7) + 2 * (quad & 1))) = make_int2(0, 0);
}

// The tile whose O waits to be written: the tree's first row, the kv head, the tile's first row and its rows.
struct Pending {
    uint32_t first_row;
    int kv, x0, rows;
};

// The outputs of four channels of a row, in one store where they are aligned.
__device__ __forceinline__ void tree_put(const TreeArgs& a, const Pending& p, int G, int row, int hd, int quad,
                                         const int2 (&o)[4], float fsc, double omsc, bool fast) {
    const int x = p.x0 + row;
    int8_t* to = a.out + ((size_t)p.first_row + node_of(x, G)) * a.out_stride +
                 (size_t)(p.kv * G + head_of(x, G)) * hd + 4 * quad;
    uint32_t y[4], word = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        y[i] = (uint32_t)output_of(o[i], a.rule.om, a.rule.os, fsc, omsc, fast) & 0xFFu;
        word |= y[i] << (8 * i);
    }
    if (reinterpret_cast<uintptr_t>(to) % 4 == 0) {
        *reinterpret_cast<uint32_t*>(to) = word;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) to[i] = (int8_t)y[i];
    }
}

// Shared memory of W warps in clusters of C blocks: O of this item and the last [2][16 HD][2] i32, then by slice
// of the item the row sums [W C][16] u64 and maxima [W C][16] i32 (each block of a cluster has all of them), the
// exponent table up to its last change.
constexpr size_t tree_smem(int W, int HD, int C, int reach) {
    return 16 * (size_t)16 * HD + (size_t)W * C * 16 * 12 + 4 * (((size_t)reach + 3) & ~(size_t)3);
}

template <int HD, int TW, int NT, bool NARROW, bool SSHI>
__global__ void __launch_bounds__(32 * TW, 2) k_tree_attention(const __grid_constant__ TreeArgs a, int tiles, int items,
                                                               int* err) {
    constexpr int TTHREADS = 32 * TW, QUADS = HD / 4;
    constexpr int S = 8 * NT;        // keys of a warp
    constexpr int TK = 2 * NT;       // keys of a thread
    constexpr int KB = HD / 64;      // 16-byte pieces of a key's row per thread
    constexpr int VB = TK / 4;       // words of a channel's values per thread
    extern __shared__ __align__(16) uint8_t s_tree[];
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    int32_t(*o)[32 * HD] = reinterpret_cast<int32_t(*)[32 * HD]>(s_tree);
    uint64_t(*wsum)[16] = reinterpret_cast<uint64_t(*)[16]>(o + 2);
    int32_t(*wmax)[16] = reinterpret_cast<int32_t(*)[16]>(wsum + TW * C);
    int32_t* sT = reinterpret_cast<int32_t*>(wmax + TW * C);
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t = lane & 3;
    const int32_t m = a.rule.sm;
    const int ss = a.rule.ss, last = a.rule.reach - 1, G = a.n_head / a.n_kv;
    const double omsc = (double)a.rule.om * exp2_neg(a.rule.os);
    const float fsc = (float)omsc;
    const bool fast = a.rule.os <= 95 && fabs(omsc) <= 1.9073486328125e-6;
    for (int i = tid; i < (a.rule.reach + 3) / 4; i += TTHREADS)
        reinterpret_cast<int4*>(sT)[i] = reinterpret_cast<const int4*>(a.rule.table)[i];
    for (int i = tid; i < 2 * 32 * HD; i += TTHREADS) o[0][i] = 0;
    auto meet = [&]() {  // of all the item's warps
        if (C > 1) cl.sync();
        else __syncthreads();
    };
    // No block of the cluster writes to another before that one runs.
    meet();
    // O of the last item out: the cluster's sum, each block some rows.
    Pending last_item{0, 0, 0, 0};
    uint32_t count = 0;  // of the items so far: item i adds to o[i & 1]
    auto put = [&]() {
        for (int i = rank * TTHREADS + tid; i < 16 * QUADS; i += C * TTHREADS) {
            const int row = i / QUADS, quad = i % QUADS;
            if (row >= last_item.rows) break;
            int2 y[4];
            o_get(o[~count & 1], row, quad, y);
            for (int b = 1; b < C; b++) {
                int2 z[4];
                o_get(cl.map_shared_rank(o[~count & 1], (rank + b) % C), row, quad, z);
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    y[x].x += z[x].x;
                    y[x].y += z[x].y;
                }
            }
            tree_put(a, last_item, G, row, HD, quad, y, fsc, omsc, fast);
        }
    };

    // The keys and values of an item's slice of this warp, on their way into L2.
    auto ask = [&](const TreeSeq& s, int kv, int tile, bool keys) {
        const int n = (int)(s.prefix + s.count), k0 = (w * C + rank) * S;
        if (!tree_seq_ok(s, a.n_rows, a.cache.slots, a.max_count, a.max_keys) || k0 >= n || 16 * tile >= (int)s.count * G)
            return;
        const size_t plane = (size_t)s.slot * a.cache.slot_stride +
                             (size_t)(a.plane0 + kv) * ((size_t)a.cache.n_ctx * HD);
        if (keys) {
            const int8_t* K = a.cache.k + plane + (size_t)k0 * HD;
            for (int x = lane * 128; x < min(S, n - k0) * HD; x += 32 * 128)
                asm volatile("prefetch.global.L2 [%0];" ::"l"(K + x));
        }
        const int8_t* V = a.cache.v + plane + k0;
        for (int ch = lane; ch < HD; ch += 32)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(V + (size_t)ch * a.cache.n_ctx));
    };
    const int stride = gridDim.x / C;
    auto seq_of = [&](int item) { return a.seqs[min(item, items - 1) / tiles / a.n_kv]; };
    TreeSeq next = seq_of(blockIdx.x / C);
    ask(next, (int)(blockIdx.x / C) / tiles % a.n_kv, (int)(blockIdx.x / C) % tiles, false);

    for (int item = blockIdx.x / C; item < items; item += stride) {
        const int tile = item % tiles, kv = (item / tiles) % a.n_kv;
        const TreeSeq s = next;
        next = seq_of(item + stride);
        if (!tree_seq_ok(s, a.n_rows, a.cache.slots, a.max_count, a.max_keys)) {
            if (tid == 0) atomicCAS(err, 0, ERR_DRAFT_SEQ);
            continue;
        }
        const int rows = (int)s.count * G - 16 * tile;  // rows of the item (the last tile has fewer)
        if (rows <= 0) continue;
        const int prefix = (int)s.prefix, n = prefix + (int)s.count;
        const int slices = (n + S - 1) / S;
        const int live = (slices - rank + C - 1) / C;  // this block's warps with keys
        const int slice = w * C + rank, k0 = slice * S;
        const bool on = w < live;
        const size_t plane = (size_t)s.slot * a.cache.slot_stride +
                             (size_t)(a.plane0 + kv) * ((size_t)a.cache.n_ctx * HD);
        const int8_t* K = a.cache.k + plane;
        const int8_t* V = a.cache.v + plane;
        int32_t c[NT][4];
        uint32_t seen[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
        bool whole = true;
        if (on) {
            uint32_t q[2 * KB][4];
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int x = g + 8 * r;
                const size_t at = (size_t)s.first_row + node_of(16 * tile + x, G);
                const int head = kv * G + head_of(16 * tile + x, G);
                const uint4* p = reinterpret_cast<const uint4*>(a.q + at * a.q_stride + (size_t)head * HD) + t;
#pragma unroll
                for (int b = 0; b < KB; b++) {
                    const uint4 v = x < rows ? p[4 * b] : make_uint4(0, 0, 0, 0);
                    q[2 * b][r] = v.x;
                    q[2 * b][2 + r] = v.y;
                    q[2 * b + 1][r] = v.z;
                    q[2 * b + 1][2 + r] = v.w;
                }
            }
            const int kcol = k0 + (g >> 1) * TK + (g & 1);
            const uint4* kp = reinterpret_cast<const uint4*>(K + (size_t)kcol * HD) + t;
            constexpr int DEEP = KB == 1 ? NT : NT < 8 ? NT : 8;  // tiles in flight
            const int rest = n - kcol;
#pragma unroll
            for (int i0 = 0; i0 < NT; i0 += DEEP) {
                uint4 kw[DEEP][KB];
                // Keys past the last row of the context are not read (their weights are 0 by the mask).
                if (k0 + S <= n) {
#pragma unroll
                    for (int i = 0; i < DEEP; i++)
#pragma unroll
                        for (int b = 0; b < KB; b++) kw[i][b] = __ldg(kp + 2 * (i0 + i) * (HD / 16) + 4 * b);
                } else {
#pragma unroll
                    for (int i = 0; i < DEEP; i++)
#pragma unroll
                        for (int b = 0; b < KB; b++) {
                            kw[i][b] = make_uint4(0, 0, 0, 0);
                            if (2 * (i0 + i) < rest) kw[i][b] = __ldg(kp + 2 * (i0 + i) * (HD / 16) + 4 * b);
                        }
                }
#pragma unroll
                for (int i = 0; i < DEEP; i++) {
                    mma_s8s8_first(c[i0 + i], q[0], kw[i][0].x, kw[i][0].y);
                    mma_s8s8(c[i0 + i], q[1], kw[i][0].z, kw[i][0].w);
#pragma unroll
                    for (int b = 1; b < KB; b++) {
                        mma_s8s8(c[i0 + i], q[2 * b], kw[i][b].x, kw[i][b].y);
                        mma_s8s8(c[i0 + i], q[2 * b + 1], kw[i][b].z, kw[i][b].w);
                    }
                }
            }
            // Slices inside the context are whole for every row.
            if (k0 + S > prefix) {
                whole = false;
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const int x = g + 8 * r;
                    const size_t at = (size_t)s.first_row + node_of(16 * tile + x, G);
                    seen[r] = x < rows ? seen_word(a.mask + at * a.mask_words, k0 + t * TK, prefix, (int)s.count) : 0;
                }
            }
            int32_t ext[2];
            tree_extremes<NT>(c, whole, seen, m, ext);
            // Lane t of a quad gives it to the blocks t, t + 4.
            for (int b = t; b < C; b += 4) {
                int32_t* to = C > 1 ? cl.map_shared_rank(&wmax[slice][0], b) : wmax[slice];
                to[g] = ext[0];
                to[g + 8] = ext[1];
            }
        }
        meet();
        if (item + stride < items) ask(next, (item + stride) / tiles % a.n_kv, (item + stride) % tiles, true);
        // Every block has read O of the item before the last, whose place this item takes.
        for (int i = tid; i < 16 * QUADS; i += TTHREADS) o_clear(o[count & 1], i / QUADS, i % QUADS);
        if (on) {
            // Lane l has row l % 16.
            int32_t e = m >= 0 ? INT32_MIN : INT32_MAX;
            for (int i = 0; i < slices; i++) e = m >= 0 ? max(e, wmax[i][lane & 15]) : min(e, wmax[i][lane & 15]);
            uint64_t sum[2];
            tree_weigh<NT, NARROW, SSHI>(c, whole, seen, e, m, ss, sT, last, sum);
            for (int b = t; b < C; b += 4) {
                uint64_t* to = C > 1 ? cl.map_shared_rank(&wsum[slice][0], b) : wsum[slice];
                to[g] = sum[0];
                to[g + 8] = sum[1];
            }
        }
        meet();
        // The words of this thread's keys in the row of a channel.
        const int kt = k0 + t * TK;
        const bool inside = k0 + S <= a.cache.n_ctx;
        auto load_v = [&](int ch, uint32_t (&v)[VB]) {
            const int8_t* vr = V + (size_t)(ch + g) * a.cache.n_ctx + kt;
            if constexpr (TK >= 16) {
#pragma unroll
                for (int b = 0; b < TK / 16; b++) {
                    // (past n the probabilities are 0: any bytes of the row do)
                    uint4 x = make_uint4(0, 0, 0, 0);
                    if (inside || kt + 16 * b < a.cache.n_ctx) x = __ldg(reinterpret_cast<const uint4*>(vr) + b);
                    v[4 * b] = x.x;
                    v[4 * b + 1] = x.y;
                    v[4 * b + 2] = x.z;
                    v[4 * b + 3] = x.w;
                }
            } else {
                uint2 x = make_uint2(0, 0);
                if (inside || kt < a.cache.n_ctx) x = __ldg(reinterpret_cast<const uint2*>(vr));
                v[0] = x.x;
                v[1] = x.y;
            }
        };
        uint32_t v[2][VB];
        if (on) {
            load_v(0, v[0]);
            uint64_t z = 0;
            for (int i = 0; i < slices; i++) z += wsum[i][lane & 15];
            tree_planes<NT>(c, z, a.rule.P);
        }
        if (on) {
#pragma unroll
            for (int j = 0; j < HD / 8; j++) {
                // The next 8 channels' values while these are multiplied.
                if (j + 1 < HD / 8) load_v(8 * j + 8, v[(j + 1) & 1]);
                int4 x[2];
                tree_multiply<NT>(c, v[j & 1], x);
                o_add(o[count & 1], j, x);
            }
        }
        put();  // (all have added to the last item's O since this item's first meeting)
        last_item = Pending{s.first_row, kv, 16 * tile, min(rows, 16)};
        count++;
    }
    meet();
    put();
    if (C > 1) cl.sync();  // no block leaves while another reads its memory
}

// The clusters of C blocks of a kernel that the current device holds at once.
int max_clusters(const void* kernel, int C, int threads, size_t smem) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)C);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)C;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) cudaGetLastError();
    return n;
}

// Which score rule fits: 0 wide; 1 narrow: every |score| is below 2^30, so distances fit in 32 bits and no
// score reaches the clamp; 2 narrow with a shift of at least 32.
int score_rule(const AttnRuleView& r, int hd) {
    const uint64_t m = (uint64_t)(r.sm < 0 ? -(int64_t)r.sm : (int64_t)r.sm);
    const bool narrow = r.ss >= 1 && r.ss <= 62 && r.sm != INT32_MIN && ((m * ((uint64_t)hd << 14)) >> r.ss) + 1 < (1ull << 30);
    return narrow ? r.ss >= 32 ? 2 : 1 : 0;
}

// A kernel's shape, and by log2 C the clusters that a device holds at once (found when a device is opened; the
// GPUs of a host are alike).
template <int HD, int TW, int NT>
struct TreeShape {
    static constexpr int KEYS = TW * NT * 8;  // of a block
    static inline std::atomic<int> fit[4];  // (host threads open their devices at once)

    static cudaError_t configure() {
        const void* fns[3] = {(const void*)k_tree_attention<HD, TW, NT, true, true>,
                              (const void*)k_tree_attention<HD, TW, NT, true, false>,
                              (const void*)k_tree_attention<HD, TW, NT, false, false>};
        for (const void* f : fns) {
            const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                       (int)tree_smem(TW, HD, TMAXC, ATTN_TABLE_MAX));
            if (e != cudaSuccess) return e;
        }
        for (int lg = 0; lg < 4; lg++) {
            int n = 1 << 30;
            for (const void* f : fns)
                n = std::min(n, max_clusters(f, 1 << lg, 32 * TW, tree_smem(TW, HD, 1 << lg, 6144)));
            fit[lg] = n;
        }
        return cudaSuccess;
    }

    template <bool NARROW, bool SSHI>
    static cudaError_t go(const TreeArgs& a, int* err, cudaStream_t st) {
        const int G = a.n_head / a.n_kv, tiles = (a.max_count * G + 15) / 16;
        const int items = (int)a.n_seq * a.n_kv * tiles;
        int lg = 0;
        while (KEYS << lg < a.max_keys) lg++;
        const int C = 1 << lg, found = fit[lg], clusters = found > 0 ? found : 1;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)((items < clusters ? items : clusters) * C));
        cfg.blockDim = dim3(32 * TW);
        cfg.dynamicSmemBytes = tree_smem(TW, HD, C, a.rule.reach);
        cfg.stream = st;
        cudaLaunchAttribute at;
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = C;
        at.val.clusterDim.y = at.val.clusterDim.z = 1;
        cfg.attrs = &at;
        cfg.numAttrs = 1;
        return cudaLaunchKernelEx(&cfg, k_tree_attention<HD, TW, NT, NARROW, SSHI>, a, tiles, items, err);
    }

    static cudaError_t launch(const TreeArgs& a, int* err, cudaStream_t st) {
        const int rule = score_rule(a.rule, HD);
        if (rule == 2) return go<true, true>(a, err, st);
        if (rule == 1) return go<true, false>(a, err, st);
        return go<false, false>(a, err, st);
    }
};

// ---- head width 64: keys and values by bulk copies ----
//
// The mathematics and the fragments of the kernel above, with the operands ahead of the work: bulk copies
// bring the keys (up to 1,024 rows) and the transposed values of a tree's kv head into shared memory. The
// last warp that has made its scores of a head asks for the next head's keys, the last that has multiplied
// asks for its values; no warp waits to copy. One block per SM, 16 warps in two groups of 8 that take the
// 16-row tiles of the head in turn, 128 keys a warp. The groups meet only within themselves, so one multiplies
// while the other weighs. At 256 trees of 64 nodes and 1,024 keys, 12 heads, 415 us: an SM issues 1.35
// instructions a cycle (34 %), the tensor pipe is busy 20 %, the integer pipes 21 and 25 %; the warps wait for
// one another's rows (25 %), for the next instruction's operands (20 %) and for first rows and masks (16 %).
// The exponent table is held up to its last change (table_reach).

constexpr int BK = 1024;                 // keys of a block
constexpr int BWARPS = 16, GROUPS = 2;
constexpr int BTHREADS = 32 * BWARPS;
constexpr int VROW = BK + 16;            // bytes of a channel's values (padded: two rows in a quarter warp's banks)

struct __align__(16) TreeBulk {
    uint8_t k[BK * 64];
    uint8_t v[64 * VROW];
    uint64_t k_full, v_full;
    uint32_t k_done, v_done;             // warps that need this head's keys (values) no more
    uint32_t k_asked, v_asked;           // copies asked for so far
    uint32_t gave_up;                    // the code of a wait of this block that ran out
};
// Behind it: the groups' O [GROUPS][16 * 64][2] i32, the warps' wsum [BWARPS][16] u64 and wmax [BWARPS][16] i32,
// and the table.
constexpr size_t bulk_smem(int reach) {
    return sizeof(TreeBulk) + 8 * (size_t)GROUPS * 16 * 64 + (size_t)BWARPS * 16 * 12 + 4 * (((size_t)reach + 3) & ~(size_t)3);
}
constexpr size_t BLOCK_SMEM = 227 * 1024;
static_assert(bulk_smem(ATTN_TABLE_MAX) <= BLOCK_SMEM, "room for every table");

// A wait for a block's copy, of at most `polls` tries. It ends early only after another wait of the block ran out
// (gave_up is then not 0; null: it does not): the error word may hold a refused record, of this call or of an
// earlier one, which is no reason to read keys that have not arrived.
__device__ __forceinline__ bool copy_wait(uint64_t* bar, uint32_t phase, const uint32_t* gave_up, uint32_t polls) {
    for (uint32_t i = 0; i < polls; i++) {
        if (mbar_try_wait(bar, phase)) return true;
        if (i > 64) __nanosleep(32);
        if (gave_up && *(const volatile uint32_t*)gave_up) break;
    }
    return false;
}

// A wait that gives up notes its code and lets its thread go on: every barrier still gets its arrivals, every later
// wait returns at once, no further copy is asked for, and the call's results count for nothing. The block then sets
// the error word and waits (again with a limit) for the copies under way before it ends.
template <bool NARROW, bool SSHI>
__global__ void __launch_bounds__(BTHREADS, 1) k_tree_attention_bulk(const __grid_constant__ TreeArgs a, int works,
                                                                     int* err) {
    constexpr int HD = 64, WPG = BWARPS / GROUPS, NT = BK / WPG / 8, S = 8 * NT, TK = 2 * NT, VB = TK / 4;
    constexpr int GTHREADS = 32 * WPG;
    static_assert(GTHREADS == 16 * HD / 4, "a thread of a group for each four channels of a tile's row");
    extern __shared__ __align__(128) uint8_t s_bulk[];
    TreeBulk& sm = *reinterpret_cast<TreeBulk*>(s_bulk);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int grp = warp / WPG, w = warp % WPG, gtid = tid - grp * GTHREADS, g = lane >> 2, t = lane & 3;
    const int G = a.n_head / a.n_kv, first = blockIdx.x, stride = gridDim.x;
    int32_t(*os)[32 * HD] = reinterpret_cast<int32_t(*)[32 * HD]>(&sm + 1);
    uint64_t(*wsums)[16] = reinterpret_cast<uint64_t(*)[16]>(os + GROUPS);
    int32_t(*wmaxs)[16] = reinterpret_cast<int32_t(*)[16]>(wsums + BWARPS);
    int32_t* table = reinterpret_cast<int32_t*>(wmaxs + BWARPS);
    int32_t* o = os[grp];
    uint64_t(*wsum)[16] = wsums + grp * WPG;
    int32_t(*wmax)[16] = wmaxs + grp * WPG;
    const int32_t m = a.rule.sm;
    const int ss = a.rule.ss, last = a.rule.reach - 1;
    const double omsc = (double)a.rule.om * exp2_neg(a.rule.os);
    const float fsc = (float)omsc;
    const bool fast = a.rule.os <= 95 && fabs(omsc) <= 1.9073486328125e-6;
    if (tid == 0) {
        mbar_init(&sm.k_full, 1);
        mbar_init(&sm.v_full, 1);
        sm.k_done = sm.v_done = sm.k_asked = sm.v_asked = sm.gave_up = 0;
        fence_barrier_init();
    }
    for (int i = tid; i < (a.rule.reach + 3) / 4; i += BTHREADS)
        reinterpret_cast<int4*>(table)[i] = reinterpret_cast<const int4*>(a.rule.table)[i];
    for (int i = gtid; i < 32 * HD; i += GTHREADS) o[i] = 0;
    __syncthreads();

    // The copies of the keys (values) of the first work from `work` on that has rows, by one warp.
    auto copy = [&](int work, bool values) {
        if (__shfl_sync(0xffffffffu, *(volatile uint32_t*)&sm.gave_up, 0)) return;  // (one answer for the warp)
        for (; work < works; work += stride) {
            const TreeSeq s = a.seqs[work / a.n_kv];
            if (!tree_seq_ok(s, a.n_rows, a.cache.slots, a.max_count, a.max_keys) || s.count == 0) continue;
            const int n = (int)(s.prefix + s.count);
            const size_t plane = (size_t)s.slot * a.cache.slot_stride +
                                 (size_t)(a.plane0 + work % a.n_kv) * ((size_t)a.cache.n_ctx * HD);
            if (values) {
                const uint32_t bytes = (uint32_t)(n + 15) & ~15u;  // (n_ctx % 16 == 0)
                if (lane == 0) {
                    sm.v_asked++;
                    mbar_arrive_expect_tx(&sm.v_full, bytes * HD);
                }
                __syncwarp();
                for (int ch = lane; ch < HD; ch += 32)
                    bulk_load(sm.v + ch * VROW, a.cache.v + plane + (size_t)ch * a.cache.n_ctx, bytes, &sm.v_full);
            } else if (lane == 0) {
                sm.k_asked++;
                mbar_arrive_expect_tx(&sm.k_full, (uint32_t)n * HD);
                bulk_load(sm.k, a.cache.k + plane, (uint32_t)n * HD, &sm.k_full);
            }
            break;
        }
    };
    if (warp == 0) copy(first, false);
    if (warp == 1) copy(first, true);
    auto wait = [&](uint64_t* bar, uint32_t phase, uint32_t code) {
        if (!copy_wait(bar, phase, &sm.gave_up, 1u << 26)) *(volatile uint32_t*)&sm.gave_up = code;
    };
    // This warp has read the keys (values) of `work`: the last one asks for the next.
    auto done = [&](int work, bool values) {
        __syncwarp();
        uint32_t before = 0;
        if (lane == 0) {
            __threadfence_block();
            before = atomicAdd(values ? &sm.v_done : &sm.k_done, 1u);
            if (before == BWARPS - 1) *(volatile uint32_t*)(values ? &sm.v_done : &sm.k_done) = 0;
        }
        if (__shfl_sync(0xffffffffu, before, 0) == BWARPS - 1) {
            __threadfence_block();
            fence_async_smem();  // the warps' reads before the copies' writes
            copy(work + stride, values);
        }
        __syncwarp();
    };
    auto group_bar = [&]() {
        __syncwarp();
        named_bar(1 + grp, GTHREADS);
    };
    // O of the group's last tile out, between two meetings: every warp has added to it, none adds yet.
    Pending last_tile{0, 0, 0, 0};
    auto put = [&]() {
        const int row = gtid / (HD / 4), quad = gtid % (HD / 4);
        int2 y[4];
        o_get(o, row, quad, y);
        o_clear(o, row, quad);
        if (row < last_tile.rows) tree_put(a, last_tile, G, row, HD, quad, y, fsc, omsc, fast);
    };
    uint32_t count = 0;
    for (int work = first; work < works; work += stride) {
        const TreeSeq s = a.seqs[work / a.n_kv];
        if (!tree_seq_ok(s, a.n_rows, a.cache.slots, a.max_count, a.max_keys)) {
            if (tid == 0) atomicCAS(err, 0, ERR_DRAFT_SEQ);
            continue;
        }
        if (s.count == 0) continue;
        const int kv = work % a.n_kv, prefix = (int)s.prefix, n = prefix + (int)s.count;
        const int total = (int)s.count * G, tiles = (total + 15) / 16, slices = (n + S - 1) / S;
        const bool on = w < slices;
        const int k0 = w * S;
        const uint32_t phase = count & 1;
        count++;
        const uint8_t* ks = sm.k + (size_t)k0 * HD;
        const uint8_t* vs = sm.v + k0 + t * TK;
        // The rows of a tile: their fragments and what they see of this thread's keys (slices inside the
        // context are whole for every row), loaded a tile ahead.
        const bool whole = k0 + S <= prefix;
        const int node0 = k0 + t * TK - prefix;  // the node of this thread's first key
        uint32_t q[2][4], words[2][2] = {};
        auto load_rows = [&](int tile) {
            if (!on) return;
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int x = 16 * tile + g + 8 * r;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (x < total)
                    v = reinterpret_cast<const uint4*>(a.q + ((size_t)s.first_row + node_of(x, G)) * a.q_stride +
                                                       (size_t)(kv * G + head_of(x, G)) * HD)[t];
                q[0][r] = v.x;
                q[0][2 + r] = v.y;
                q[1][r] = v.z;
                q[1][2 + r] = v.w;
                if (!whole) {
                    // The mask words that hold the nodes k0 + t TK - prefix .. + 31 (put together at the tile).
                    const uint32_t* of = a.mask + ((size_t)s.first_row + node_of(x, G)) * a.mask_words;
                    words[r][0] = words[r][1] = 0;
                    if (x < total && node0 > -32) {
                        if (node0 >= 0 && node0 < (int)s.count) words[r][0] = of[node0 >> 5];
                        const int up = node0 < 0 ? 0 : (node0 >> 5) + 1;
                        if (32 * up < (int)s.count) words[r][1] = of[up];
                    }
                }
            }
        };
        load_rows(grp);
        for (int tile = grp; tile < tiles; tile += GROUPS) {
            const int rows = total - 16 * tile;
            int32_t c[NT][4];
            uint32_t seen[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
            if (on && !whole) {
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    // Keys before node 0 are the context's; nodes from `count` on are none.
                    const uint32_t lo = node0 >= 0 ? words[r][0] : 0xFFFFFFFFu;
                    const uint32_t bits = __funnelshift_r(lo, words[r][1], node0 & 31);
                    const int left = (int)s.count - node0;
                    seen[r] = 16 * tile + g + 8 * r >= total || left <= 0 ? 0u
                              : node0 <= -32                              ? 0xFFFFFFFFu
                              : left >= 32                                ? bits
                                                                          : bits & ((1u << left) - 1u);
                }
            }
            if (tile == grp) wait(&sm.k_full, phase, 55);
            if (on) {
                const uint4* kp = reinterpret_cast<const uint4*>(ks + ((g >> 1) * TK + (g & 1)) * HD) + t;
#pragma unroll
                for (int i = 0; i < NT; i++) {
                    const uint4 kw = kp[2 * i * (HD / 16)];
                    mma_s8s8_first(c[i], q[0], kw.x, kw.y);
                    mma_s8s8(c[i], q[1], kw.z, kw.w);
                }
                int32_t ext[2];
                tree_extremes<NT>(c, whole, seen, m, ext);
                if (t == 0) {
                    wmax[w][g] = ext[0];
                    wmax[w][g + 8] = ext[1];
                }
            }
            if (tile + GROUPS >= tiles) done(work, false);  // the group's last scores of this head
            group_bar();
            put();
            if (on) {
                // Lane l has row l % 16.
                int32_t e = m >= 0 ? INT32_MIN : INT32_MAX;
                for (int i = 0; i < slices; i++) e = m >= 0 ? max(e, wmax[i][lane & 15]) : min(e, wmax[i][lane & 15]);
                uint64_t sum[2];
                tree_weigh<NT, NARROW, SSHI>(c, whole, seen, e, m, ss, table, last, sum);
                if (t == 0) {
                    wsum[w][g] = sum[0];
                    wsum[w][g + 8] = sum[1];
                }
            }
            group_bar();
            if (tile + GROUPS < tiles) load_rows(tile + GROUPS);
            if (on) {
                uint64_t z = 0;
                for (int i = 0; i < slices; i++) z += wsum[i][lane & 15];
                tree_planes<NT>(c, z, a.rule.P);
            }
            if (tile == grp) wait(&sm.v_full, phase, 56);
            if (on) {
#pragma unroll
                for (int j = 0; j < HD / 8; j++) {
                    uint32_t v[VB];
#pragma unroll
                    for (int b = 0; b < TK / 16; b++) {
                        const uint4 x = *reinterpret_cast<const uint4*>(vs + (8 * j + g) * VROW + 16 * b);
                        v[4 * b] = x.x;
                        v[4 * b + 1] = x.y;
                        v[4 * b + 2] = x.z;
                        v[4 * b + 3] = x.w;
                    }
                    int4 x[2];
                    tree_multiply<NT>(c, v, x);
                    o_add(o, j, x);
                }
            }
            if (tile + GROUPS >= tiles) done(work, true);  // the group's last product of this head
            last_tile = Pending{s.first_row, kv, 16 * tile, min(rows, 16)};
        }
        if (grp >= tiles) {
            // No tile for this group: the copies are not needed, but each is waited for, so that the counts are
            // this head's.
            wait(&sm.k_full, phase, 55);
            done(work, false);
            wait(&sm.v_full, phase, 56);
            done(work, true);
        }
    }
    group_bar();
    put();
    __syncthreads();
    if (tid == 0 && sm.gave_up) {
        atomicCAS(err, 0, (int)sm.gave_up);
        // (else every copy has been waited for; copy n completes phase n - 1 of its barrier)
        if (sm.k_asked) copy_wait(&sm.k_full, (sm.k_asked - 1) & 1, nullptr, 1u << 22);
        if (sm.v_asked) copy_wait(&sm.v_full, (sm.v_asked - 1) & 1, nullptr, 1u << 22);
    }
}

template <bool NARROW, bool SSHI>
cudaError_t launch_bulk(const TreeArgs& a, int num_sms, int* err, cudaStream_t st) {
    const int works = (int)a.n_seq * a.n_kv;
    k_tree_attention_bulk<NARROW, SSHI>
        <<<works < num_sms ? works : num_sms, BTHREADS, bulk_smem(a.rule.reach), st>>>(a, works, err);
    return cudaGetLastError();
}

cudaError_t configure_bulk() {
    for (const void* f : {(const void*)k_tree_attention_bulk<true, true>, (const void*)k_tree_attention_bulk<true, false>,
                          (const void*)k_tree_attention_bulk<false, false>}) {
        const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)BLOCK_SMEM);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

// Head width, warps, key tiles of a warp (times by repeated calls, 12 heads). A warp that holds few keys leaves a short context to more warps: 256 keys a
// block of 64-wide heads take 9.4 us (one tree of 8 at 200 keys, 12 heads) and 22.9 us (64 trees of 16 at 256),
// 1,024 a block 12.9 and 31.2 us. Above that the longer slices win: 64 trees of 16 at 1,024 keys 50 us, 89 us in
// clusters of four short blocks. Heads of 128, 512 or 1,024 keys a block: one tree of 8 at 512 keys 14.4 and 15.7
// us, 64 of 16 at 512 keys 47 and 60 us, at 1,024 keys 95 (two blocks) and 85 us.
using Short64 = TreeShape<64, 8, 4>;
using Long64 = TreeShape<64, 8, 16>;
using Short128 = TreeShape<128, 8, 8>;
using Long128 = TreeShape<128, 8, 16>;

}  // namespace

cudaError_t launch_tree_attention(const TreeArgs& a, int num_sms, int* err, cudaStream_t st) {
    if (a.n_seq == 0 || a.max_count == 0) return cudaSuccess;
    const bool vec = a.cache.vec && reinterpret_cast<uintptr_t>(a.q) % 16 == 0 && a.q_stride % 16 == 0 &&
                     a.rule.tlen <= ATTN_TABLE_MAX;
    if (vec && a.cache.hd == 64) {
        if (a.max_keys <= Short64::KEYS) return Short64::launch(a, err, st);
        // More than one tile a head, and K and V fit in a block: 64 trees of 31 nodes at 1,024 keys take 74 us, 84 by
        // the kernel without copies, 256 trees of 64 nodes 405 and 558 us. One tile reads K and V once anyway: 64
        // trees of 16 nodes 60 us with the copies, 50 without. (In clusters, for longer contexts, they lose: 8 trees
        // of 31 at 8,192 keys 138 us, 111 without.)
        if (a.max_keys <= BK && a.max_count * (a.n_head / a.n_kv) > 16) {
            const int rule = score_rule(a.rule, 64);
            return rule == 2   ? launch_bulk<true, true>(a, num_sms, err, st)
                   : rule == 1 ? launch_bulk<true, false>(a, num_sms, err, st)
                               : launch_bulk<false, false>(a, num_sms, err, st);
        }
        return Long64::launch(a, err, st);
    }
    if (vec && a.cache.hd == 128)
        return a.max_keys <= Short128::KEYS ? Short128::launch(a, err, st) : Long128::launch(a, err, st);
    const size_t smem = 4 * (size_t)a.max_keys + (size_t)a.cache.hd;
    const dim3 grid(a.n_seq * (uint32_t)a.max_count, (uint32_t)a.n_head);
    k_tree_attention_any<<<grid, ANY_THREADS, smem, st>>>(a, err);
    return cudaGetLastError();
}

cudaError_t configure_draft_kernels() {
    cudaError_t e = Short64::configure();
    if (e == cudaSuccess) e = Long64::configure();
    if (e == cudaSuccess) e = Short128::configure();
    if (e == cudaSuccess) e = Long128::configure();
    if (e == cudaSuccess) e = configure_bulk();
    if (e == cudaSuccess) e = configure_beam();
    if (e != cudaSuccess) return e;
    return cudaFuncSetAttribute((const void*)k_tree_attention_any, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                4 * MAX_ATTN_CTX + 1024);
}

}  // namespace hs
