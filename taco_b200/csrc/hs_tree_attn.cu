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

// ---- head widths 64 and 128, 16-byte aligned caches: int8 matrix instructions ----
//
// The unit of work is an item: 16 query rows (nodes, times the query heads of a kv head) of one tree and
// kv head. A cluster of C thread blocks of 8 warps takes an item; its keys are cut into slices of 8 NT
// keys, one for each warp, dealt round-robin to the blocks. A warp holds its 16 x 8 NT scores, then
// weights, then probabilities in registers from the first product to the second:
//   S = Q K^T (mma m16n8k32, s8 x s8), the row maxima over the cluster, e and the row sums over the
//   cluster, p = floor(e 2^P / sum) by an exact multiply-shift, p cut into four unsigned bytes, O += P V
//   (u8 x s8) for each byte plane, the planes joined in 64 bits, O summed over warps and blocks.
// Whole-number sums in any order: the split changes nothing.
//
// Operands come straight from global memory in the layout of the fragments. The order of the channels in
// a dot product is free, so thread t of a quad takes bytes 16 t .. 16 t + 15 of a key's row (and of the
// query's) as its fragment words: one 16-byte load per key. The order of the keys in O is free as long
// as P and V agree: column c of key tile i is key (c / 2) 2 NT + 2 i + c % 2 of the slice, so that the
// accumulators of thread t hold its 2 NT consecutive keys, which are the bytes of V^T rows it loads.

constexpr int TW = 8;              // warps of a block
constexpr int TTHREADS = 32 * TW;
constexpr int CH = 16;             // channels of O at a time
constexpr int PSTRIDE = CH + 2;    // 64-bit words of a row of the warps' O (padded against bank conflicts)

__device__ __forceinline__ void mma_s8s8(int32_t (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_u8s8(int32_t (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

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

// What the rows of an item share: per row the maximum's score, then the multiplier and shift of p.
struct RowState {
    int64_t top;
    uint32_t mh, ml;
    int shift;
};

struct TreeSmem {
    int32_t wmax[TW][16];
    uint64_t wsum[TW][16];
    int32_t bmax[16];   // of this block
    uint64_t bsum[16];
    RowState row[16];
    int64_t part[2][TW][16][PSTRIDE];  // O of each warp, 16 channels, two buffers
};

template <int HD>
constexpr size_t tree_smem() {
    return 4 * ATTN_TABLE_MAX + sizeof(TreeSmem) + 8 * 16 * HD;
}

template <int HD, int NT, bool NARROW, bool SSHI>
__global__ void __launch_bounds__(TTHREADS, 2) k_tree_attention(const __grid_constant__ TreeArgs a, int tiles, int items,
                                                                int* err) {
    constexpr int S = 8 * NT;        // keys of a warp
    constexpr int TK = 2 * NT;       // keys of a thread
    constexpr int KB = HD / 64;      // 16-byte pieces of a key's row per thread
    extern __shared__ __align__(16) uint8_t s_tree[];
    int32_t* sT = reinterpret_cast<int32_t*>(s_tree);
    TreeSmem& sm = *reinterpret_cast<TreeSmem*>(s_tree + 4 * ATTN_TABLE_MAX);
    int64_t* sO = reinterpret_cast<int64_t*>(s_tree + 4 * ATTN_TABLE_MAX + sizeof(TreeSmem));  // [16][HD] (clusters)
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t = lane & 3;
    const int32_t m = a.rule.sm;
    const int ss = a.rule.ss, last = a.rule.tlen - 1, G = a.n_head / a.n_kv;
    const int64_t half = ss >= 1 && ss <= 62 ? 1LL << (ss - 1) : 0;  // the narrow rule
    const double omsc = (double)a.rule.om * exp2_neg(a.rule.os);
    for (int i = tid; i < (a.rule.tlen + 3) / 4; i += TTHREADS)
        reinterpret_cast<int4*>(sT)[i] = reinterpret_cast<const int4*>(a.rule.table)[i];
    __syncthreads();

    for (int item = blockIdx.x / C; item < items; item += gridDim.x / C) {
        const int tile = item % tiles, kv = (item / tiles) % a.n_kv;
        const TreeSeq s = a.seqs[item / tiles / a.n_kv];
        if (!tree_seq_ok(s, a.n_rows, a.cache.slots, a.max_count, a.max_keys)) {
            if (tid == 0) atomicCAS(err, 0, ERR_DRAFT_SEQ);
            continue;
        }
        const int rows = (int)s.count * G - 16 * tile;  // rows of the item (the last tile has fewer)
        if (rows <= 0) continue;
        const int prefix = (int)s.prefix, n = prefix + (int)s.count;
        const int slices = (n + S - 1) / S;
        const int live = (slices - rank + C - 1) / C;  // this block's warps with keys
        const int k0 = (w * C + rank) * S;
        const bool on = w < live;
        const size_t plane = (size_t)s.slot * a.cache.slot_stride +
                             (size_t)(a.plane0 + kv) * ((size_t)a.cache.n_ctx * HD);
        const int8_t* K = a.cache.k + plane;
        const int8_t* V = a.cache.v + plane;
        int32_t c[NT][4];
        uint32_t seen[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
        bool whole = true;
        if (on) {
            // V of this warp's keys on its way into L2 while the scores are made.
            for (int ch = lane; ch < HD; ch += 32)
                asm volatile("prefetch.global.L2 [%0];" ::"l"(V + (size_t)ch * a.cache.n_ctx + k0));
            uint32_t q[2 * KB][4];
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int x = g + 8 * r;
                const size_t at = (size_t)s.first_row + (16 * tile + x) / G;
                const int head = kv * G + (16 * tile + x) % G;
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
#pragma unroll
            for (int i = 0; i < NT; i++) {
                c[i][0] = c[i][1] = c[i][2] = c[i][3] = 0;
                const int key = kcol + 2 * i;
                const uint4* p = reinterpret_cast<const uint4*>(K + (size_t)key * HD) + t;
#pragma unroll
                for (int b = 0; b < KB; b++) {
                    const uint4 v = key < n ? __ldg(p + 4 * b) : make_uint4(0, 0, 0, 0);
                    mma_s8s8(c[i], q[2 * b], v.x, v.y);
                    mma_s8s8(c[i], q[2 * b + 1], v.z, v.w);
                }
            }
            // Slices inside the context are whole for every row.
            if (k0 + S > prefix) {
                whole = false;
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const int x = g + 8 * r;
                    const size_t at = (size_t)s.first_row + (16 * tile + x) / G;
                    seen[r] = x < rows ? seen_word(a.mask + at * a.mask_words, k0 + t * TK, prefix, (int)s.count) : 0;
                }
            }
        }
        // The row extremes of the dots: score() rises with the dot, or falls if the multiplier is negative.
        const int32_t none = m >= 0 ? INT32_MIN : INT32_MAX;
        int32_t ext[2] = {none, none};
        if (on) {
            auto scan = [&](auto better) {
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
            if (m >= 0) scan([](int32_t x, int32_t y) { return max(x, y); });
            else scan([](int32_t x, int32_t y) { return min(x, y); });
            if (t == 0) {
                sm.wmax[w][g] = ext[0];
                sm.wmax[w][g + 8] = ext[1];
            }
        }
        __syncthreads();
        if (tid < 16) {
            int32_t e = none;
            for (int i = 0; i < live; i++) e = m >= 0 ? max(e, sm.wmax[i][tid]) : min(e, sm.wmax[i][tid]);
            sm.bmax[tid] = e;
        }
        if (C > 1) cl.sync();
        if (tid < 16) {
            int32_t e = sm.bmax[tid];
            for (int i = 0; i < C; i++) {
                const int32_t o = *cl.map_shared_rank(&sm.bmax[tid], i);
                e = m >= 0 ? max(e, o) : min(e, o);
            }
            sm.row[tid].top = e == none ? 0 : NARROW ? ((int64_t)e * m + half) >> ss : tree_score(e, m, ss);
        }
        __syncthreads();
        // The weights and their sums.
        if (on) {
            const int64_t top[2] = {sm.row[g].top, sm.row[g + 8].top};
            uint64_t sum[2] = {0, 0};
            auto weigh = [&](auto all) {
#pragma unroll
                for (int i = 0; i < NT; i++) {
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        int32_t d;
                        if constexpr (NARROW) {
                            const int64_t p = (int64_t)c[i][x] * (int64_t)m + half;
                            int32_t y;
                            if constexpr (SSHI) y = (int32_t)(p >> 32) >> (ss - 32);
                            else y = (int32_t)__funnelshift_r((uint32_t)p, (uint32_t)((uint64_t)p >> 32), ss);
                            d = (int32_t)top[x >> 1] - y;
                            d = (uint32_t)d < (uint32_t)last ? d : last;
                        } else {
                            const int64_t dd = top[x >> 1] - tree_score(c[i][x], m, ss);
                            d = (int32_t)((uint64_t)dd < (uint64_t)last ? dd : (int64_t)last);
                        }
                        uint32_t e = (uint32_t)sT[d];
                        if constexpr (!decltype(all)::value)
                            if (((seen[x >> 1] >> (2 * i + (x & 1))) & 1) == 0) e = 0;
                        c[i][x] = (int32_t)e;
                        sum[x >> 1] += e;
                    }
                }
            };
            if (whole) weigh(std::true_type{});
            else weigh(std::false_type{});
#pragma unroll
            for (int o = 1; o <= 2; o <<= 1)
#pragma unroll
                for (int r = 0; r < 2; r++) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], o);
            if (t == 0) {
                sm.wsum[w][g] = sum[0];
                sm.wsum[w][g + 8] = sum[1];
            }
        }
        __syncthreads();
        if (tid < 16) {
            uint64_t v = 0;
            for (int i = 0; i < live; i++) v += sm.wsum[i][tid];
            sm.bsum[tid] = v;
        }
        if (C > 1) cl.sync();
        if (tid < 16) {
            uint64_t v = 0;
            for (int i = 0; i < C; i++) v += *cl.map_shared_rank(&sm.bsum[tid], i);
            if (v == 0) v = 1;
            int l = 64 - __clzll((long long)(v - 1));  // v <= 2^l
            if (l < 1) l = 1;
            const uint64_t mg = ceil_pow2_div(31 + a.rule.P + l, v);
            sm.row[tid].mh = (uint32_t)(mg >> 32);
            sm.row[tid].ml = (uint32_t)mg;
            sm.row[tid].shift = l - 1;
        }
        __syncthreads();
        // The probabilities as byte planes, in the fragments of the second product: c[4 s + plane]
        // becomes the four A words of plane `plane` for the 32 keys of step s.
        if (on) {
            const RowState r0 = sm.row[g], r1 = sm.row[g + 8];
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
                            const RowState& z = r ? r1 : r0;
                            const uint64_t u = (uint64_t)e * z.mh + __umulhi(e, z.ml);
                            p[k] = (uint32_t)(u >> z.shift);
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
        // O, 16 channels at a time: each warp its keys' part, then the sum over the warps.
        const int orow = tid / CH, och = tid % CH;
#pragma unroll 1
        for (int ch0 = 0; ch0 < HD; ch0 += CH) {
            int64_t(*part)[16][PSTRIDE] = sm.part[(ch0 / CH) & 1];
            if (on) {
#pragma unroll
                for (int j = 0; j < CH / 8; j++) {
                    // The bytes of this thread's keys in the row of channel ch0 + 8 j + g.
                    uint32_t v[TK / 4];
                    const int8_t* vr = V + (size_t)(ch0 + 8 * j + g) * a.cache.n_ctx;
                    const int kt = k0 + t * TK;
                    if constexpr (TK >= 16) {
#pragma unroll
                        for (int b = 0; b < TK / 16; b++) {
                            const uint4 x = kt + 16 * b < n ? __ldg(reinterpret_cast<const uint4*>(vr + kt) + b)
                                                            : make_uint4(0, 0, 0, 0);
                            v[4 * b] = x.x;
                            v[4 * b + 1] = x.y;
                            v[4 * b + 2] = x.z;
                            v[4 * b + 3] = x.w;
                        }
                    } else {
                        const uint2 x = kt < n ? __ldg(reinterpret_cast<const uint2*>(vr + kt)) : make_uint2(0, 0);
                        v[0] = x.x;
                        v[1] = x.y;
                    }
                    int32_t o[4][4] = {};
#pragma unroll
                    for (int st = 0; st < NT / 4; st++)
#pragma unroll
                        for (int pl = 0; pl < 4; pl++) {
                            const uint32_t A[4] = {(uint32_t)c[4 * st + pl][0], (uint32_t)c[4 * st + pl][1],
                                                   (uint32_t)c[4 * st + pl][2], (uint32_t)c[4 * st + pl][3]};
                            mma_u8s8(o[pl], A, v[2 * st], v[2 * st + 1]);
                        }
                    // A plane's sum is at most S * 255 * 128 < 2^22 in magnitude.
#pragma unroll
                    for (int x = 0; x < 4; x++)
                        part[w][g + 8 * (x >> 1)][8 * j + 2 * t + (x & 1)] =
                            (int64_t)(o[2][x] + o[3][x] * 256) * 65536 + (o[0][x] + o[1][x] * 256);
                }
            }
            __syncthreads();
            int64_t acc = 0;
            for (int i = 0; i < live; i++) acc += part[i][orow][och];
            if (C > 1) {
                sO[orow * HD + ch0 + och] = acc;
            } else if (orow < rows) {
                const size_t at = (size_t)s.first_row + (16 * tile + orow) / G;
                a.out[at * a.out_stride + (size_t)(kv * G + (16 * tile + orow) % G) * HD + ch0 + och] =
                    (int8_t)rescale_clamp127(acc, a.rule.om, a.rule.os, omsc);
            }
        }
        if (C > 1) {
            cl.sync();
            for (int i = rank * TTHREADS + tid; i < 16 * HD; i += C * TTHREADS) {
                int64_t acc = 0;
                for (int b = 0; b < C; b++) acc += *cl.map_shared_rank(&sO[i], b);
                const int r = i / HD;
                if (r < rows) {
                    const size_t at = (size_t)s.first_row + (16 * tile + r) / G;
                    a.out[at * a.out_stride + (size_t)(kv * G + (16 * tile + r) % G) * HD + i % HD] =
                        (int8_t)rescale_clamp127(acc, a.rule.om, a.rule.os, omsc);
                }
            }
        }
    }
    if (C > 1) cl.sync();  // no block leaves while another reads its memory
}

template <int HD, int NT, bool NARROW, bool SSHI>
cudaError_t launch_tree_mma(const TreeArgs& a, int C, int num_sms, int* err, cudaStream_t st) {
    const int G = a.n_head / a.n_kv, tiles = (a.max_count * G + 15) / 16;
    const int items = (int)a.n_seq * a.n_kv * tiles;
    cudaLaunchConfig_t cfg{};
    const int clusters = 2 * num_sms / C;
    cfg.gridDim = dim3((unsigned)(items < clusters ? items : clusters) * C);
    cfg.blockDim = dim3(TTHREADS);
    cfg.dynamicSmemBytes = tree_smem<HD>();
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = C;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_tree_attention<HD, NT, NARROW, SSHI>, a, tiles, items, err);
}

template <int HD, int NT>
cudaError_t launch_tree_rule(const TreeArgs& a, int C, int num_sms, int* err, cudaStream_t st) {
    // Narrow: every |score| is below 2^30, so distances fit in 32 bits and no score reaches the clamp.
    const int ss = a.rule.ss;
    const uint64_t m = (uint64_t)(a.rule.sm < 0 ? -(int64_t)a.rule.sm : (int64_t)a.rule.sm);
    const bool narrow = ss >= 1 && ss <= 62 && ((m * ((uint64_t)HD << 14)) >> ss) + 1 < (1ull << 30);
    if (narrow && ss >= 32) return launch_tree_mma<HD, NT, true, true>(a, C, num_sms, err, st);
    if (narrow) return launch_tree_mma<HD, NT, true, false>(a, C, num_sms, err, st);
    return launch_tree_mma<HD, NT, false, false>(a, C, num_sms, err, st);
}

template <int HD>
cudaError_t launch_tree_width(const TreeArgs& a, int num_sms, int* err, cudaStream_t st) {
    int C = 1;
    while (C * TW * 128 < a.max_keys) C *= 2;
    return launch_tree_rule<HD, 16>(a, C, num_sms, err, st);
}

template <int HD>
cudaError_t configure_tree() {
    const void* fns[3] = {(const void*)k_tree_attention<HD, 16, true, true>,
                          (const void*)k_tree_attention<HD, 16, true, false>,
                          (const void*)k_tree_attention<HD, 16, false, false>};
    for (const void* f : fns) {
        const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)tree_smem<HD>());
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace

cudaError_t launch_tree_attention(const TreeArgs& a, int num_sms, int* err, cudaStream_t st) {
    if (a.n_seq == 0 || a.max_count == 0) return cudaSuccess;
    const bool vec = a.cache.vec && reinterpret_cast<uintptr_t>(a.q) % 16 == 0 && a.q_stride % 16 == 0 &&
                     a.rule.tlen <= ATTN_TABLE_MAX;
    if (vec && a.cache.hd == 64) return launch_tree_width<64>(a, num_sms, err, st);
    if (vec && a.cache.hd == 128) return launch_tree_width<128>(a, num_sms, err, st);
    const size_t smem = 4 * (size_t)a.max_keys + (size_t)a.cache.hd;
    const dim3 grid(a.n_seq * (uint32_t)a.max_count, (uint32_t)a.n_head);
    k_tree_attention_any<<<grid, ANY_THREADS, smem, st>>>(a, err);
    return cudaGetLastError();
}

cudaError_t configure_draft_kernels() {
    cudaError_t e = configure_tree<64>();
    if (e == cudaSuccess) e = configure_tree<128>();
    if (e == cudaSuccess) e = configure_beam();
    if (e != cudaSuccess) return e;
    return cudaFuncSetAttribute((const void*)k_tree_attention_any, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                4 * MAX_ATTN_CTX + 1024);
}

}  // namespace hs
