// The selection of a beam search over beams and vocabulary (hs_op_beam_select, hs_batch_beam_step).
//
// A row of logits is read as the LM head leaves it: u16 distances from the tile maxima. A symbol's
// distance D from the row maximum is the whole number of table units that its log weight lies below
// the largest, so D is its cost up to the row's normaliser: cost = base + N + D with N = #{j :
// table[j] W > table[0]^2}, the least j at which table[j] / table[0] is not above table[0] / W.
// Candidates are ordered by cost, then beam, then symbol: id = beam << 16 | symbol.
//
// A cluster of blocks takes a group; its items are the rows' segments (1 to 8 a row), dealt round-robin
// to the blocks. A block reads a segment once, sums its weights and keeps the smallest distance of every 32
// symbols. Its threads form 64 sets, and the keep-th smallest of the sets' minima is a distance that at
// least `keep` symbols are not above: only symbols up to it are candidates (about `keep` of them, unless
// distances tie in great numbers; then a bisection finds the threshold). The groups of 32 symbols that hold
// one are read again (from L2), and each candidate finds its place by counting. The lists and sums go to
// the first block's shared memory, which adds the normalisers and merges the lists.
//
// The sums are one table look-up per symbol, in shared memory at random banks (about 5,500 cycles a row: 39 us of
// the 256 groups below; the rest is the barriers and phases of a row). The look-ups take 32 bits, floor(table[j] /
// 2^s), so the sum is known to lie in [L 2^s, L 2^s + vocab (2^s - 1)]. N does not decrease with W, so where both
// ends give one N it is exact; where they differ (W next to a border) the low bits are summed as well.
//
// Measured (vocabulary 50257, repeated calls): 256 groups of 8 beams 108 us, 30 % of HBM's rate (206 MB of
// distances); 64 groups 30 us from L2; one group of 4 beams 12 us, the latency of its six phases. With L2 flushed
// before each call 123 and 33 us. A group that holds a row next to a border ends 15 us later (64 groups with one
// such row 49 us): its first block alone reads that row again.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "hs_common.cuh"
#include "hs_draft.hpp"

namespace cg = cooperative_groups;

namespace hs {

namespace {

constexpr int BT = 256;          // threads of a block
constexpr int BW = BT / 32;
constexpr int BEAM_BLOCKS = 4;   // blocks of an SM (registers)
constexpr int BU = 4;            // vectors of 8 symbols that a thread has in flight, and of a kept minimum
constexpr int SETS = 64;         // sets of four threads
constexpr int HITS = 256;        // groups of 32 symbols to read again
constexpr int FOUND = 512;       // candidates of a segment up to the threshold
constexpr int MAX_ITEMS = 2 * MAX_BEAMS;
constexpr uint32_t NO_KEY = 0xFFFFFFFFu;
constexpr int64_t BASE_LIMIT = 1LL << 62;
static_assert(4 * SETS == BT && BW == 8 && MAX_KEEP <= SETS, "the reductions and the threshold");

struct BeamSmem {
    // Of the first block, written by the cluster: per item the list's length and the sum, per row the
    // maximum. The lists [items][keep] and the merge's places are behind this struct.
    uint64_t sum[MAX_ITEMS];
    int64_t top[MAX_BEAMS];
    uint32_t len[MAX_ITEMS];
    // Of the first block: the rows.
    int64_t row[MAX_BEAMS];       // base + N
    uint8_t state[MAX_BEAMS];     // 0 dead, 1 alive, 2 ended, 3 alive with a sum next to a border
    // The segment in work.
    uint32_t cut, hits, found, border;
    int64_t red[BW];
    uint64_t redu[BW];
    __align__(16) uint32_t set[SETS];
    uint32_t hit[HITS], key[FOUND];
    uint16_t off[MAX_CODER_VOCAB / 64];  // the tiles' distances from the row maximum, cut at the table
};

// The sizes of a launch.
struct BeamShape {
    int segs, seg_vecs, batches, cut_bits;
};

__device__ __forceinline__ int64_t warp_max8(int64_t v) {  // over lanes 0..7 (and their copies)
    for (int o = 4; o > 0; o >>= 1) {
        const int64_t x = __shfl_xor_sync(0xffffffffu, v, o);
        v = x > v ? x : v;
    }
    return v;
}

// The cluster barrier in two halves, each by all threads of all blocks. Nothing written before it is read behind
// it, so the arrival orders no memory.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait;" ::: "memory"); }

// VEC: rows of 16-byte vectors; else symbol by symbol. One cluster per group.
template <bool VEC>
__global__ void __launch_bounds__(BT, BEAM_BLOCKS) k_beam_select(const __grid_constant__ BeamArgs a,
                                                                 const __grid_constant__ BeamShape sh) {
    extern __shared__ __align__(16) uint8_t s_beam[];
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    // No block writes to the first one's shared memory before that one runs: all arrive here and wait behind
    // the loads below (the cluster's other meeting is the one before the merge).
    if (C > 1) cluster_arrive();
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    const int last = a.tlen - 1, tiles = (a.vocab + (1 << a.tsh) - 1) >> a.tsh;
    const uint32_t keep = (uint32_t)a.keep, no_symbol = (uint32_t)a.tlen;
    const int vecs = (a.vocab + 7) / 8, whole = VEC ? a.vocab / 8 : 0;  // vectors that are read whole
    const int items = a.beams * sh.segs;
    const size_t row0 = (size_t)(blockIdx.x / C) * a.beams;  // the group's first row
    uint32_t* sT = reinterpret_cast<uint32_t*>(s_beam);  // tlen weights / 2^cut_bits, then 0 for no symbol
    BeamSmem& sm = *reinterpret_cast<BeamSmem*>(s_beam + 16 * (((size_t)a.tlen + 4) / 4));
    uint32_t* s_list = reinterpret_cast<uint32_t*>(&sm + 1);        // [items][keep]
    uint32_t* s_place = s_list + items * a.keep;                    // [items][keep]
    uint16_t* s_near = reinterpret_cast<uint16_t*>(s_place + items * a.keep);  // [batches][BT]

    auto state_of = [&](int b) {
        const int64_t base = a.base[row0 + b];
        return base < 0 || base >= BASE_LIMIT ? 0 : a.finished && a.finished[row0 + b] ? 2 : 1;
    };
    auto lrow_of = [&](int b) { return a.row_of ? (size_t)a.row_of[row0 + b] : row0 + b; };
    // An item's first vectors and the thread's part of its row maximum, loaded ahead.
    uint4 raw[BU];
    int64_t part = INT64_MIN;
    int next_state = 0;
    auto load = [&](const uint16_t* dist, int v, int end) {
#pragma unroll
        for (int k = 0; k < BU; k++)
            if (v + k * BT < min(end, whole)) raw[k] = __ldg(reinterpret_cast<const uint4*>(dist) + v + k * BT);
    };
    auto ahead = [&](int item) {
        if (item >= items) return;
        const int b = item / sh.segs, v0 = item % sh.segs * sh.seg_vecs;
        next_state = state_of(b);
        if (next_state != 1) return;
        const size_t lrow = lrow_of(b);
        const uint16_t* dist = a.dist + lrow * a.dist_stride;
        const int end = min(min(v0 + sh.seg_vecs, vecs), whole);
        load(dist, v0 + tid, end);
        part = INT64_MIN;
        for (int t = tid; t < tiles; t += BT) {
            const int64_t x = a.tops[lrow * a.tops_stride + t];
            part = x > part ? x : part;
        }
    };
    ahead(rank);
    for (int i = tid; i <= a.tlen / 4; i += BT)
        reinterpret_cast<uint4*>(sT)[i] = __ldg(reinterpret_cast<const uint4*>(a.high) + i);
    if (C > 1) cluster_wait();

    for (int item = rank; item < items; item += C) {
        const int b = item / sh.segs, seg = item % sh.segs;
        if (next_state != 1) {
            // A dead beam has no candidates; one that has ended is a candidate itself.
            if (tid == 0) {
                const bool one = next_state == 2 && seg == 0;
                *cl.map_shared_rank(&sm.len[item], 0) = one ? 1 : 0;
                if (one) *cl.map_shared_rank(&s_list[item * keep], 0) = 0;
            }
            ahead(item + C);
            continue;
        }
        const size_t lrow = lrow_of(b);
        const uint16_t* dist = a.dist + lrow * a.dist_stride;
        const int64_t* tops = a.tops + lrow * a.tops_stride;
        const int v0 = seg * sh.seg_vecs, v1 = min(v0 + sh.seg_vecs, vecs);
        const bool fetch = VEC && tid == 0 && item + C < items && state_of((item + C) / sh.segs) == 1;
        for (int o = 16; o > 0; o >>= 1) {
            const int64_t x = __shfl_xor_sync(0xffffffffu, part, o);
            part = x > part ? x : part;
        }
        if (lane == 0) sm.red[w] = part;
        __syncthreads();  // (and the item before is done with the shared memory)
        const int64_t mx = warp_max8(sm.red[lane % BW]);
        // The offset as an unsigned difference: right for any maxima, and never below 0.
        for (int t = tid; t < tiles; t += BT) {
            const uint64_t o = (uint64_t)mx - (uint64_t)tops[t];
            sm.off[t] = (uint16_t)(o < (uint64_t)last ? o : (uint64_t)last);
        }
        if (tid == 0) {
            sm.hits = sm.found = 0;
            if (seg == 0) *cl.map_shared_rank(&sm.top[b], 0) = mx;
        }
        __syncthreads();
        // The next segment on its way into L2, if its beam has logits (those of the others may not be there).
        if (fetch) {
            const int f0 = (item + C) % sh.segs * sh.seg_vecs, f1 = min(f0 + sh.seg_vecs, whole);
            if (f1 > f0)
                asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(
                                 a.dist + lrow_of((item + C) / sh.segs) * a.dist_stride + 8 * (size_t)f0),
                             "r"(16 * (f1 - f0)));
        }
        uint64_t sum = 0;
        uint32_t nearest = no_symbol;
        // D = min(offset + distance, last) = offset + min(distance, last - offset), two symbols at a time:
        // no half carries into the other.
        auto add = [&](int v, uint4 d) -> uint32_t {
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
            for (int j = 0; j < 8; j++) sum = add_wide(sum, e[j]);  // (the adds of the distances keep the other pipe)
            return __vminu2(__vminu2(x[0], x[1]), __vminu2(x[2], x[3]));
        };
        auto far_of = [&](int s) -> uint32_t {
            const uint32_t o = sm.off[s >> a.tsh];
            return o + min((uint32_t)dist[s], (uint32_t)last - o);
        };
        for (int i = 0; i < sh.batches; i++) {
            const int v = v0 + tid + i * BU * BT;
            uint4 cur[BU];
#pragma unroll
            for (int k = 0; k < BU; k++) cur[k] = raw[k];
            if (i + 1 < sh.batches) load(dist, v + BU * BT, v1);
            else ahead(item + C);
            uint32_t m2 = no_symbol * 0x10001u;
#pragma unroll
            for (int k = 0; k < BU; k++)
                if (v + k * BT < min(v1, whole)) m2 = __vminu2(m2, add(v + k * BT, cur[k]));
            uint32_t m = min(m2 & 0xFFFFu, m2 >> 16);
            // The vectors that are not whole (the vocabulary's end), or not aligned.
            if (v + (BU - 1) * BT >= whole)
                for (int k = 0; k < BU; k++) {
                    const int x = v + k * BT;
                    if (x < whole || x >= v1) continue;
                    for (int s = 8 * x; s < 8 * x + 8 && s < a.vocab; s++) {
                        const uint32_t D = far_of(s);
                        sum += sT[D];
                        m = min(m, D);
                    }
                }
            s_near[i * BT + tid] = (uint16_t)m;
            nearest = min(nearest, m);
        }
        uint32_t least = min(nearest, __shfl_xor_sync(0xffffffffu, nearest, 1));
        least = min(least, __shfl_xor_sync(0xffffffffu, least, 2));
        if ((lane & 3) == 0) sm.set[tid >> 2] = least;
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) sm.redu[w] = sum;
        __syncthreads();
        {
            // The place of a minimum among the sets' (equal ones by their index): four threads a set.
            const int i = tid >> 2, o0 = (tid & 3) * (SETS / 4);
            const uint32_t me = sm.set[i];
            uint32_t at = 0;
#pragma unroll
            for (int k = 0; k < SETS / 4; k += 4) {
                const uint4 o = *reinterpret_cast<const uint4*>(&sm.set[o0 + k]);
                const int j = o0 + k;
                at += (o.x < me + (j < i)) + (o.y < me + (j + 1 < i)) + (o.z < me + (j + 2 < i)) + (o.w < me + (j + 3 < i));
            }
            at += __shfl_xor_sync(0xffffffffu, at, 1);
            at += __shfl_xor_sync(0xffffffffu, at, 2);
            if ((tid & 3) == 0 && at == keep - 1) sm.cut = me;
            if (w == BW - 1) {
                uint64_t all = sm.redu[lane % BW];
                for (int o = 4; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
                if (lane == 0) *cl.map_shared_rank(&sm.sum[item], 0) = all;
            }
        }
        __syncthreads();
        const uint32_t cut = min(sm.cut, (uint32_t)a.last_weight);
        // The groups of 32 symbols that hold a candidate, then a lane for each of their symbols.
        if (nearest <= cut)
            for (int i = 0; i < sh.batches; i++)
                if (s_near[i * BT + tid] <= cut) {
                    const uint32_t at = atomicAdd(&sm.hits, 1u);
                    if (at < HITS) sm.hit[at] = (uint32_t)(i * BT + tid);
                }
        auto open = [&](uint32_t hit, uint32_t upto, auto f) {
            const int v = v0 + (int)(hit / BT) * BU * BT + (lane >> 3) * BT + (int)(hit % BT), s = 8 * v + (lane & 7);
            if (v >= v1 || s >= a.vocab) return;
            const uint32_t key = far_of(s) << 16 | (uint32_t)s;
            if (key <= upto) f(key);
        };
        auto take = [&](uint32_t key) {
            const uint32_t at = atomicAdd(&sm.found, 1u);
            if (at < FOUND) sm.key[at] = key;
        };
        __syncthreads();
        if (sm.hits <= HITS) {
#pragma unroll 4
            for (uint32_t i = w; i < sm.hits; i += BW) open(sm.hit[i], cut << 16 | 0xFFFFu, take);
        }
        __syncthreads();
        if (sm.hits > HITS || sm.found > FOUND) {
            // Distances tie in great numbers: the least key that `keep` keys are not above, by bisection.
            auto each = [&](uint32_t upto, auto f) {
                for (int i = 32 * w; i < sh.batches * BT; i += BT) {
                    uint32_t any = __ballot_sync(0xffffffffu, s_near[i + lane] <= upto >> 16);
                    for (; any; any &= any - 1) open((uint32_t)(i + __ffs(any) - 1), upto, f);
                }
            };
            uint32_t lo = 0, hi = cut << 16 | 0xFFFFu;
            while (lo < hi) {
                const uint32_t mid = lo + (hi - lo) / 2;
                __syncthreads();
                if (tid == 0) sm.found = 0;
                __syncthreads();
                uint32_t n = 0;
                each(mid, [&](uint32_t) { n++; });
                n = __reduce_add_sync(0xffffffffu, n);
                if (lane == 0) atomicAdd(&sm.found, n);
                __syncthreads();
                if (sm.found >= keep) hi = mid;
                else lo = mid + 1;
            }
            __syncthreads();
            if (tid == 0) sm.found = 0;
            __syncthreads();
            each(lo, take);
            __syncthreads();
        }
        const uint32_t n = sm.found;
        for (uint32_t i = tid; i < n; i += BT) {
            const uint32_t key = sm.key[i];
            uint32_t at = 0;
            for (uint32_t k = 0; k < n; k++) at += sm.key[k] < key;
            if (at < keep) *cl.map_shared_rank(&s_list[item * keep + at], 0) = key;
        }
        if (tid == 0) *cl.map_shared_rank(&sm.len[item], 0) = n < keep ? n : keep;
    }
    cl.sync();
    if (rank != 0) return;

    // The first block: the normalisers, a warp for a row.
    const u128 one = (u128)a.first * a.first;
    auto norm_of = [&](uint64_t W, auto weight) {  // the entries weight(j) with weight(j) W > one
        int lo = 0, hi = a.tlen;  // the entries below lo pass, those from hi on do not
        while (lo < hi) {
            const int step = (hi - lo + 31) / 32, j = lo + step * lane;
            const int pass = __popc(__ballot_sync(0xffffffffu, j < hi && (u128)weight(j) * W > one));
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
    auto sum_of = [&](int b) {
        uint64_t W = 0;
        for (int k = 0; k < sh.segs; k++) W += sm.sum[b * sh.segs + k];
        return W << sh.cut_bits;
    };
    if (tid == 0) sm.border = 0;
    for (uint32_t i = tid; i < (uint32_t)items * keep; i += BT) s_place[i] = i % keep;
    __syncthreads();
    const uint64_t low = (1ull << sh.cut_bits) - 1;
    for (int b = w; b < a.beams; b += BW) {
        const int state = state_of(b);
        int N = 0;
        bool border = false;
        if (state == 1) {
            // The weights without their low bits, from shared memory, give a lower bound of N. It is N unless the
            // whole entry there passes at the upper end of the sum. The entries there are about table[0]^2 / W, at
            // least table[0] / 2^16, and the bits left out below table[0] / 2^31, so that is rare. Entries of one
            // value pass together, and may be thousands: none is tried one by one, the row takes the exact way below.
            const uint64_t W = sum_of(b), out = (uint64_t)a.vocab * low, up = W + out < W ? UINT64_MAX : W + out;
            N = norm_of(W, [&](int j) { return (uint64_t)sT[j] << sh.cut_bits; });
            border = N < a.tlen && (u128)a.table[N] * up > one;
        }
        if (lane == 0) {
            sm.row[b] = a.base[row0 + b] + N;
            sm.state[b] = border ? 3 : state;
            if (border) sm.border = 1;
        }
    }
    __syncthreads();
    if (sm.border) {
        // Sums next to a border of N: the low bits of the weights too, in the place of the table.
        for (int i = tid; i < a.tlen; i += BT) sT[i] = (uint32_t)(a.table[i] & low);
        __syncthreads();
        for (int b = 0; b < a.beams; b++) {
            if (sm.state[b] != 3) continue;
            const size_t lrow = lrow_of(b);
            uint64_t W = 0;
#pragma unroll 8
            for (int v = tid; v < a.vocab; v += BT) {
                const uint64_t o = (uint64_t)sm.top[b] - (uint64_t)a.tops[lrow * a.tops_stride + (v >> a.tsh)];
                const uint32_t d = a.dist[lrow * a.dist_stride + v];
                W += sT[o < (uint64_t)last ? (uint32_t)o + min(d, (uint32_t)last - (uint32_t)o) : (uint32_t)last];
            }
            for (int o = 16; o > 0; o >>= 1) W += __shfl_xor_sync(0xffffffffu, W, o);
            if (lane == 0) sm.redu[w] = W;
            __syncthreads();
            if (w == 0) {
                W = sum_of(b);
                for (int i = 0; i < BW; i++) W += sm.redu[i];
                const int N = norm_of(W, [&](int j) { return a.table[j]; });
                if (lane == 0) sm.row[b] = a.base[row0 + b] + N;
            }
            __syncthreads();
        }
    }
    // The merge of the lists: a candidate's place is the number of candidates before it (by cost, then
    // beam, then symbol). Each (candidate, list) pair is a bisection of its own.
    const uint32_t all = (uint32_t)items * keep;
    for (uint32_t i = tid; i < all * (uint32_t)items; i += BT) {
        const uint32_t cand = i / (uint32_t)items;
        const int o = (int)(i - cand * (uint32_t)items), l = (int)(cand / keep);
        const uint32_t hi0 = sm.len[o];
        if (o == l || cand - l * keep >= sm.len[l] || hi0 == 0) continue;
        const int b = l / sh.segs, ob = o / sh.segs;
        const uint32_t key = s_list[cand];
        const int64_t gap = sm.row[b] + (key >> 16) - sm.row[ob];  // candidates of o with a smaller D are before
        uint32_t lo = 0, hi = hi0;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2, k2 = s_list[o * keep + mid];
            const int64_t d = k2 >> 16;
            const bool before = ob == b ? k2 < key : d < gap || (d == gap && ob < b);
            if (before) lo = mid + 1;
            else hi = mid;
        }
        if (lo) atomicAdd(&s_place[cand], lo);
    }
    __syncthreads();
    uint32_t total = 0;
    for (int l = 0; l < items; l++) total += sm.len[l];
    const size_t to = (size_t)(blockIdx.x / C) * keep;
    for (uint32_t i = tid; i < all; i += BT) {
        const int l = (int)(i / keep), b = l / sh.segs;
        const uint32_t at = s_place[i];
        if (i - l * keep >= sm.len[l] || at >= keep) continue;
        const uint32_t key = s_list[i];
        a.parent[to + at] = (uint32_t)b;
        a.token[to + at] = sm.state[b] == 2 ? NO_KEY : key & 0xFFFFu;
        a.cost[to + at] = sm.row[b] + (key >> 16);
    }
    for (uint32_t i = total + tid; i < keep; i += BT) {
        a.parent[to + i] = NO_KEY;
        a.token[to + i] = NO_KEY;
        a.cost[to + i] = -1;
    }
}

size_t beam_smem(const BeamArgs& a, const BeamShape& sh) {
    return 16 * (((size_t)a.tlen + 4) / 4) + sizeof(BeamSmem) + 8 * (size_t)a.beams * sh.segs * a.keep +
           2 * (size_t)sh.batches * BT;
}

BeamShape beam_shape(const BeamArgs& a, int segs) {
    BeamShape sh;
    sh.segs = segs;
    sh.seg_vecs = ((a.vocab + 7) / 8 + segs - 1) / segs;
    sh.batches = (sh.seg_vecs + BU * BT - 1) / (BU * BT);
    sh.cut_bits = a.cut_bits;
    return sh;
}

constexpr size_t BEAM_SMEM_MAX = 227 * 1024;

}  // namespace

cudaError_t configure_beam() {
    cudaError_t e = cudaFuncSetAttribute((const void*)k_beam_select<true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)BEAM_SMEM_MAX);
    if (e != cudaSuccess) return e;
    return cudaFuncSetAttribute((const void*)k_beam_select<false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)BEAM_SMEM_MAX);
}

cudaError_t launch_beam_select(const BeamArgs& a, int num_sms, cudaStream_t st) {
    if (a.groups == 0) return cudaSuccess;
    // The split: `segs` segments a row and clusters of C blocks, by the time of the segments of the busiest
    // block (a fixed part each, and one that grows with their symbols and with the blocks that share an SM)
    // and of the end of a group. Measured by repeated calls: 256 groups of 8, one segment, C = 1, 2, 4, 8: 118, 99, 101, 101 us (two
    // segments 134 at best); 64 groups of 8: 81, 46, 33, 31 us (42); one group of 4: 43, 25, 17, 17 us, two
    // segments and C = 8 15 us, four 19 us; one lone beam 17 us whole, 11 us in eight segments. The rule takes the
    // best of each, or one within 1 %.
    int C = 1;
    BeamShape sh = beam_shape(a, 1);
    double best = 1e300;
    for (int s = 1; s <= 8; s *= 2) {
        if (s > 1 && (a.beams * s > MAX_ITEMS || a.vocab / s < 4 * BT)) break;
        const BeamShape x = beam_shape(a, s);
        for (int c = 1; c <= 8; c *= 2) {
            const double load = (double)a.groups * c / num_sms;  // blocks of an SM, over the whole launch
            const double waves = load > BEAM_BLOCKS ? load / BEAM_BLOCKS : 1.0;
            const double share = load < 1 ? 1.0 : load < BEAM_BLOCKS ? load : BEAM_BLOCKS;
            const double time = waves * ((a.beams * s + c - 1) / c * (3.0 + 6e-5 * a.vocab / s * share) + 6.0);
            if (time < best) {
                best = time;
                sh = x;
                C = c;
            }
        }
    }
    const bool vec = reinterpret_cast<uintptr_t>(a.dist) % 16 == 0 && a.dist_stride % 8 == 0;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)a.groups * C);
    cfg.blockDim = dim3(BT);
    cfg.dynamicSmemBytes = beam_smem(a, sh);
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)C;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return vec ? cudaLaunchKernelEx(&cfg, k_beam_select<true>, a, sh) : cudaLaunchKernelEx(&cfg, k_beam_select<false>, a, sh);
}

}  // namespace hs
