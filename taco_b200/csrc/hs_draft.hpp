// The kernels of drafts that branch: attention of draft trees, beam selection, and the moves of
// cache rows (beams' states, accepted paths). Launchers; every argument is checked by the caller.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <vector>

#include "hs_device.hpp"

namespace hs {

constexpr int MAX_TREE = 128;
constexpr int MAX_BEAMS = 32;
constexpr int MAX_KEEP = 64;
constexpr int ATTN_TABLE_MAX = 8192;

// A cache and its geometry (hs_kv_cache with the stride filled in).
struct CacheView {
    int8_t* k;
    int8_t* v;
    uint64_t slot_stride;
    uint32_t slots, planes;
    int n_ctx, hd;
    bool vec;  // 16-byte vectors fit every row of k and v
};

struct AttnRuleView {
    int32_t sm, om;
    int ss, os, P, tlen;
    const int32_t* table;  // padded to 4 entries
    int reach;             // the entries from table[reach - 1] on are equal (table_reach)
};

// The least length that gives every look-up of table[min(d, n - 1)].
inline int table_reach(const int32_t* table, int n) {
    while (n > 1 && table[n - 2] == table[n - 1]) n--;
    return n;
}

// hs_tree_seq on the device.
struct TreeSeq {
    uint32_t first_row, count, slot, prefix;
};

struct TreeArgs {
    CacheView cache;
    AttnRuleView rule;
    const int8_t* q;
    int8_t* out;
    uint64_t q_stride, out_stride;
    const TreeSeq* seqs;
    const uint32_t* mask;
    uint32_t plane0, n_rows, n_seq;
    int n_head, n_kv, max_count, max_keys, mask_words;
};

// hs_beam_select, with the table of the weight rule.
struct BeamArgs {
    const uint16_t* dist;
    const int64_t* tops;
    uint64_t dist_stride, tops_stride;
    const uint32_t* row_of;  // the logits row of each beam (null: beam i has row i)
    const int64_t* base;
    const uint8_t* finished;
    uint32_t* parent;
    uint32_t* token;
    int64_t* cost;
    const uint64_t* table;
    const uint32_t* high;   // table[j] >> cut_bits, then zeros to the next multiple of 4 past tlen
    uint64_t first;         // table[0]
    int tlen, last_weight;  // the last entry that is not 0
    int cut_bits;           // the low bits of a weight that a 32-bit look-up leaves out
    int tsh, vocab, groups, beams, keep;
};

// The bits of table[0] above 32.
inline int weight_cut_bits(uint64_t first) {
    int bits = 0;
    while ((first >> bits) >> 32) bits++;
    return bits;
}

// BeamArgs::high of a table.
inline std::vector<uint32_t> weight_high(const uint64_t* table, size_t n) {
    std::vector<uint32_t> t((n + 4) / 4 * 4, 0);
    const int bits = weight_cut_bits(table[0]);
    for (size_t j = 0; j < n; j++) t[j] = (uint32_t)(table[j] >> bits);
    return t;
}

cudaError_t configure_draft_kernels();  // the attention's, then the others'
cudaError_t configure_beam();
cudaError_t launch_tree_attention(const TreeArgs& a, int num_sms, int* err, cudaStream_t st);
cudaError_t launch_beam_select(const BeamArgs& a, int num_sms, cudaStream_t st);
cudaError_t launch_cache_reorder(const CacheView& c, const uint32_t* slots, const uint32_t* parents,
                                 const uint32_t* rows, uint32_t groups, uint32_t beams, int num_sms, int* err,
                                 cudaStream_t st);
cudaError_t launch_cache_commit(const CacheView& c, const TreeSeq* seqs, const uint32_t* path, const uint32_t* lengths,
                                uint32_t n_seq, uint32_t path_stride, int* err, cudaStream_t st);

}  // namespace hs
