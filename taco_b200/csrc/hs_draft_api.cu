// The C entry points of the device-resident operators (drafts that branch): argument checks on the
// host, then one launch on the caller's stream. Nothing here waits or allocates except the making and
// freeing of a rule.
#include <cuda_runtime.h>

#include <memory>
#include <new>
#include <string>
#include <vector>

#include "../../include/hardshell_b200.h"
#include "hs_device.hpp"
#include "hs_draft.hpp"
#include "hs_host.hpp"

using namespace hs;

static_assert(sizeof(hs_tree_seq) == sizeof(TreeSeq), "the sequence record of the ABI and of the kernels");
static_assert(HS_MAX_TREE == MAX_TREE && HS_MAX_BEAMS == MAX_BEAMS && HS_MAX_KEEP == MAX_KEEP, "the ABI's limits");

struct hs_attn_rule {
    DevInfo dev;
    AttnRuleView view{};
    int32_t* table = nullptr;
};

struct hs_weight_rule {
    DevInfo dev;
    uint64_t first = 0;
    int len = 0, last_weight = 0;
    uint64_t* table = nullptr;  // then the 32-bit look-ups
    uint32_t* high = nullptr;
};

namespace {

// Makes the device current and puts the caller's back at the end.
struct DeviceScope {
    int before = -1;
    cudaError_t e;
    explicit DeviceScope(int ordinal) {
        e = cudaGetDevice(&before);
        if (e == cudaSuccess && before != ordinal) e = cudaSetDevice(ordinal);
        else before = -1;
    }
    ~DeviceScope() {
        if (before >= 0) cudaSetDevice(before);
    }
};

int cuda_fail(const char* what, cudaError_t e) {
    cudaGetLastError();
    return host_fail(HS_CUDA, std::string(what) + " failed: " + cudaGetErrorString(e));
}

// An entry point's body: C++ exceptions (memory, strings) end here.
template <class F>
int guarded(F&& f) {
    try {
        return f();
    } catch (const std::bad_alloc&) {
        return host_fail(HS_CUDA, "out of host memory");
    } catch (...) {
        return host_fail(HS_CUDA, "an internal error");
    }
}

// The pointer is device (or managed) memory of this GPU.
int need_device(const void* p, int ordinal, const char* name) {
    if (!p) return host_fail(HS_BAD_ARGUMENT, std::string(name) + " is null");
    cudaPointerAttributes at;
    const cudaError_t e = cudaPointerGetAttributes(&at, p);
    if (e != cudaSuccess) return cuda_fail("cudaPointerGetAttributes", e);
    if ((at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged) || at.device != ordinal)
        return host_fail(HS_BAD_ARGUMENT, std::string(name) + " is not memory of GPU " + std::to_string(ordinal));
    return HS_OK;
}

// A table into device memory. The copy from pageable memory may return before its last part has arrived, so the
// call waits: the caller's stream may use the rule at once.
cudaError_t put_table(void* to, const void* of, size_t bytes) {
    const cudaError_t e = cudaMemcpy(to, of, bytes, cudaMemcpyHostToDevice);
    return e != cudaSuccess ? e : cudaStreamSynchronize(cudaStreamLegacy);
}

int need_aligned(const void* p, size_t to, const char* name) {
    if (reinterpret_cast<uintptr_t>(p) % to != 0)
        return host_fail(HS_BAD_ARGUMENT, std::string(name) + " is not aligned to " + std::to_string(to) + " bytes");
    return HS_OK;
}

template <typename T>
int need_array(const T* p, int ordinal, const char* name) {
    const int rc = need_device(p, ordinal, name);
    return rc ? rc : need_aligned(p, alignof(T), name);
}

int cache_view(const hs_kv_cache& c, int ordinal, CacheView* out) {
    int rc;
    if ((rc = need_device(c.k, ordinal, "cache.k")) || (rc = need_device(c.v, ordinal, "cache.v"))) return rc;
    if (c.slots == 0 || c.planes == 0 || c.planes > 65535 || c.n_ctx == 0 || c.n_ctx > (uint32_t)MAX_ATTN_CTX ||
        c.head_dim == 0 || c.head_dim > 1024 || (uint64_t)c.slots * c.planes >= (1ull << 31))
        return host_fail(HS_UNSUPPORTED, "the cache's slots, planes, n_ctx or head_dim are out of range");
    const uint64_t dense = (uint64_t)c.planes * c.n_ctx * c.head_dim;
    const uint64_t stride = c.slot_stride ? c.slot_stride : dense;
    if (stride < dense || stride > (1ull << 48)) return host_fail(HS_BAD_ARGUMENT, "slot_stride is less than a slot");
    *out = CacheView{c.k, c.v, stride, c.slots, c.planes, (int)c.n_ctx, (int)c.head_dim, false};
    out->vec = reinterpret_cast<uintptr_t>(c.k) % 16 == 0 && reinterpret_cast<uintptr_t>(c.v) % 16 == 0 &&
               stride % 16 == 0 && c.n_ctx % 16 == 0 && c.head_dim % 16 == 0;
    return HS_OK;
}

// The stream belongs to the device (a legacy or per-thread default stream belongs to the current one).
int check_stream(void* stream, int ordinal) {
    cudaStream_t st = (cudaStream_t)stream;
    if (!st || st == cudaStreamLegacy || st == cudaStreamPerThread) return HS_OK;
    // A capturing stream cannot be asked for its device; a launch on the wrong one fails by itself.
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    cudaError_t e = cudaStreamIsCapturing(st, &cap);
    if (e != cudaSuccess) return cuda_fail("cudaStreamIsCapturing", e);
    if (cap != cudaStreamCaptureStatusNone) return HS_OK;
    int dev = -1;
    e = cudaStreamGetDevice(st, &dev);
    if (e != cudaSuccess) return cuda_fail("cudaStreamGetDevice", e);
    if (dev != ordinal)
        return host_fail(HS_BAD_ARGUMENT, "the stream is one of GPU " + std::to_string(dev) + ", the handle of GPU " +
                                              std::to_string(ordinal));
    return HS_OK;
}

template <class F>
int launch(int ordinal, void* stream, const char* what, F&& f) {
    int rc = check_stream(stream, ordinal);
    if (rc) return rc;
    DeviceScope on(ordinal);
    if (on.e != cudaSuccess) return cuda_fail("cudaSetDevice", on.e);
    cudaGetLastError();  // an earlier call's error, already reported to its caller
    const cudaError_t e = f((cudaStream_t)stream);
    if (e != cudaSuccess) return cuda_fail(what, e);
    count_launch();
    return HS_OK;
}

// The checks of a call and the arguments of its launch. A call with nothing to do leaves `out` as it is: without
// trees, groups or beams.
int tree_args(const hs_attn_rule* rule, const hs_tree_attention* a, TreeArgs* out) {
    const int o = rule->dev.ordinal;
    if (a->n_seq == 0 || a->n_rows == 0 || a->max_count == 0) return HS_OK;
    TreeArgs t{};
    int rc;
    if ((rc = cache_view(a->cache, o, &t.cache)) || (rc = need_array(a->q, o, "q")) ||
        (rc = need_array(a->out, o, "out")) || (rc = need_array(a->seqs, o, "seqs")) ||
        (rc = need_array(a->mask, o, "mask")))
        return rc;
    if (a->n_head == 0 || a->n_head > 65535 || a->n_kv_head == 0 || a->n_head % a->n_kv_head != 0)
        return host_fail(HS_UNSUPPORTED, "n_head must be a multiple of n_kv_head");
    if (a->plane0 > a->cache.planes || a->n_kv_head > a->cache.planes - a->plane0)
        return host_fail(HS_BAD_ARGUMENT, "the layer's planes lie outside the cache");
    if (a->max_count > HS_MAX_TREE) return host_fail(HS_UNSUPPORTED, "a tree has at most 128 nodes");
    if (a->max_keys == 0 || a->max_keys > a->cache.n_ctx || a->max_count > a->max_keys)
        return host_fail(HS_BAD_ARGUMENT, "max_keys must be max_count to n_ctx");
    if (a->mask_words > 1024 || (uint64_t)a->mask_words * 32 < a->max_count)
        return host_fail(HS_BAD_ARGUMENT, "the mask has too few words for max_count nodes");
    if (a->n_seq > (1u << 20) || a->n_rows > (1u << 27)) return host_fail(HS_UNSUPPORTED, "too many trees or rows");
    const uint64_t tiles = ((uint64_t)a->max_count * (a->n_head / a->n_kv_head) + 15) / 16;
    if (a->n_seq * (uint64_t)a->n_kv_head * tiles > (1u << 30))
        return host_fail(HS_UNSUPPORTED, "too many trees times heads");
    const uint64_t width = (uint64_t)a->n_head * a->cache.head_dim;
    t.q_stride = a->q_stride ? a->q_stride : width;
    t.out_stride = a->out_stride ? a->out_stride : width;
    if (t.q_stride < width || t.out_stride < width)
        return host_fail(HS_BAD_ARGUMENT, "q_stride or out_stride is less than a row");
    t.rule = rule->view;
    t.q = a->q;
    t.out = a->out;
    t.seqs = reinterpret_cast<const TreeSeq*>(a->seqs);
    t.mask = a->mask;
    t.plane0 = a->plane0;
    t.n_rows = a->n_rows;
    t.n_seq = a->n_seq;
    t.n_head = (int)a->n_head;
    t.n_kv = (int)a->n_kv_head;
    t.max_count = (int)a->max_count;
    t.max_keys = (int)a->max_keys;
    t.mask_words = (int)a->mask_words;
    *out = t;
    return HS_OK;
}

int beam_args(const hs_weight_rule* rule, const hs_beam_select* a, BeamArgs* out) {
    const int o = rule->dev.ordinal;
    if (a->groups == 0 || a->keep == 0) return HS_OK;
    int rc;
    if ((rc = need_array(a->dist, o, "dist")) || (rc = need_array(a->tops, o, "tops")) ||
        (rc = need_array(a->base, o, "base")) || (rc = need_array(a->parent, o, "parent")) ||
        (rc = need_array(a->token, o, "token")) || (rc = need_array(a->cost, o, "cost")) ||
        (a->finished && (rc = need_array(a->finished, o, "finished"))))
        return rc;
    if (a->tile_shift != 6 && a->tile_shift != 7) return host_fail(HS_UNSUPPORTED, "tile_shift must be 6 or 7");
    if (a->vocab < 2 || a->vocab > (uint32_t)MAX_CODER_VOCAB)
        return host_fail(HS_UNSUPPORTED, "the vocabulary needs 2 to 65536 symbols");
    if (a->beams == 0 || a->beams > HS_MAX_BEAMS) return host_fail(HS_UNSUPPORTED, "a group has 1 to 32 beams");
    if (a->keep > HS_MAX_KEEP) return host_fail(HS_UNSUPPORTED, "keep is more than 64");
    if (a->groups > (1u << 24)) return host_fail(HS_UNSUPPORTED, "too many groups");
    if (rule->first > UINT64_MAX / a->vocab)
        return host_fail(HS_UNSUPPORTED, "vocab times the largest weight does not fit in 64 bits");
    const uint64_t tiles = (a->vocab + (1u << a->tile_shift) - 1) >> a->tile_shift;
    BeamArgs b{};
    b.dist_stride = a->dist_stride ? a->dist_stride : a->vocab;
    b.tops_stride = a->tops_stride ? a->tops_stride : tiles;
    if (b.dist_stride < a->vocab || b.tops_stride < tiles)
        return host_fail(HS_BAD_ARGUMENT, "dist_stride or tops_stride is less than a row");
    b.dist = a->dist;
    b.tops = a->tops;
    b.base = a->base;
    b.finished = a->finished;
    b.parent = a->parent;
    b.token = a->token;
    b.cost = a->cost;
    b.table = rule->table;
    b.high = rule->high;
    b.tlen = rule->len;
    b.last_weight = rule->last_weight;
    b.cut_bits = weight_cut_bits(rule->first);
    b.first = rule->first;
    b.tsh = (int)a->tile_shift;
    b.vocab = (int)a->vocab;
    b.groups = (int)a->groups;
    b.beams = (int)a->beams;
    b.keep = (int)a->keep;
    *out = b;
    return HS_OK;
}

int reorder_args(const DevInfo& d, const hs_cache_reorder* a, CacheView* out) {
    if (a->groups == 0 || a->beams == 0) return HS_OK;
    CacheView c;
    int rc;
    if ((rc = cache_view(a->cache, d.ordinal, &c)) || (rc = need_array(a->parents, d.ordinal, "parents")) ||
        (rc = need_array(a->rows, d.ordinal, "rows")) ||
        (a->slots && (rc = need_array(a->slots, d.ordinal, "slots"))))
        return rc;
    if (a->beams > HS_MAX_BEAMS) return host_fail(HS_UNSUPPORTED, "a group has 1 to 32 beams");
    if ((uint64_t)a->groups * a->beams > a->cache.slots)
        return host_fail(HS_BAD_ARGUMENT, "more beams than the cache has slots");
    *out = c;
    return HS_OK;
}

int commit_args(const DevInfo& d, const hs_cache_commit* a, CacheView* out) {
    if (a->n_seq == 0) return HS_OK;
    CacheView c;
    int rc;
    if ((rc = cache_view(a->cache, d.ordinal, &c)) || (rc = need_array(a->seqs, d.ordinal, "seqs")) ||
        (rc = need_array(a->path, d.ordinal, "path")) || (rc = need_array(a->lengths, d.ordinal, "lengths")))
        return rc;
    if (a->n_seq > a->cache.slots) return host_fail(HS_BAD_ARGUMENT, "more trees than the cache has slots");
    *out = c;
    return HS_OK;
}

}  // namespace

extern "C" {

int hs_dev_check(hs_dev* dev, void* stream) {
    if (!dev) return host_fail(HS_BAD_ARGUMENT, "null argument");
    return guarded([&]() -> int {
        const DevInfo d = dev_info(dev);
        int rc = check_stream(stream, d.ordinal);
        if (rc) return rc;
        DeviceScope on(d.ordinal);
        if (on.e != cudaSuccess) return cuda_fail("cudaSetDevice", on.e);
        cudaStream_t st = (cudaStream_t)stream;
        // A wait would end the capture with an error (the legacy stream is never one that captures).
        cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
        cudaError_t e = st && st != cudaStreamLegacy ? cudaStreamIsCapturing(st, &cap) : cudaSuccess;
        if (e != cudaSuccess) return cuda_fail("cudaStreamIsCapturing", e);
        if (cap != cudaStreamCaptureStatusNone) return host_fail(HS_BAD_ARGUMENT, "the stream is being captured");
        e = cudaStreamSynchronize(st);
        if (e != cudaSuccess) return cuda_fail("cudaStreamSynchronize", e);
        int code = 0;
        if ((e = cudaMemcpyAsync(&code, d.op_err, sizeof(int), cudaMemcpyDeviceToHost, st)) != cudaSuccess ||
            (e = cudaStreamSynchronize(st)) != cudaSuccess)
            return cuda_fail("the read of the error word", e);
        if (code == 0) return HS_OK;
        if ((e = cudaMemsetAsync(d.op_err, 0, sizeof(int), st)) != cudaSuccess ||
            (e = cudaStreamSynchronize(st)) != cudaSuccess)
            return cuda_fail("the clearing of the error word", e);
        if (code == ERR_DRAFT_SEQ)
            return host_fail(HS_BAD_ARGUMENT, "a tree's rows, slot or prefix are out of range");
        if (code == ERR_DRAFT_PARENT)
            return host_fail(HS_BAD_ARGUMENT, "a beam's parent, slot or rows are out of range");
        if (code == ERR_DRAFT_PATH)
            return host_fail(HS_BAD_ARGUMENT, "a path is not strictly increasing inside its tree");
        return host_fail(HS_CUDA, "a kernel wait timed out (code " + std::to_string(code) + ")");
    });
}

int hs_attn_rule_new(hs_dev* dev, int32_t score_m, uint32_t score_s, int32_t out_m, uint32_t out_s, uint32_t softmax_p,
                     const int32_t* exp_table, uint32_t table_len, hs_attn_rule** out) {
    if (!dev || !exp_table || !out) return host_fail(HS_BAD_ARGUMENT, "null argument");
    *out = nullptr;
    return guarded([&]() -> int {
        if (table_len == 0 || table_len > (uint32_t)ATTN_TABLE_MAX)
            return host_fail(HS_UNSUPPORTED, "the exponent table needs 1 to 8192 entries");
        if (softmax_p > 30) return host_fail(HS_UNSUPPORTED, "the softmax precision is more than 30");
        if (score_s > 127 || out_s > 127) return host_fail(HS_UNSUPPORTED, "a shift is more than 127");
        for (uint32_t j = 0; j < table_len; j++)
            if (exp_table[j] < 0) return host_fail(HS_BAD_ARGUMENT, "an entry of the exponent table is negative");
        auto r = std::make_unique<hs_attn_rule>();
        r->dev = dev_info(dev);
        DeviceScope on(r->dev.ordinal);
        if (on.e != cudaSuccess) return cuda_fail("cudaSetDevice", on.e);
        std::vector<int32_t> t(exp_table, exp_table + table_len);
        t.resize((t.size() + 3) & ~(size_t)3, 0);
        cudaError_t e = cudaMalloc(&r->table, 4 * t.size());
        if (e != cudaSuccess) return cuda_fail("cudaMalloc", e);
        e = put_table(r->table, t.data(), 4 * t.size());
        if (e != cudaSuccess) {
            cudaFree(r->table);
            return cuda_fail("the copy of the table", e);
        }
        r->view = AttnRuleView{score_m, out_m, (int)score_s, (int)out_s, (int)softmax_p, (int)table_len, r->table,
                               table_reach(exp_table, (int)table_len)};
        *out = r.release();
        return HS_OK;
    });
}

void hs_attn_rule_free(hs_attn_rule* rule) {
    if (!rule) return;
    DeviceScope on(rule->dev.ordinal);
    cudaFree(rule->table);
    delete rule;
}

int hs_op_tree_attention_check(const hs_attn_rule* rule, const hs_tree_attention* a) {
    if (!rule || !a) return host_fail(HS_BAD_ARGUMENT, "null argument");
    TreeArgs t{};
    return guarded([&]() -> int { return tree_args(rule, a, &t); });
}

int hs_op_tree_attention(hs_attn_rule* rule, const hs_tree_attention* a, void* stream) {
    if (!rule || !a) return host_fail(HS_BAD_ARGUMENT, "null argument");
    return guarded([&]() -> int {
        TreeArgs t{};
        const int rc = tree_args(rule, a, &t);
        if (rc || t.n_seq == 0) return rc;
        return launch(rule->dev.ordinal, stream, "the tree attention", [&](cudaStream_t st) {
            return launch_tree_attention(t, rule->dev.num_sms, rule->dev.op_err, st);
        });
    });
}

int hs_weight_rule_new(hs_dev* dev, const uint64_t* table, uint32_t table_len, hs_weight_rule** out) {
    if (!dev || !table || !out) return host_fail(HS_BAD_ARGUMENT, "null argument");
    *out = nullptr;
    return guarded([&]() -> int {
        if (table_len == 0 || table_len > (uint32_t)MAX_LOGIT_TABLE)
            return host_fail(HS_UNSUPPORTED, "the weight table needs 1 to 16384 entries");
        if (table[0] == 0) return host_fail(HS_BAD_ARGUMENT, "the first weight is 0");
        for (uint32_t j = 1; j < table_len; j++)
            if (table[j] > table[j - 1]) return host_fail(HS_BAD_ARGUMENT, "the weight table increases");
        auto r = std::make_unique<hs_weight_rule>();
        r->dev = dev_info(dev);
        r->first = table[0];
        r->len = (int)table_len;
        while (r->last_weight + 1 < r->len && table[r->last_weight + 1] != 0) r->last_weight++;
        DeviceScope on(r->dev.ordinal);
        if (on.e != cudaSuccess) return cuda_fail("cudaSetDevice", on.e);
        const std::vector<uint32_t> high = weight_high(table, table_len);
        const size_t bytes = 8 * (((size_t)table_len + 1) & ~(size_t)1);  // `high` starts 16-byte aligned
        cudaError_t e = cudaMalloc(&r->table, bytes + 4 * high.size());
        if (e != cudaSuccess) return cuda_fail("cudaMalloc", e);
        r->high = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(r->table) + bytes);
        if ((e = put_table(r->table, table, 8 * (size_t)table_len)) != cudaSuccess ||
            (e = put_table(r->high, high.data(), 4 * high.size())) != cudaSuccess) {
            cudaFree(r->table);
            return cuda_fail("the copy of the table", e);
        }
        *out = r.release();
        return HS_OK;
    });
}

void hs_weight_rule_free(hs_weight_rule* rule) {
    if (!rule) return;
    DeviceScope on(rule->dev.ordinal);
    cudaFree(rule->table);
    delete rule;
}

int hs_op_beam_select_check(const hs_weight_rule* rule, const hs_beam_select* a) {
    if (!rule || !a) return host_fail(HS_BAD_ARGUMENT, "null argument");
    BeamArgs b{};
    return guarded([&]() -> int { return beam_args(rule, a, &b); });
}

int hs_op_beam_select(hs_weight_rule* rule, const hs_beam_select* a, void* stream) {
    if (!rule || !a) return host_fail(HS_BAD_ARGUMENT, "null argument");
    return guarded([&]() -> int {
        BeamArgs b{};
        const int rc = beam_args(rule, a, &b);
        if (rc || b.groups == 0) return rc;
        return launch(rule->dev.ordinal, stream, "the beam selection",
                      [&](cudaStream_t st) { return launch_beam_select(b, rule->dev.num_sms, st); });
    });
}

int hs_op_cache_reorder_check(hs_dev* dev, const hs_cache_reorder* a) {
    if (!dev || !a) return host_fail(HS_BAD_ARGUMENT, "null argument");
    CacheView c{};
    return guarded([&]() -> int { return reorder_args(dev_info(dev), a, &c); });
}

int hs_op_cache_reorder(hs_dev* dev, const hs_cache_reorder* a, void* stream) {
    if (!dev || !a) return host_fail(HS_BAD_ARGUMENT, "null argument");
    return guarded([&]() -> int {
        const DevInfo d = dev_info(dev);
        CacheView c{};
        const int rc = reorder_args(d, a, &c);
        if (rc || !c.k) return rc;
        return launch(d.ordinal, stream, "the cache reorder", [&](cudaStream_t st) {
            return launch_cache_reorder(c, a->slots, a->parents, a->rows, a->groups, a->beams, d.num_sms, d.op_err, st);
        });
    });
}

int hs_op_cache_commit_check(hs_dev* dev, const hs_cache_commit* a) {
    if (!dev || !a) return host_fail(HS_BAD_ARGUMENT, "null argument");
    CacheView c{};
    return guarded([&]() -> int { return commit_args(dev_info(dev), a, &c); });
}

int hs_op_cache_commit(hs_dev* dev, const hs_cache_commit* a, void* stream) {
    if (!dev || !a) return host_fail(HS_BAD_ARGUMENT, "null argument");
    return guarded([&]() -> int {
        const DevInfo d = dev_info(dev);
        CacheView c{};
        const int rc = commit_args(d, a, &c);
        if (rc || !c.k) return rc;
        return launch(d.ordinal, stream, "the cache commit", [&](cudaStream_t st) {
            return launch_cache_commit(c, reinterpret_cast<const TreeSeq*>(a->seqs), a->path, a->lengths, a->n_seq,
                                       a->path_stride, d.op_err, st);
        });
    });
}

}  // extern "C"
