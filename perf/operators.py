"""The operators of speculative drafting, measured alone: attention of a tree of drafted tokens over
the cache, the selection of beams over the vocabulary, the reordering of the beams' caches and the
commit of an accepted path. Whole numbers throughout: HardShell's integer rules (the exponent tables
of 8,192 entries with a unit of 2^-8, probabilities in units of 2^-30), so the outputs of the plain
forms and of the kernels are equal, bit for bit.
"""

import functools

import numpy as np
import torch

own = False

TABLE_LEN = 8192
SOFTMAX_P = 30
ATTN_EXP, LOGIT_EXP = 30, 40  # table[0] = 2^30 and 2^40
LAST = TABLE_LEN - 1
NONE = -1                     # the parent and token of an output that no candidate fills
FAR = 1 << 62
WEIGHT_OF = {64: 35, 128: 36}  # the score shift that gives scores of about 1.5 nats at a head width


def exp_table(e):
    """round(2^e exp(-j / 256)): the tables of the synthetic model (attention 2^30, logits 2^40)."""
    return np.rint(2.0 ** e * np.exp(-np.arange(TABLE_LEN) / 256.0)).astype(np.int64)


ATTN_TABLE, LOGIT_TABLE = exp_table(ATTN_EXP), exp_table(LOGIT_EXP)
LAST_WEIGHT = int(np.flatnonzero(LOGIT_TABLE > 0)[-1])  # symbols farther than this have weight 0
SCORE_M, OUT_M, OUT_S = 1_346_000_000, 1_181_116_006, 58


@functools.lru_cache(maxsize=None)
def on_gpu(name):
    return torch.from_numpy(ATTN_TABLE if name == "attn" else LOGIT_TABLE).cuda()


# ---- the cases ----


def tree(name, n_seq, count, n_ctx, keys, heads=12, kv_heads=12, width=64, ragged=True):
    return {"name": name, "op": "tree", "n_seq": n_seq, "count": count, "n_ctx": n_ctx, "keys": keys,
            "heads": heads, "kv_heads": kv_heads, "width": width, "ragged": ragged}


def beam(name, groups, beams, keep, vocab):
    return {"name": name, "op": "beam", "groups": groups, "beams": beams, "keep": keep, "vocab": vocab}


def reorder(name, groups, beams, planes, n_ctx, rows, width=64):
    return {"name": name, "op": "reorder", "groups": groups, "beams": beams, "planes": planes, "n_ctx": n_ctx,
            "rows": rows, "width": width}


def commit(name, n_seq, count, path, planes, n_ctx, width=64):
    return {"name": name, "op": "commit", "n_seq": n_seq, "count": count, "path": path, "planes": planes,
            "n_ctx": n_ctx, "width": width}


def listed():
    return [
        # One stream verifies a small tree in one layer of GPT-2 124M: latency.
        tree("tree 1x8 at 200", 1, 8, 1024, 200),
        # A batch of streams, trees of up to 16 nodes, full contexts: the ordinary step of an unfold.
        tree("tree 64x16 at 1024", 64, 16, 1024, 1024),
        # Many streams with wide trees: the largest pass.
        tree("tree 256x64 at 1024", 256, 64, 1024, 1024),
        # The longest context of the engine (8,192 rows), few streams: the key axis has to be split.
        tree("tree 8x31 at 8192", 8, 31, 8192, 8192),
        # One stream drafts with 4 beams over GPT-2's vocabulary.
        beam("beam 1x4", 1, 4, 4, 50257),
        # 64 streams with 8 beams each.
        beam("beam 64x8", 64, 8, 8, 50257),
        # 256 streams with 8 beams, 16 kept (a tree that widens): 206 MB of logits.
        beam("beam 256x8 keep 16", 256, 8, 16, 50257),
        # The caches of one group of 8 beams, all layers of GPT-2 124M, 300 rows held.
        reorder("reorder 1x8 at 300", 1, 8, 144, 1024, 300),
        # 32 groups of 4 beams at 700 rows: 1.6 GB held in the caches' first rows.
        reorder("reorder 32x4 at 700", 32, 4, 144, 1024, 700),
        # One stream accepts 5 of 16 drafted nodes.
        commit("commit 1x16 path 5", 1, 16, 5, 144, 1024),
        # 64 streams accept up to 8 of 32 nodes.
        commit("commit 64x32 path 8", 64, 32, 8, 144, 1024),
        # 64 streams accept long paths of wide trees.
        commit("commit 64x128 path 24", 64, 128, 24, 144, 1024),
    ]


def log_between(rng, a, b):
    """A whole number of [a, b], spread over its logarithm."""
    return min(b, max(a, int(round(a * (b / a) ** rng.random()))))


def draw(rng):
    op = rng.choice(("tree", "tree", "beam", "reorder", "commit"))
    if op == "tree":
        n_ctx = rng.choice((512, 1024, 1040, 2048, 4096, 8192))
        heads, kv_heads, width = rng.choice(((12, 12, 64), (2, 2, 64), (16, 16, 64), (12, 4, 64), (16, 2, 64),
                                             (8, 8, 128), (16, 4, 128)))
        keys = log_between(rng, 16, n_ctx)
        count = min(log_between(rng, 1, 128), keys)
        most = min(256 * 64 * 12 * 1024 // (count * heads * keys), 256 * 12 * 1024 * 64 // (kv_heads * n_ctx * width))
        c = tree("", log_between(rng, 1, max(1, min(256, most))), count, n_ctx, keys, heads, kv_heads, width,
                 rng.random() < 0.7)
    elif op == "beam":
        vocab = rng.choice((50257, 50257, log_between(rng, 300, 65536)))
        beams = log_between(rng, 1, 32)
        groups = log_between(rng, 1, max(1, min(256, 2048 * 50257 // (beams * vocab))))
        c = beam("", groups, beams, log_between(rng, 1, min(64, 2 * beams)), vocab)
    elif op == "reorder":
        n_ctx, planes = rng.choice(((512, 4), (1024, 24), (1024, 144), (2048, 48)))
        beams = log_between(rng, 2, 32)
        most = 128 * 144 * 1024 // (planes * n_ctx * beams)
        c = reorder("", log_between(rng, 1, max(1, min(64, most))), beams, planes, n_ctx, log_between(rng, 1, n_ctx))
    else:
        n_ctx, planes = rng.choice(((512, 4), (1024, 24), (1024, 144), (2048, 48)))
        count = log_between(rng, 2, 128)
        most = 64 * 144 * 1024 // (planes * n_ctx)
        c = commit("", log_between(rng, 1, max(1, min(64, most))), count, log_between(rng, 1, min(count, 24)), planes,
                   n_ctx)
    del c["name"]
    return c


# ---- the inputs ----


def small_ints(shape, std, g):
    """int8 activations as the calibrated engine has them: normal, the largest at 127."""
    return (torch.randn(shape, generator=g, device="cuda") * std).round_().clamp_(-127, 127).to(torch.int8)


def noise(shape, g):
    return torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)


def seqs_of(case, r):
    """[n_seq, 4] (first row, count, slot, prefix): ragged trees over ragged contexts, slots shuffled."""
    n, keys = case["n_seq"], case["keys"]
    count = np.full(n, case["count"], np.int64)
    total = np.full(n, keys, np.int64)
    if case["ragged"]:
        # The same sizes for every seed (from half to the whole), dealt to the sequences by the seed.
        count = r.permutation(np.linspace(case["count"] - case["count"] // 2, case["count"], n).round().astype(np.int64))
        total = r.permutation(np.linspace(max(case["count"], keys - keys // 2), keys, n).round().astype(np.int64))
    first = np.concatenate([[0], np.cumsum(count)[:-1]])
    return np.stack([first, count, r.permutation(n), total - count], 1).astype(np.int32)


def masks_of(count, words, r):
    """Bit j of a row: node j is the row's node or one of its ancestors. Random trees, a node's
    parent among the 4 nodes before it (or the last token of the context)."""
    out = np.zeros((int(count.sum()), words), np.uint32)
    row = 0
    for c in count.tolist():
        parent = np.maximum(np.arange(c) - r.integers(1, 5, c), -1)
        for i, p in enumerate(parent.tolist()):
            if p >= 0:
                out[row + i] = out[row + p]
            out[row + i, i >> 5] |= np.uint32(1 << (i & 31))
        row += c
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = np.random.default_rng(seed)
    s = {"case": case}
    if case["op"] == "tree":
        seqs = seqs_of(case, r)
        rows, words = int(seqs[:, 1].sum()), (case["count"] + 31) // 32
        cache = (case["n_seq"], case["kv_heads"])
        s["k"] = small_ints(cache + (case["n_ctx"], case["width"]), 33.0, g)
        s["v"] = small_ints(cache + (case["width"], case["n_ctx"]), 33.0, g)  # transposed, as the engine keeps it
        s["q"] = small_ints((rows, case["heads"], case["width"]), 33.0, g)
        s["seqs"] = torch.from_numpy(seqs).cuda()
        s["mask"] = torch.from_numpy(masks_of(seqs[:, 1], words, r).view(np.int32)).cuda()
        s["out"] = torch.zeros_like(s["q"])
    elif case["op"] == "beam":
        rows, vocab = case["groups"] * case["beams"], case["vocab"]
        ld, tiles = -(-vocab // 256) * 256, -(-vocab // 128)
        # Logits of 2.5 nats' spread, and a few likely tokens a row; in the form of the LM head: the
        # maximum of each tile of 128 symbols and every symbol's distance from it, cut at the table.
        logits = torch.randn((rows, tiles * 128), generator=g, device="cuda") * 640
        likely = torch.randint(0, vocab, (rows, 24), generator=g, device="cuda")
        logits.scatter_add_(1, likely, torch.rand((rows, 24), generator=g, device="cuda") * 2600)
        logits[:, vocab:] = -1e9
        logits = logits.round_().to(torch.int32).view(rows, tiles, 128)
        top = logits.amax(2)
        s["tops"] = top.to(torch.int64) + 12345
        dist = (top[:, :, None] - logits).clamp_(max=LAST).to(torch.int16).view(rows, tiles * 128)
        s["dist"] = torch.zeros((rows, ld), dtype=torch.int16, device="cuda")
        s["dist"][:, :vocab] = dist[:, :vocab]
        base = r.integers(0, 4000, rows).astype(np.int64)
        s["base"] = torch.from_numpy(base).cuda()
        n = (case["groups"], case["keep"])
        s["parent"], s["token"] = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2))
        s["cost"] = torch.zeros(n, dtype=torch.int64, device="cuda")
    else:
        slots = case["groups"] * case["beams"] if case["op"] == "reorder" else case["n_seq"]
        s["k"] = noise((slots, case["planes"], case["n_ctx"], case["width"]), g)
        s["v"] = noise((slots, case["planes"], case["width"], case["n_ctx"]), g)
        if case["op"] == "reorder":
            # The parents of a beam step: about half of the beams live on, in any order.
            likely = r.integers(0, case["beams"], (case["groups"], case["beams"] // 2 + 1))
            pick = r.integers(0, likely.shape[1], (case["groups"], case["beams"]))
            s["parent"] = torch.from_numpy(np.take_along_axis(likely, pick, 1).astype(np.int32)).cuda()
            s["slots"] = torch.from_numpy(r.permutation(slots).astype(np.int32)).cuda()
            s["rows"] = torch.full((slots,), case["rows"], dtype=torch.int32, device="cuda")
        else:
            n = case["n_seq"]
            count = np.full(n, case["count"], np.int64)
            prefix = r.integers(0, case["n_ctx"] - case["count"] + 1, n)
            s["seqs"] = torch.from_numpy(
                np.stack([np.cumsum(count) - count, count, r.permutation(n), prefix], 1).astype(np.int32)).cuda()
            length = r.integers((case["path"] + 1) // 2, case["path"] + 1, n)
            length[0] = case["path"]
            picks = np.sort(np.stack([r.permutation(case["count"])[: case["path"]] for _ in range(n)]), 1)
            s["path"] = torch.from_numpy(picks.astype(np.int32)).cuda()
            s["length"] = torch.from_numpy(length.astype(np.int32)).cuda()
    return s


# ---- one pass ----


def plain_tree(s):
    c = s["case"]
    n, kv, hd, group = c["n_seq"], c["kv_heads"], c["width"], c["heads"] // c["kv_heads"]
    first, count, slot, prefix = s["seqs"].long().unbind(1)
    node = torch.arange(c["count"], device="cuda")
    key = torch.arange(c["keys"], device="cuda")
    row = (first[:, None] + node.clamp(max=c["count"] - 1)).clamp(max=s["q"].shape[0] - 1)  # [n, count]
    q = s["q"][row].view(n, c["count"], kv, group, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, hd).float()
    dot = (q @ s["k"][slot, :, : c["keys"]].float().transpose(2, 3)).long()  # below 2^24: exact in 32 bits
    j = key - prefix[:, None]  # [n, keys]: the node of a key, below 0 in the context
    word = (j.clamp(0, c["count"] - 1) >> 5)[:, None].expand(n, c["count"], c["keys"])
    bit = (s["mask"][row].long().gather(2, word) >> (j.clamp(0, c["count"] - 1) & 31)[:, None]) & 1
    seen = (j < 0)[:, None] | ((j < count[:, None])[:, None] & (bit != 0))  # [n, count, keys]
    seen = seen[:, None, None].expand(n, kv, group, c["count"], c["keys"]).reshape(dot.shape)
    shift = WEIGHT_OF[hd]
    score = ((dot * SCORE_M + (1 << (shift - 1))) >> shift).masked_fill(~seen, -FAR)
    far = (score.amax(3, keepdim=True) - score).clamp(0, LAST)
    e = on_gpu("attn")[far].masked_fill(~seen, 0)
    p = (e << SOFTMAX_P) // e.sum(3, keepdim=True).clamp(min=1)
    acc = (p.double() @ s["v"][slot, :, :, : c["keys"]].double().transpose(2, 3))  # below 2^38: exact in 64 bits
    # acc * OUT_M takes up to 68 bits: its two halves apart, acc = hi 2^16 + lo.
    acc = acc.long()
    hi, lo = acc >> 16, acc & 0xFFFF
    out = (hi * OUT_M + ((lo * OUT_M + (1 << (OUT_S - 1))) >> 16)) >> (OUT_S - 16)
    out = out.clamp(-127, 127).to(torch.int8).view(n, kv, group, c["count"], hd).permute(0, 3, 1, 2, 4)
    alive = node < count[:, None]
    full = torch.zeros_like(s["q"])
    full[row[alive]] = out.reshape(n, c["count"], c["heads"], hd)[alive]
    return full


def plain_beam(s):
    c = s["case"]
    rows, vocab = c["groups"] * c["beams"], c["vocab"]
    symbol = torch.arange(vocab, device="cuda")
    off = s["tops"].amax(1, keepdim=True) - s["tops"]
    far = (off[:, symbol >> 7] + s["dist"][:, :vocab]).clamp(max=LAST)
    w = on_gpu("logits")[far]
    total = w.sum(1, dtype=torch.int64)
    # table[j] * total > table[0]^2, as table[j] > 2^80 / total
    border = float(1 << (2 * LOGIT_EXP)) / total.double()
    norm = (on_gpu("logits").double() > border[:, None]).sum(1)
    cost = (s["base"] + norm)[:, None] + far
    # Equal costs go to the lower beam, then the lower symbol: the place is part of the key.
    place = torch.arange(c["beams"] * vocab, device="cuda")
    key = (cost * (c["beams"] * vocab)).masked_fill(w == 0, FAR).view(c["groups"], -1)
    key = torch.where(key < FAR, key + place, key)
    best = key.sort(1).values[:, : c["keep"]]
    have = best < FAR
    at = best % (c["beams"] * vocab)
    return {"parent": torch.where(have, at // vocab, NONE).int(), "token": torch.where(have, at % vocab, NONE).int(),
            "cost": torch.where(have, best // (c["beams"] * vocab), NONE)}


def plain_reorder(s):
    c = s["case"]
    groups = s["slots"].long().view(c["groups"], c["beams"])
    source = torch.empty_like(s["slots"].long())
    source[groups.view(-1)] = groups.gather(1, s["parent"].long()).view(-1)
    n = c["rows"]
    s["k"][:, :, :n] = s["k"][source, :, :n]
    s["v"][:, :, :, :n] = s["v"][source, :, :, :n]
    return {"k": s["k"], "v": s["v"]}


def plain_commit(s):
    _, _, slot, prefix = s["seqs"].long().unbind(1)
    j = torch.arange(s["path"].shape[1], device="cuda")
    moved = torch.where(j < s["length"][:, None], s["path"].long(), j)  # past a path's end a row stays
    to, of = prefix[:, None] + j, prefix[:, None] + moved
    s["k"][slot[:, None], :, to] = s["k"][slot[:, None], :, of]
    s["v"][slot[:, None], :, :, to] = s["v"][slot[:, None], :, :, of]
    return {"k": s["k"], "v": s["v"]}


PLAIN = {"tree": plain_tree, "beam": plain_beam, "reorder": plain_reorder, "commit": plain_commit}


@functools.lru_cache(maxsize=None)
def engine(what, width=0):
    """The device handle and the model's rules, made once as a loaded model has them."""
    from taco_b200 import backend as B

    if what == "device":
        return B.CudaDevice(torch.cuda.current_device())
    if what == "attn":
        return B.AttnRule(engine("device"), SCORE_M, WEIGHT_OF[width], OUT_M, OUT_S, SOFTMAX_P, ATTN_TABLE)
    return B.WeightRule(engine("device"), LOGIT_TABLE)


def call_of(s):
    """The framework's call on these buffers: its arguments are bound once, as a decoding loop does."""
    from taco_b200 import backend as B

    c = s["case"]
    if c["op"] == "beam":
        return B.BeamSelect(engine("logits"), dist=s["dist"], tops=s["tops"], vocab=c["vocab"], groups=c["groups"],
                            beams=c["beams"], keep=c["keep"], base=s["base"], parent=s["parent"], token=s["token"],
                            cost=s["cost"])
    cache = B.KvCache(k=s["k"], v=s["v"], slots=s["k"].shape[0], planes=s["k"].shape[1], n_ctx=c["n_ctx"],
                      head_dim=c["width"])
    if c["op"] == "tree":
        return B.TreeAttention(engine("attn", c["width"]), cache, heads=c["heads"], kv_heads=c["kv_heads"],
                               q=s["q"], out=s["out"], rows=s["q"].shape[0], seqs=s["seqs"], n_seq=c["n_seq"],
                               max_count=c["count"], max_keys=c["keys"], mask=s["mask"],
                               mask_words=s["mask"].shape[1])
    if c["op"] == "reorder":
        return B.CacheReorder(engine("device"), cache, groups=c["groups"], beams=c["beams"], slots=s["slots"],
                              parent=s["parent"], rows=s["rows"])
    return B.CacheCommit(engine("device"), cache, seqs=s["seqs"], n_seq=c["n_seq"], path=s["path"],
                         path_ld=s["path"].shape[1], length=s["length"])


def run(state):
    if not own:
        return PLAIN[state["case"]["op"]](state)
    if "call" not in state:
        state["call"] = call_of(state)
    state["call"].run(torch.cuda.current_stream().cuda_stream)
    op = state["case"]["op"]
    if op == "tree":
        return state["out"]
    return {k: state[k] for k in (("parent", "token", "cost") if op == "beam" else ("k", "v"))}


# ---- what a pass cannot do without ----


def work(case):
    if case["op"] == "tree":
        part = 0.75 if case["ragged"] and case["n_seq"] > 1 else 1.0  # the mean of the ragged sizes
        rows, keys = case["n_seq"] * case["count"] * part, case["keys"] * part
        return {"bytes": 2 * case["n_seq"] * case["kv_heads"] * keys * case["width"]
                + 2 * rows * case["heads"] * case["width"], "flops": 4 * rows * case["heads"] * keys * case["width"]}
    if case["op"] == "beam":
        rows = case["groups"] * case["beams"]
        return {"bytes": rows * (2 * case["vocab"] + 8 * (-(-case["vocab"] // 128))) + 16 * case["groups"] * case["keep"],
                "flops": 3 * rows * case["vocab"]}
    row = 2 * case["planes"] * case["width"]  # the bytes of a row's keys and values
    if case["op"] == "reorder":
        # A slot is written when its parent is another beam; a source is read once.
        b = case["beams"]
        live = b // 2 + 1
        distinct = b * (1 - (1 - 1 / b) ** live)
        return {"bytes": row * case["rows"] * case["groups"] * (b * (1 - 1 / b) + distinct), "flops": 0}
    moved = case["n_seq"] * case["path"] * (0.75 if case["n_seq"] > 1 else 1.0)
    return {"bytes": 2 * row * moved, "flops": 0}


# ---- the operators' definitions in 64 bits, sequence by sequence ----


def exact_tree(s):
    c = s["case"]
    group, table = c["heads"] // c["kv_heads"], torch.from_numpy(ATTN_TABLE).double().cuda()
    out = torch.zeros_like(s["q"])
    for first, count, slot, prefix in s["seqs"].tolist():
        n = prefix + count
        words = s["mask"][first : first + count].long() & 0xFFFFFFFF
        bits = ((words[:, :, None] >> torch.arange(32, device="cuda")) & 1).reshape(count, -1)[:, :count].bool()
        seen = torch.cat([torch.ones((count, prefix), dtype=torch.bool, device="cuda"), bits], 1)
        for h in range(c["heads"]):
            k, v = s["k"][slot, h // group, :n].double(), s["v"][slot, h // group, :, :n].double()
            x = s["q"][first : first + count, h].double() @ k.T * SCORE_M  # below 2^53
            x = torch.floor((x + 2.0 ** (WEIGHT_OF[c["width"]] - 1)) * 2.0 ** -WEIGHT_OF[c["width"]])
            x = torch.where(seen, x, -torch.inf)
            d = torch.where(seen, (x.max(1, keepdim=True).values - x).clamp(max=LAST), 0).long()
            e = torch.where(seen, table[d], 0)
            p = ((e.long() << SOFTMAX_P) // e.long().sum(1, keepdim=True)).double()
            acc = (p @ v.T).long().cpu().numpy().astype(object)
            y = np.floor_divide(acc * OUT_M + (1 << (OUT_S - 1)), 1 << OUT_S)
            out[first : first + count, h] = torch.from_numpy(np.clip(y, -127, 127).astype(np.int8)).cuda()
    return out


def exact_beam(s):
    c = s["case"]
    table, squared = LOGIT_TABLE, 1 << (2 * LOGIT_EXP)
    parent, token, cost = (np.full((c["groups"], c["keep"]), NONE, np.int64) for _ in range(3))
    base, tops = s["base"].tolist(), s["tops"].cpu().numpy()
    for g in range(c["groups"]):
        found = []
        for b in range(c["beams"]):
            row = g * c["beams"] + b
            off = np.repeat(tops[row].max() - tops[row], 128)[: c["vocab"]]
            d = np.minimum(off + s["dist"][row, : c["vocab"]].cpu().numpy(), LAST)
            total = int(table[d].sum())
            norm = sum(1 for t in np.unique(table[table > squared // total]) for _ in range(int((table == t).sum()))
                       if int(t) * total > squared)
            near = np.lexsort((np.arange(c["vocab"]), d))[: c["keep"]]
            found += [(base[row] + norm + int(d[i]), b, int(i)) for i in near if d[i] <= LAST_WEIGHT]
        for i, (x, b, t) in enumerate(sorted(found)[: c["keep"]]):
            parent[g, i], token[g, i], cost[g, i] = b, t, x
    return {"parent": torch.from_numpy(parent).int(), "token": torch.from_numpy(token).int(),
            "cost": torch.from_numpy(cost)}


def exact_reorder(s):
    c = s["case"]
    k, v = s["k"].clone(), s["v"].clone()
    slots, parents = s["slots"].tolist(), s["parent"].tolist()
    for g in range(c["groups"]):
        for b in range(c["beams"]):
            to, of = slots[g * c["beams"] + b], slots[g * c["beams"] + parents[g][b]]
            k[to, :, : c["rows"]] = s["k"][of, :, : c["rows"]]
            v[to, :, :, : c["rows"]] = s["v"][of, :, :, : c["rows"]]
    return {"k": k, "v": v}


def exact_commit(s):
    k, v = s["k"].clone(), s["v"].clone()
    for (_, _, slot, prefix), path, n in zip(s["seqs"].tolist(), s["path"].tolist(), s["length"].tolist()):
        for j, i in enumerate(path[:n]):
            k[slot, :, prefix + j] = s["k"][slot, :, prefix + i]
            v[slot, :, :, prefix + j] = s["v"][slot, :, :, prefix + i]
    return {"k": k, "v": v}


def exact(case, seed):
    if case["op"] == "tree" and case["n_seq"] * case["heads"] > 1500 or \
            case["op"] == "beam" and case["groups"] * case["beams"] > 700:
        return None
    return {"tree": exact_tree, "beam": exact_beam, "reorder": exact_reorder, "commit": exact_commit}[case["op"]](
        prepare(case, seed))
