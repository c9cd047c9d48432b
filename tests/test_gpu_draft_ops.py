"""The device-resident draft operators (hs_op_tree_attention, hs_op_beam_select, hs_op_cache_reorder,
hs_op_cache_commit) against plain 64-bit implementations: whole numbers, always equal."""

from __future__ import annotations

import numpy as np
import pytest

import tests.draft_ref as R
from taco_b200 import backend as B

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def exp_table(e, n, unit=256.0):
    return np.rint(2.0 ** e * np.exp(-np.arange(n) / unit)).astype(np.int64)


RULE = {"score_m": 1_346_000_000, "score_s": 35, "out_m": 1_181_116_006, "out_s": 58, "P": 30,
        "table": exp_table(30, 8192)}


@pytest.fixture(scope="module")
def dev():
    d = B.CudaDevice(0)
    yield d
    d.close()


def gpu(x, dtype=None):
    x = np.ascontiguousarray(x if dtype is None else np.asarray(x).astype(dtype))
    view = {np.dtype(np.uint32): np.int32, np.dtype(np.uint16): np.int16, np.dtype(np.uint64): np.int64}.get(x.dtype)
    return torch.from_numpy(x.view(view) if view else x).cuda()


def tree_case(seed, counts, prefixes, n_ctx, heads=2, kv=2, hd=64, planes=None, plane0=0, slots=None, spread=33.0,
              gap=0, mask_words=None):
    r = np.random.default_rng(seed)
    n = len(counts)
    planes, slots = planes or plane0 + kv, slots or n
    small = lambda *s: np.clip(np.rint(r.normal(0, spread, s)), -128, 127).astype(np.int8)  # noqa: E731
    first, rows = [], 0
    for c in counts:
        first.append(rows)
        rows += c + gap
    rows = max(rows, 1)
    words = mask_words or (max(max(counts), 1) + 31) // 32
    mask = r.integers(0, 1 << 32, (rows, words), dtype=np.uint32)  # bits past the tree: to be ignored
    for f, c in zip(first, counts):
        parents = [int(max(i - r.integers(1, 5), -1)) for i in range(c)]
        tree = R.ancestors(parents, words)
        low = np.zeros(words, np.uint32)
        for j in range(c):
            low[j >> 5] |= np.uint32(1 << (j & 31))
        mask[f:f + c] = (mask[f:f + c] & ~low) | tree
    return {"k": small(slots, planes, n_ctx, hd), "v": small(slots, planes, hd, n_ctx), "q": small(rows, heads, hd),
            "seqs": np.stack([first, counts, r.permutation(slots)[:n], prefixes], 1).astype(np.int32), "mask": mask,
            "kv": kv, "plane0": plane0, "n_ctx": n_ctx, "hd": hd,
            "max_count": max(max(counts), 1), "max_keys": max(c + p for c, p in zip(counts, prefixes))}


def run_tree(dev, c, rule=RULE, pad=0, slot_pad=0, stream=0, max_keys=None):
    rows, heads, hd = c["q"].shape
    slots, planes = c["k"].shape[:2]
    size = planes * c["n_ctx"] * hd

    def cache(x):
        flat = np.full((slots, size + slot_pad), 77, np.int8)
        flat[:, :size] = x.reshape(slots, size)
        return gpu(flat)

    q = np.full((rows, heads * hd + pad), 55, np.int8)
    q[:, :heads * hd] = c["q"].reshape(rows, -1)
    out = gpu(np.full((rows, heads * hd + pad), 99, np.int8))
    k, v, q, seqs, mask = cache(c["k"]), cache(c["v"]), gpu(q), gpu(c["seqs"]), gpu(c["mask"])
    h = B.AttnRule(dev, rule["score_m"], rule["score_s"], rule["out_m"], rule["out_s"], rule["P"], rule["table"])
    kv = B.KvCache(k, v, slots, planes, c["n_ctx"], hd, size + slot_pad if slot_pad else 0)
    op = B.TreeAttention(h, kv, heads, c["kv"], q, out, rows, seqs, len(c["seqs"]), c["max_count"],
                         max_keys or c["max_keys"], mask, c["mask"].shape[1], c["plane0"],
                         heads * hd + pad if pad else 0, heads * hd + pad if pad else 0)
    torch.cuda.synchronize()
    op.run(stream)
    dev.check(stream)
    got = out.cpu().numpy()
    h.close()
    assert (got[:, heads * hd:] == 99).all()
    return got[:, :heads * hd].reshape(rows, heads, hd)


def want_tree(c, rule=RULE):
    return R.tree_attention(c["k"], c["v"], c["q"], c["seqs"], c["mask"], rule, c["kv"], c["plane0"],
                            np.full(c["q"].shape, 99, np.int8))


def check_tree(dev, c, rule=RULE, **kw):
    assert np.array_equal(run_tree(dev, c, rule, **kw), want_tree(c, rule))


@pytest.mark.parametrize("counts,prefixes,n_ctx", [
    ([1], [0], 16), ([1], [1], 16), ([2], [14], 16), ([7], [0], 48), ([16], [1], 64), ([17], [111], 128),
    ([16], [112], 128), ([5, 16, 1], [3, 100, 127], 128), ([64], [960], 1024), ([128], [0], 128), ([128], [896], 1024),
    ([33, 12], [500, 1012], 1024), ([31], [8161], 8192), ([1, 1, 1], [0, 255, 256], 512), ([9], [1015], 1040),
    ([100], [1100], 2048), ([127], [2000], 4096)])
def test_tree_sizes(dev, counts, prefixes, n_ctx):
    check_tree(dev, tree_case(1, counts, prefixes, n_ctx))


@pytest.mark.parametrize("hd", [16, 20, 24, 32, 48, 64, 80, 96, 128, 256])
@pytest.mark.parametrize("n_ctx", [64, 50])
def test_tree_head_widths(dev, hd, n_ctx):
    check_tree(dev, tree_case(2, [5, 9], [40, 7], n_ctx, hd=hd))


@pytest.mark.parametrize("heads,kv,plane0,planes", [(1, 1, 0, 1), (3, 3, 2, 9), (4, 2, 1, 4), (12, 4, 0, 4), (8, 1, 3, 4),
                                                    (32, 2, 0, 2)])
@pytest.mark.parametrize("hd", [64, 128, 16])
def test_tree_shared_heads(dev, heads, kv, plane0, planes, hd):
    check_tree(dev, tree_case(3, [6, 21], [70, 100], 128, heads, kv, hd, planes, plane0))


@pytest.mark.parametrize("score_m,score_s", [
    (1_346_000_000, 16), (1_346_000_000, 21), (1_346_000_000, 22), (1_346_000_000, 31), (1_346_000_000, 32),
    (1_346_000_000, 33), (1_346_000_000, 40), (1_346_000_000, 62), (1_346_000_000, 63), (1_346_000_000, 96),
    (-1_346_000_000, 35), (-1_346_000_000, 20), (-2**31, 32), (2**31 - 1, 0), (5, 0), (0, 35), (0, 0), (77, 10)])
@pytest.mark.parametrize("hd", [64, 128, 24])
def test_tree_score_rules(dev, score_m, score_s, hd):
    check_tree(dev, tree_case(4, [18], [60], 96, hd=hd), dict(RULE, score_m=score_m, score_s=score_s))


@pytest.mark.parametrize("table", [exp_table(30, 1), exp_table(30, 7, 2.0), np.zeros(5, np.int64),
                                   np.full(8192, 2**31 - 1, np.int64), exp_table(12, 3000), exp_table(3, 8191, 900.0),
                                   np.array([0, 0, 5, 7, 0]), np.array([1])])
@pytest.mark.parametrize("P", [0, 13, 30])
@pytest.mark.parametrize("hd", [64, 16])
def test_tree_tables_and_precisions(dev, table, P, hd):
    out_s = max(0, 58 - 30 + P)
    check_tree(dev, tree_case(5, [11], [200], 256, hd=hd), dict(RULE, table=table, P=P, out_s=out_s))


@pytest.mark.parametrize("out_m,out_s", [(0, 58), (-1_181_116_006, 58), (2**31 - 1, 0), (-2**31, 20), (1 << 30, 95),
                                         (1 << 30, 96), (1 << 30, 60), (1, 31), (3, 32)])
def test_tree_output_rules(dev, out_m, out_s):
    check_tree(dev, tree_case(6, [20], [150], 192), dict(RULE, out_m=out_m, out_s=out_s))


@pytest.mark.parametrize("hd", [64, 128, 16])
def test_tree_extreme_values(dev, hd):
    c = tree_case(7, [16, 3], [100, 900], 1024, hd=hd)
    for name in ("q", "k", "v"):
        c[name][...] = np.where(np.random.default_rng(8).random(c[name].shape) < 0.5, -128, 127)
    check_tree(dev, c, dict(RULE, score_m=2**31 - 1, score_s=32))
    for name in ("q", "k", "v"):
        c[name][...] = -128
    check_tree(dev, c)
    check_tree(dev, c, dict(RULE, score_m=-2**31, score_s=22))


@pytest.mark.parametrize("hd", [64, 16])
def test_tree_rows_that_see_nothing(dev, hd):
    c = tree_case(9, [10, 16, 4], [0, 30, 0], 64, hd=hd)
    c["mask"][:3] = 0          # no context, no node
    c["mask"][10:14] = 0       # the context alone
    c["mask"][26:30] = 0       # a whole tree that sees nothing
    got = run_tree(dev, c)
    assert np.array_equal(got, want_tree(c))
    assert (got[:3] == 0).all() and (got[26:30] == 0).all()


@pytest.mark.parametrize("hd", [64, 128, 20])
def test_tree_any_mask(dev, hd):
    """Masks that are no trees: any set of nodes, later ones among them."""
    c = tree_case(10, [128, 40, 1], [70, 3, 9], 256, hd=hd)
    c["mask"][...] = np.random.default_rng(11).integers(0, 1 << 32, c["mask"].shape, dtype=np.uint32)
    check_tree(dev, c)


def test_tree_mask_wider_than_needed_and_loose_bounds(dev):
    c = tree_case(12, [5, 30], [100, 20], 512, mask_words=9)
    c["max_count"] = 77
    check_tree(dev, c, max_keys=512)


@pytest.mark.parametrize("pad,slot_pad", [(16, 16), (4, 0), (1, 0), (0, 48), (48, 7), (8, 64)])
@pytest.mark.parametrize("hd", [64, 16])
def test_tree_strides(dev, pad, slot_pad, hd):
    check_tree(dev, tree_case(13, [12, 7], [33, 90], 128, hd=hd), pad=pad, slot_pad=slot_pad)


def test_tree_rows_of_no_tree_and_empty_trees(dev):
    c = tree_case(14, [6, 0, 9], [50, 20, 0], 64, gap=3)
    check_tree(dev, c)


def test_tree_many_sequences(dev):
    r = np.random.default_rng(15)
    counts = r.integers(1, 20, 300).tolist()
    check_tree(dev, tree_case(15, counts, r.integers(0, 100, 300).tolist(), 128, heads=3, kv=3))


def test_tree_of_many_keys_and_sequences(dev):
    """More (sequence, head) pairs than the GPU holds at once, with the key axis split."""
    r = np.random.default_rng(16)
    counts = r.integers(1, 34, 24).tolist()
    pre = r.integers(0, 2000, 24)
    pre[0] = 2048 - 33
    check_tree(dev, tree_case(16, counts, [min(int(p), 2048 - c) for p, c in zip(pre, counts)], 2048, heads=12, kv=12))


@pytest.mark.parametrize("counts,prefixes,n_ctx", [([40, 9], [900, 20], 1024), ([33], [2000], 2048), ([5], [700], 1024)])
def test_tree_table_that_changes_to_its_end(dev, counts, prefixes, n_ctx):
    """8,192 different entries: no shared memory is left for the copies of keys and values."""
    table = (1 << 30) - 100_000 * np.arange(8192, dtype=np.int64)
    check_tree(dev, tree_case(54, counts, prefixes, n_ctx), dict(RULE, table=table))


@pytest.mark.parametrize("seed", range(8))
def test_tree_random_batches(dev, seed):
    """Ragged batches of every size of context, with empty trees and heads shared or not."""
    r = np.random.default_rng(1000 + seed)
    n_ctx = int(r.choice([512, 1024, 1040, 2048, 4096]))
    kv, group = int(r.integers(1, 4)), int(r.choice([1, 1, 2, 5]))
    counts = [int(c) for c in r.integers(0, int(r.choice([5, 17, 60, 129])), 9)]
    counts[0] = max(counts[0], 1)
    prefixes = [int(r.integers(0, n_ctx - c + 1)) for c in counts]
    prefixes[0] = n_ctx - counts[0]
    check_tree(dev, tree_case(2000 + seed, counts, prefixes, n_ctx, kv * group, kv, gap=int(r.integers(0, 2))),
               pad=int(r.choice([0, 16])))


def test_tree_on_a_side_stream_and_in_a_graph(dev):
    c = tree_case(17, [16, 5], [100, 30], 128)
    st = torch.cuda.Stream()
    check_tree(dev, c, stream=st.cuda_stream)
    want = want_tree(c)
    k, v, q, seqs, mask = gpu(c["k"]), gpu(c["v"]), gpu(c["q"]), gpu(c["seqs"]), gpu(c["mask"])
    out = torch.full(c["q"].shape, 99, dtype=torch.int8, device="cuda")
    h = B.AttnRule(dev, *(RULE[n] for n in ("score_m", "score_s", "out_m", "out_s", "P", "table")))
    op = B.TreeAttention(h, B.KvCache(k, v, 2, 2, 128, 64), 2, 2, q, out, q.shape[0], seqs, 2, 16, 116, mask, 1)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        op.run(torch.cuda.current_stream().cuda_stream)
    assert (out == 99).all()
    for _ in range(2):
        out.fill_(99)
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy(), want)
    # New records in the captured buffers: the replay reads them.
    c["seqs"][:, 3] = [7, 12]
    seqs.copy_(gpu(c["seqs"]))
    g.replay()
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(), want_tree(c))
    dev.check()


@pytest.mark.parametrize("at,value", [(0, 14), (1, 17), (2, 2), (3, 113), (3, -1), (0, -5), (1, -1), (2, 1 << 30)])
@pytest.mark.parametrize("hd", [64, 16])
def test_tree_bad_record_is_left_out(dev, at, value, hd):
    c = tree_case(18, [12, 16], [40, 100], 128, hd=hd)
    want = want_tree(c)
    bad = {k: (x.copy() if isinstance(x, np.ndarray) else x) for k, x in c.items()}
    bad["seqs"][1, at] = value
    with pytest.raises(B.HardShellError, match="a tree's rows") as e:
        run_tree(dev, bad, max_keys=116)
    assert e.value.code == B.HS_BAD_ARGUMENT
    dev.check()  # the word is cleared
    del want


# ---- beam selection ----


def beam_case(seed, groups, beams, vocab, spread=300.0, tile_shift=7, ld=None, table_len=2048, far=None):
    r = np.random.default_rng(seed)
    rows, tile = groups * beams, 1 << tile_shift
    tiles = (vocab + tile - 1) // tile
    logits = np.rint(r.normal(0, spread, (rows, vocab))).astype(np.int64) + int(r.integers(-10**6, 10**6))
    padded = np.full((rows, tiles * tile), -10**12, np.int64)
    padded[:, :vocab] = logits
    tops = padded.reshape(rows, tiles, tile).max(2)
    d = np.minimum(np.repeat(tops, tile, 1)[:, :vocab] - logits, far or table_len - 1)
    dist = r.integers(0, 1 << 16, (rows, ld or (vocab + 255) // 256 * 256)).astype(np.uint16)  # junk past the row
    dist[:, :vocab] = d
    return {"dist": dist, "tops": tops, "vocab": vocab, "groups": groups, "beams": beams, "tile_shift": tile_shift,
            "base": r.integers(0, 200, rows).astype(np.int64), "finished": None,
            "table": exp_table(40, table_len, 100.0)}


def run_beam(dev, c, keep, stream=0, shift=0):
    rule = B.WeightRule(dev, c["table"])
    n = (c["groups"], keep)
    parent, token = (torch.full(n, 7, dtype=torch.int32, device="cuda") for _ in range(2))
    cost = torch.full(n, 7, dtype=torch.int64, device="cuda")
    flat = np.zeros(c["dist"].size + shift, np.uint16)
    flat[shift:] = c["dist"].reshape(-1)
    dist = gpu(flat)
    fin = None if c["finished"] is None else gpu(c["finished"], np.uint8)
    tops = gpu(c["tops"])
    op = B.BeamSelect(rule, dist.data_ptr() + 2 * shift, tops, c["vocab"], c["groups"], c["beams"], keep,
                      gpu(c["base"]), parent, token, cost, fin, c["dist"].shape[1], c["tops"].shape[1],
                      c["tile_shift"])
    torch.cuda.synchronize()
    op.run(stream)
    dev.check(stream)
    rule.close()
    return [x.cpu().numpy().astype(np.int64) for x in (parent, token, cost)]


def check_beam(dev, c, keep, **kw):
    want = R.beam_select(c["dist"], c["tops"], c["tile_shift"], c["vocab"], c["beams"], keep, c["base"], c["finished"],
                         c["table"])
    got = run_beam(dev, c, keep, **kw)
    for a, b, name in zip(got, want, ("parent", "token", "cost")):
        assert np.array_equal(a, b), name


@pytest.mark.parametrize("vocab", [2, 3, 63, 64, 127, 128, 129, 300, 1000, 4099, 16384])
@pytest.mark.parametrize("groups,beams,keep", [(1, 1, 1), (1, 4, 4), (3, 5, 7), (2, 8, 16)])
def test_beam_sizes(dev, vocab, groups, beams, keep):
    check_beam(dev, beam_case(21, groups, beams, vocab), keep)


@pytest.mark.parametrize("groups,beams,keep,vocab", [(1, 2, 3, 50257), (1, 1, 64, 50257), (1, 3, 5, 65536)])
def test_beam_large_vocabularies(dev, groups, beams, keep, vocab):
    check_beam(dev, beam_case(22, groups, beams, vocab, 500.0), keep)


@pytest.mark.parametrize("groups,beams,keep", [(1, 32, 64), (2, 32, 1), (5, 31, 33), (40, 3, 3), (1, 16, 16), (1, 17, 9)])
def test_beam_groups(dev, groups, beams, keep):
    check_beam(dev, beam_case(23, groups, beams, 700), keep)


@pytest.mark.parametrize("tile_shift", [6, 7])
@pytest.mark.parametrize("ld,shift", [(1000, 0), (1001, 0), (1008, 3), (1024, 8), (1013, 1)])
def test_beam_strides_and_alignment(dev, tile_shift, ld, shift):
    check_beam(dev, beam_case(24, 2, 3, 1000, tile_shift=tile_shift, ld=ld), 6, shift=shift)


@pytest.mark.parametrize("vocab", [600, 50257])
def test_beam_all_equal(dev, vocab):
    """Every symbol as likely as any other: the lowest symbols of the lowest beam win."""
    c = beam_case(25, 1, 2, vocab)
    c["dist"][:, :vocab] = 0
    c["tops"][...] = 5
    c["base"][:] = 3
    check_beam(dev, c, 64)
    c["base"][:] = [4, 3]
    check_beam(dev, c, 64)


def test_beam_likely_symbols_together(dev):
    """The likely symbols lie together, or at the multiples of a power of two: no luck of the order."""
    for step in (1, 2, 8, 64, 256, 512, 1024, 2048):
        c = beam_case(26, 1, 2, 50257, 30.0)
        c["dist"][:, :50257] = np.minimum(c["dist"][:, :50257].astype(np.int64) + 900, 2047)
        at = (np.arange(400) * step) % 50257
        c["dist"][:, at] = (np.arange(400) * 7 % 300).astype(np.uint16)
        c["tops"][...] = 0
        check_beam(dev, c, 64)


@pytest.mark.parametrize("table", [np.array([5]), np.array([5, 0]), np.array([1 << 40, 1, 0, 0]),
                                   np.full(300, 1 << 40), exp_table(40, 16384, 500.0), np.array([1 << 47, 1 << 20, 3])])
def test_beam_tables(dev, table):
    c = beam_case(27, 2, 3, 500, far=len(table) - 1)
    c["table"] = table
    check_beam(dev, c, 8)
    check_beam(dev, c, 64)


def test_beam_distances_past_the_table(dev):
    """Distances above the table's last entry, up to 65535, count as the last."""
    c = beam_case(28, 2, 2, 900, 4000.0, far=65535)
    check_beam(dev, c, 16)


def test_beam_extreme_maxima(dev):
    c = beam_case(29, 1, 2, 600)
    c["tops"][0, 0], c["tops"][0, 1] = 2**63 - 1, -2**63
    c["tops"][1, :] = -2**63
    check_beam(dev, c, 12)


@pytest.mark.parametrize("finished,base", [([0, 1, 0, 1], [5, 9, 300, 0]), ([1, 1, 1, 1], [4, 4, 2, 9]),
                                           ([0, 0, 0, 0], [-1, 3, 1 << 62, 0]), ([1, 0, 1, 0], [-1, -1, 5, -7]),
                                           ([0, 0, 0, 0], [-1, -1, -1, -1]), ([0, 0, 0, 0], [(1 << 62) - 1, 0, 0, 0])])
def test_beam_finished_and_dead(dev, finished, base):
    c = beam_case(30, 1, 4, 300)
    c["finished"], c["base"] = np.array(finished), np.array(base, dtype=np.int64)
    check_beam(dev, c, 5)
    check_beam(dev, c, 64)


def test_beam_few_candidates(dev):
    c = beam_case(31, 2, 2, 40)
    c["dist"][:, :40] = 2000
    c["dist"][:, 7] = 0
    c["tops"][...] = 0
    c["table"] = exp_table(40, 2048, 20.0)  # weight 0 at 2000
    assert c["table"][2000] == 0
    check_beam(dev, c, 9)


def test_beam_in_a_graph_and_on_a_stream(dev):
    c = beam_case(32, 3, 4, 1000)
    check_beam(dev, c, 4, stream=torch.cuda.Stream().cuda_stream)
    rule = B.WeightRule(dev, c["table"])
    parent, token = (torch.zeros((3, 4), dtype=torch.int32, device="cuda") for _ in range(2))
    cost = torch.zeros((3, 4), dtype=torch.int64, device="cuda")
    dist, tops, base = gpu(c["dist"]), gpu(c["tops"]), gpu(c["base"])
    op = B.BeamSelect(rule, dist, tops, 1000, 3, 4, 4, base, parent, token, cost)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        op.run(torch.cuda.current_stream().cuda_stream)
    for add in (0, 50):
        base += add
        c["base"] += add
        g.replay()
        torch.cuda.synchronize()
        want = R.beam_select(c["dist"], c["tops"], 7, 1000, 4, 4, c["base"], None, c["table"])
        for a, b in zip((parent, token, cost), want):
            assert np.array_equal(a.cpu().numpy(), b)


# ---- moves of cache rows ----


def cache_case(seed, slots, planes, n_ctx, hd):
    r = np.random.default_rng(seed)
    return (r.integers(-128, 128, (slots, planes, n_ctx, hd)).astype(np.int8),
            r.integers(-128, 128, (slots, planes, hd, n_ctx)).astype(np.int8), r)


@pytest.mark.parametrize("n_ctx,hd", [(64, 16), (64, 64), (50, 16), (64, 20), (33, 7), (1024, 64)])
@pytest.mark.parametrize("groups,beams", [(1, 2), (3, 4), (2, 7), (1, 16), (2, 32)])
def test_reorder(dev, n_ctx, hd, groups, beams):
    slots, planes = groups * beams + 3, 3
    k, v, r = cache_case(41, slots, planes, n_ctx, hd)
    ids = r.permutation(slots)[:groups * beams]
    for kind in ("any", "swap", "one", "none", "cycle"):
        parents = np.tile(np.arange(beams), (groups, 1))
        if kind == "any":
            parents = r.integers(0, beams, (groups, beams))
        elif kind == "swap":
            parents = parents[:, ::-1]
        elif kind == "one":
            parents[:] = beams - 1
        elif kind == "cycle":
            parents = (parents + 1) % beams
            parents[0, 0] = -1  # no move
        rows = r.integers(0, n_ctx + 1, groups * beams)
        rows[0], rows[-1] = n_ctx, 0
        want = R.reorder(k, v, ids, parents, rows, beams)
        dk, dv = gpu(k), gpu(v)
        B.CacheReorder(dev, B.KvCache(dk, dv, slots, planes, n_ctx, hd), groups, beams, gpu(parents, np.int32),
                       gpu(rows, np.int32), gpu(ids, np.int32)).run()
        dev.check()
        assert np.array_equal(dk.cpu().numpy(), want[0]) and np.array_equal(dv.cpu().numpy(), want[1]), kind


@pytest.mark.parametrize("slot_pad,shift", [(16, 0), (5, 0), (0, 16), (0, 1)])
def test_reorder_identity_slots_strides_and_alignment(dev, slot_pad, shift):
    slots, planes, n_ctx, hd = 6, 2, 48, 32
    k, v, r = cache_case(42, slots, planes, n_ctx, hd)
    size = planes * n_ctx * hd

    def flat(x):
        f = np.full(shift + slots * (size + slot_pad), 55, np.int8)
        f[shift:].reshape(slots, -1)[:, :size] = x.reshape(slots, size)
        return f

    parents, rows = r.integers(0, 3, (2, 3)), r.integers(0, n_ctx + 1, 6)
    want = R.reorder(k, v, np.arange(6), parents, rows, 3)
    dk, dv = gpu(flat(k)), gpu(flat(v))
    B.CacheReorder(dev, B.KvCache(dk.data_ptr() + shift, dv.data_ptr() + shift, slots, planes, n_ctx, hd,
                                  size + slot_pad), 2, 3, gpu(parents, np.int32), gpu(rows, np.int32)).run()
    dev.check()
    assert np.array_equal(dk.cpu().numpy(), flat(want[0])) and np.array_equal(dv.cpu().numpy(), flat(want[1]))


@pytest.mark.parametrize("what,value", [("parent", 3), ("parent", -2), ("slot", 6), ("slot", -1), ("rows", 49)])
def test_reorder_bad_entries_are_left_out(dev, what, value):
    slots, planes, n_ctx, hd = 6, 2, 48, 16
    k, v, _ = cache_case(43, slots, planes, n_ctx, hd)
    parents, rows, ids = np.array([[1, 2, 0], [0, 0, 0]]), np.full(6, 30), np.arange(6)
    good = parents.copy()
    if what == "parent":
        parents[0, 1], good[0, 1] = value, 1
    elif what == "slot":
        ids[3], good[1, :] = value, [0, 1, 2]  # the source of the second group
    else:
        rows[3], good[1, :] = value, [0, 1, 2]
    want = R.reorder(k, v, np.arange(6), good, np.full(6, 30), 3)
    dk, dv = gpu(k), gpu(v)
    B.CacheReorder(dev, B.KvCache(dk, dv, slots, planes, n_ctx, hd), 2, 3, gpu(parents, np.int32), gpu(rows, np.int32),
                   gpu(ids, np.int32)).run()
    with pytest.raises(B.HardShellError, match="a beam's parent"):
        dev.check()
    assert np.array_equal(dk.cpu().numpy(), want[0]) and np.array_equal(dv.cpu().numpy(), want[1])


@pytest.mark.parametrize("n_ctx,hd", [(160, 16), (160, 64), (131, 16), (144, 20), (160, 7), (1024, 64), (256, 128)])
def test_commit(dev, n_ctx, hd):
    slots, planes = 9, 3
    k, v, r = cache_case(44, slots, planes, n_ctx, hd)
    counts = np.array([1, 2, 16, 40, 128, 128, 5])
    n = counts.size
    prefix = np.array([int(r.integers(0, n_ctx - c + 1)) for c in counts])
    prefix[4] = n_ctx - 128
    lengths = np.array([1, 1, 7, 33, 128, 90, 0])
    path = np.full((n, 128), -3, np.int64)
    for i in range(n):
        path[i, :lengths[i]] = np.sort(r.permutation(counts[i])[:lengths[i]])
    seqs = np.stack([np.cumsum(counts) - counts, counts, r.permutation(slots)[:n], prefix], 1)
    want = R.commit(k, v, seqs, path, lengths)
    dk, dv = gpu(k), gpu(v)
    B.CacheCommit(dev, B.KvCache(dk, dv, slots, planes, n_ctx, hd), gpu(seqs, np.int32), n, gpu(path, np.int32), 128,
                  gpu(lengths, np.int32)).run()
    dev.check()
    assert np.array_equal(dk.cpu().numpy(), want[0]) and np.array_equal(dv.cpu().numpy(), want[1])


@pytest.mark.parametrize("path,length,seq", [([0, 2, 2], 3, None), ([3, 1, 4], 3, None), ([0, 1, 5], 3, None),
                                             ([0, 1, -1], 3, None), ([0, 1, 2], 4, None), ([0, 1, 2], -1, None),
                                             ([0, 1, 2], 3, [0, 5, 2, 10]), ([0, 1, 2], 3, [0, 5, 1, 60]),
                                             ([0, 1, 2], 3, [0, 129, 1, 0])])
def test_commit_bad_paths_are_left_out(dev, path, length, seq):
    k, v, _ = cache_case(45, 2, 2, 64, 16)
    seqs = np.array([seq or [0, 5, 1, 10], [5, 4, 0, 20]])
    paths, lengths = np.array([path, [1, 2, 3]]), np.array([length, 3])
    want = R.commit(k, v, seqs[1:], paths[1:], lengths[1:])
    dk, dv = gpu(k), gpu(v)
    B.CacheCommit(dev, B.KvCache(dk, dv, 2, 2, 64, 16), gpu(seqs, np.int32), 2, gpu(paths, np.int32), 3,
                  gpu(lengths, np.int32)).run()
    with pytest.raises(B.HardShellError, match="a path is not"):
        dev.check()
    assert np.array_equal(dk.cpu().numpy(), want[0]) and np.array_equal(dv.cpu().numpy(), want[1])


def test_moves_in_graphs(dev):
    k, v, r = cache_case(46, 4, 2, 64, 32)
    dk, dv = gpu(k), gpu(v)
    cache = B.KvCache(dk, dv, 4, 2, 64, 32)
    parents, rows, ids = np.array([[1, 0, 3, 3]]), np.array([10, 20, 30, 64]), np.arange(4)
    seqs, path, lengths = np.array([[0, 8, 2, 30]]), np.array([[1, 3, 6]]), np.array([3])
    keep = [gpu(x, np.int32) for x in (parents, rows, ids, seqs, path, lengths)]
    a = B.CacheReorder(dev, cache, 1, 4, keep[0], keep[1], keep[2])
    b = B.CacheCommit(dev, cache, keep[3], 1, keep[4], 3, keep[5])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        st = torch.cuda.current_stream().cuda_stream
        a.run(st)
        b.run(st)
    for _ in range(3):
        g.replay()
        k, v = R.reorder(k, v, ids, parents, rows, 4)
        k, v = R.commit(k, v, seqs, path, lengths)
    torch.cuda.synchronize()
    dev.check()
    assert np.array_equal(dk.cpu().numpy(), k) and np.array_equal(dv.cpu().numpy(), v)


# ---- refusals of the host ----


def test_refusals(dev):
    c = tree_case(50, [4], [20], 64)
    k, v, q, seqs, mask = gpu(c["k"]), gpu(c["v"]), gpu(c["q"]), gpu(c["seqs"]), gpu(c["mask"])
    out = torch.zeros_like(q)
    h = B.AttnRule(dev, *(RULE[n] for n in ("score_m", "score_s", "out_m", "out_s", "P", "table")))
    good = dict(heads=2, kv_heads=2, q=q, out=out, rows=4, seqs=seqs, n_seq=1, max_count=4, max_keys=24, mask=mask,
                mask_words=1)
    cache = dict(k=k, v=v, slots=1, planes=2, n_ctx=64, head_dim=64)

    def refused(code, cache_kw=None, **kw):
        with pytest.raises(B.HardShellError) as e:
            B.TreeAttention(h, B.KvCache(**dict(cache, **(cache_kw or {}))), **dict(good, **kw)).run()
        assert e.value.code == code, str(e.value)

    B.TreeAttention(h, B.KvCache(**cache), **good).run()
    host = torch.zeros(4096, dtype=torch.int8)
    pinned = torch.zeros(4096, dtype=torch.int8).pin_memory()
    for name in ("q", "out", "seqs", "mask"):
        for bad in (None, host, pinned):
            refused(B.HS_BAD_ARGUMENT, **{name: bad})
    refused(B.HS_BAD_ARGUMENT, seqs=seqs.data_ptr() + 2)
    refused(B.HS_BAD_ARGUMENT, dict(k=host))
    refused(B.HS_BAD_ARGUMENT, dict(v=None))
    for kw in (dict(slots=0), dict(planes=0), dict(n_ctx=0), dict(n_ctx=8193), dict(head_dim=0), dict(head_dim=1025),
               dict(planes=65536), dict(slots=1 << 30)):
        refused(B.HS_UNSUPPORTED, kw)
    refused(B.HS_BAD_ARGUMENT, dict(slot_stride=100))
    refused(B.HS_UNSUPPORTED, heads=3)
    refused(B.HS_UNSUPPORTED, heads=0)
    refused(B.HS_UNSUPPORTED, kv_heads=0)
    refused(B.HS_BAD_ARGUMENT, plane0=1)
    refused(B.HS_BAD_ARGUMENT, plane0=0xFFFFFFFF)
    refused(B.HS_UNSUPPORTED, max_count=129)
    refused(B.HS_BAD_ARGUMENT, max_keys=65)
    refused(B.HS_BAD_ARGUMENT, max_keys=3)
    refused(B.HS_BAD_ARGUMENT, max_count=33, max_keys=64)
    refused(B.HS_BAD_ARGUMENT, q_stride=127)
    refused(B.HS_BAD_ARGUMENT, out_stride=1)
    dev.check()
    for args in ((1, 128, 1, 1, 30, [1]), (1, 1, 1, 128, 30, [1]), (1, 1, 1, 1, 31, [1]), (1, 1, 1, 1, 30, []),
                 (1, 1, 1, 1, 30, np.ones(8193))):
        with pytest.raises(B.HardShellError) as e:
            B.AttnRule(dev, *args)
        assert e.value.code == B.HS_UNSUPPORTED
    for rule, table in ((B.WeightRule, [0]), (B.WeightRule, [3, 4])):
        with pytest.raises(B.HardShellError) as e:
            rule(dev, table)
        assert e.value.code == B.HS_BAD_ARGUMENT
    with pytest.raises(B.HardShellError):
        B.AttnRule(dev, 1, 1, 1, 1, 30, [3, -1])
    for n in (0, 16385):
        with pytest.raises(B.HardShellError):
            B.WeightRule(dev, np.ones(n))


def test_beam_and_move_refusals(dev):
    c = beam_case(51, 1, 2, 300)
    dist, tops, base = gpu(c["dist"]), gpu(c["tops"]), gpu(c["base"])
    parent, token = (torch.zeros(4, dtype=torch.int32, device="cuda") for _ in range(2))
    cost = torch.zeros(4, dtype=torch.int64, device="cuda")
    rule = B.WeightRule(dev, c["table"])
    good = dict(dist=dist, tops=tops, vocab=300, groups=1, beams=2, keep=4, base=base, parent=parent, token=token,
                cost=cost)

    def refused(code, rule=rule, **kw):
        with pytest.raises(B.HardShellError) as e:
            B.BeamSelect(rule, **dict(good, **kw)).run()
        assert e.value.code == code, str(e.value)

    B.BeamSelect(rule, **good).run()
    for name in ("dist", "tops", "base", "parent", "token", "cost"):
        refused(B.HS_BAD_ARGUMENT, **{name: torch.zeros(600, dtype=torch.int64)})
        refused(B.HS_BAD_ARGUMENT, **{name: None})
    refused(B.HS_BAD_ARGUMENT, finished=torch.zeros(4))
    refused(B.HS_BAD_ARGUMENT, cost=cost.data_ptr() + 4)
    for kw in (dict(vocab=1), dict(vocab=65537), dict(beams=0), dict(beams=33), dict(keep=65), dict(tile_shift=5)):
        refused(B.HS_UNSUPPORTED, **kw)
    refused(B.HS_BAD_ARGUMENT, dist_stride=299)
    refused(B.HS_BAD_ARGUMENT, tops_stride=2)
    refused(B.HS_UNSUPPORTED, B.WeightRule(dev, [1 << 60, 1]))
    k, v, _ = cache_case(52, 4, 1, 16, 16)
    cache = B.KvCache(gpu(k), gpu(v), 4, 1, 16, 16)
    ids = torch.zeros(64, dtype=torch.int32, device="cuda")
    for groups, beams, code in ((1, 33, B.HS_UNSUPPORTED), (3, 2, B.HS_BAD_ARGUMENT), (1 << 31, 2, B.HS_BAD_ARGUMENT)):
        with pytest.raises(B.HardShellError) as e:
            B.CacheReorder(dev, cache, groups, beams, ids, ids).run()
        assert e.value.code == code
    with pytest.raises(B.HardShellError):
        B.CacheReorder(dev, cache, 2, 2, ids, None).run()
    with pytest.raises(B.HardShellError):
        B.CacheCommit(dev, cache, ids, 5, ids, 2, ids).run()
    with pytest.raises(B.HardShellError):
        B.CacheCommit(dev, cache, ids, 1, torch.zeros(4), 2, ids).run()
    # Nothing to do: nothing is looked at.
    B.CacheReorder(dev, cache, 0, 2, None, None).run()
    B.CacheCommit(dev, cache, None, 0, None, 0, None).run()
    dev.check()


def test_the_current_device_and_the_launch_count(dev):
    before = B.launch_count()
    c = tree_case(53, [3], [5], 16)
    run_tree(dev, c)
    assert B.launch_count() == before + 1
    assert torch.cuda.current_device() == 0


@pytest.mark.parametrize("vocab", [2, 3, 100, 1000])
def test_beam_sums_next_to_a_border(dev, vocab):
    """Weights whose low bits decide the normaliser: 32 bits of each do not, the whole ones do."""
    c = beam_case(33, 4, 2, vocab)
    c["dist"][:, :vocab] = 0
    c["tops"][...] = 0
    for low in (0, 1, 255, 511):
        top = (1 << 40) + low
        for near in (0, 1, -1):
            # table[1] * (vocab * table[0]) against table[0]^2: just below, at and above the border.
            c["table"] = np.array([top, top // vocab + near, 1, 0])
            check_beam(dev, c, 3)
    c["table"] = np.array([1 << 40] + [(1 << 40) // vocab + 2 - i for i in range(5)] + [511, 511, 3])
    c["dist"][:, :vocab] = np.random.default_rng(34).integers(0, 9, (8, vocab))
    c["dist"][:, 0] = 0
    check_beam(dev, c, 3)


def test_beam_weights_below_the_looked_up_bits(dev):
    """A row without a symbol at distance 0 whose weights are all small."""
    c = beam_case(35, 1, 2, 700)
    c["table"] = np.array([1 << 45] + [100] * 50 + [3])
    c["dist"][:, :700] = np.random.default_rng(36).integers(1, 60, (2, 700))
    c["tops"][...] = 0
    check_beam(dev, c, 20)
    c["finished"] = np.array([1, 0])
    check_beam(dev, c, 20)


# ---- the calls at the edges of what the documentation allows ----


def tree_op(dev, c):
    """The op of a case on new buffers, its outputs and the rule to close."""
    rows, heads, hd = c["q"].shape
    slots, planes = c["k"].shape[:2]
    out = torch.full(c["q"].shape, 99, dtype=torch.int8, device="cuda")
    h = B.AttnRule(dev, *(RULE[n] for n in ("score_m", "score_s", "out_m", "out_s", "P", "table")))
    op = B.TreeAttention(h, B.KvCache(gpu(c["k"]), gpu(c["v"]), slots, planes, c["n_ctx"], hd), heads, c["kv"], gpu(c["q"]),
                         out, rows, gpu(c["seqs"]), len(c["seqs"]), c["max_count"], c["max_keys"], gpu(c["mask"]),
                         c["mask"].shape[1], c["plane0"])
    torch.cuda.synchronize()
    return op, out, h


@pytest.mark.parametrize("counts,prefixes,n_ctx", [
    ([33, 20, 40], [500, 900, 12], 1024),      # several tiles a head, one block
    ([16, 9, 12], [500, 900, 300], 1024),      # one tile a head
    ([40, 16, 20], [3000, 100, 1500], 4096)])  # clusters
@pytest.mark.parametrize("bad", [0, 1, 2])
@pytest.mark.parametrize("at,value", [(0, 1 << 20), (1, 41), (2, 3), (3, -1)])
def test_tree_bad_record_keeps_its_rows_and_the_others_theirs(dev, counts, prefixes, n_ctx, bad, at, value):
    c = tree_case(60, counts, prefixes, n_ctx, gap=1)
    want = want_tree(c)
    first, count = c["seqs"][bad, :2]
    want[first:first + count] = 99
    c["seqs"][bad, at] = value
    op, out, h = tree_op(dev, c)
    op.run(0)
    with pytest.raises(B.HardShellError, match="a tree's rows"):
        dev.check(0)
    dev.check(0)
    assert np.array_equal(out.cpu().numpy(), want)
    h.close()


@pytest.mark.parametrize("n_ctx,most", [(512, 40), (512, 16), (1040, 40)])
def test_tree_works_that_follow_one_another(dev, n_ctx, most):
    """More heads than the GPU has blocks: empty trees, heads of one tile and of several in every block's turn."""
    r = np.random.default_rng(61)
    counts = [0 if i % 5 == 4 else int(r.integers(1, most + 1)) for i in range(160)]
    prefixes = [int(r.integers(0, n_ctx - most + 1)) for _ in counts]
    prefixes[0], counts[0] = n_ctx - most, most
    check_tree(dev, tree_case(61, counts, prefixes, n_ctx, heads=4, kv=4))


def test_trees_of_one_slot(dev):
    """Two drafts of one context: their records name one slot, and each sees its own nodes' cache rows."""
    c = tree_case(62, [20, 20], [300, 300], 512, slots=2)
    c["seqs"][:, 2] = 1
    check_tree(dev, c)


@pytest.mark.parametrize("counts,prefixes,n_ctx", [([40, 33], [500, 900], 1024), ([9, 16], [900, 20], 1024),
                                                   ([31, 5], [3000, 10], 4096)])
def test_two_tree_calls_at_once_and_replayed(dev, counts, prefixes, n_ctx):
    """Two streams and two graphs run the operator at once: no state of one reaches the other."""
    cases = [tree_case(63 + i, counts, prefixes, n_ctx) for i in range(2)]
    ops = [tree_op(dev, c) for c in cases]
    wants = [want_tree(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in ops]
    for _ in range(20):
        for (op, _, _), st in zip(ops, streams):
            op.run(st.cuda_stream)
    for st in streams:
        dev.check(st.cuda_stream)
    graphs = []
    for op, out, _ in ops:
        assert np.array_equal(out.cpu().numpy(), wants[len(graphs)])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            op.run(torch.cuda.current_stream().cuda_stream)
        out.fill_(99)
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for (_, out, h), want in zip(ops, wants):
        assert np.array_equal(out.cpu().numpy(), want)
        h.close()
    dev.check(0)


def test_check_of_a_captured_stream_is_refused(dev):
    c = tree_case(65, [5], [30], 64)
    op, out, h = tree_op(dev, c)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        st = torch.cuda.current_stream().cuda_stream
        op.run(st)
        with pytest.raises(B.HardShellError, match="captured") as e:
            dev.check(st)
        assert e.value.code == B.HS_BAD_ARGUMENT
    g.replay()
    dev.check(0)
    assert np.array_equal(out.cpu().numpy(), want_tree(c))
    h.close()


def test_tree_refuses_more_items_than_it_counts(dev):
    buf = torch.zeros(64, dtype=torch.int32, device="cuda")
    h = B.AttnRule(dev, *(RULE[n] for n in ("score_m", "score_s", "out_m", "out_s", "P", "table")))
    op = B.TreeAttention(h, B.KvCache(buf, buf, 1, 4096, 16, 16), 4096, 4096, buf, buf, 1, buf, 1 << 20, 1, 16, buf, 1)
    with pytest.raises(B.HardShellError, match="too many trees") as e:
        op.run(0)
    assert e.value.code == B.HS_UNSUPPORTED
    h.close()


def test_reorder_where_all_beams_take_one(dev):
    """The same parent for every beam, its own among them."""
    r = np.random.default_rng(66)
    k = r.integers(-128, 128, (8, 3, 32, 64)).astype(np.int8)
    v = r.integers(-128, 128, (8, 3, 64, 32)).astype(np.int8)
    rows = np.full(8, 29, np.uint32)
    parent = np.full(8, 5, np.uint32)
    gk, gv = gpu(k), gpu(v)
    op = B.CacheReorder(dev, B.KvCache(gk, gv, 8, 3, 32, 64), 1, 8, gpu(parent), gpu(rows))
    op.run(0)
    dev.check(0)
    wk, wv = k.copy(), v.copy()
    wk[:, :, :29] = k[5, :, :29]
    wv[:, :, :, :29] = v[5, :, :, :29]
    assert np.array_equal(gk.cpu().numpy(), wk) and np.array_equal(gv.cpu().numpy(), wv)


def test_reorder_of_every_length(dev):
    """Rows that end at every byte of a 16-byte unit; the bytes behind them stay."""
    n, beams = 48, 3
    r = np.random.default_rng(67)
    k = r.integers(-128, 128, (n * beams, 2, 48, 16)).astype(np.int8)
    v = r.integers(-128, 128, (n * beams, 2, 16, 48)).astype(np.int8)
    rows = np.repeat(np.arange(1, n + 1), beams).astype(np.uint32)
    parent = np.tile([1, 2, 1], n).astype(np.uint32)
    gk, gv = gpu(k), gpu(v)
    B.CacheReorder(dev, B.KvCache(gk, gv, n * beams, 2, 48, 16), n, beams, gpu(parent), gpu(rows)).run(0)
    dev.check(0)
    wk, wv = k.copy(), v.copy()
    for g in range(n):
        for j in range(beams):
            to, of, m = g * beams + j, g * beams + parent[g * beams + j], g + 1
            wk[to, :, :m], wv[to, :, :, :m] = k[of, :, :m], v[of, :, :, :m]
    assert np.array_equal(gk.cpu().numpy(), wk) and np.array_equal(gv.cpu().numpy(), wv)
