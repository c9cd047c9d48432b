"""What the draft operators' documentation promises around the results: entries that are left out, calls
beside one another, and the first and last blocks of a launch. Plain 64-bit implementations as in
test_gpu_draft_ops.py; whole numbers, always equal."""

from __future__ import annotations

import numpy as np
import pytest

import tests.draft_ref as R
from taco_b200 import backend as B
from taco_b200 import synth
from tests.test_gpu_draft_ops import (RULE, beam_case, check_tree, dev, gpu, run_beam, tree_case, tree_op,  # noqa: F401
                                      want_tree)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# ---- tree attention ----


def bad_reorder(dev):
    """A call whose parent is out of range: it sets the handle's error word and moves nothing."""
    z = torch.zeros((2, 1, 16, 16), dtype=torch.int8, device="cuda")
    ids = torch.tensor([1, 9], dtype=torch.int32, device="cuda")
    B.CacheReorder(dev, B.KvCache(z, z.clone(), 2, 1, 16, 16), 1, 2, ids, torch.zeros_like(ids)).run()


def many_trees(seed, n, most, n_ctx, heads):
    """More (tree, head) pairs than the GPU has blocks."""
    r = np.random.default_rng(seed)
    counts = [int(x) for x in r.integers(1, most + 1, n)]
    counts[0] = most
    prefixes = [int(r.integers(n_ctx // 2, n_ctx - most + 1)) for _ in counts]
    prefixes[0] = n_ctx - most
    return tree_case(seed, counts, prefixes, n_ctx, heads=heads, kv=heads)


@pytest.mark.parametrize("n,most,n_ctx,heads", [(45, 20, 512, 4), (15, 20, 1024, 12), (15, 20, 1040, 12), (45, 16, 512, 4)])
def test_trees_beside_an_unreported_error(dev, n, most, n_ctx, heads):
    """An error that nobody has asked about yet changes nothing for later calls on the handle."""
    c = many_trees(71, n, most, n_ctx, heads)
    op, out, h = tree_op(dev, c)
    bad_reorder(dev)
    want = want_tree(c)
    for _ in range(5):
        out.fill_(99)
        op.run(0)
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy(), want)
    with pytest.raises(B.HardShellError, match="a beam's parent"):
        dev.check()
    dev.check()
    h.close()


@pytest.mark.parametrize("n,most,n_ctx,heads", [(45, 20, 512, 4), (15, 20, 1024, 12), (45, 16, 512, 4)])
def test_bad_records_among_more_trees_than_blocks(dev, n, most, n_ctx, heads):
    """Records that are not valid, the first among them: every other tree has its outputs."""
    c = many_trees(72, n, most, n_ctx, heads)
    want = want_tree(c)
    for i in (0, n // 3, n - 1):
        first, count = c["seqs"][i, :2]
        want[first:first + count] = 99
        c["seqs"][i, 2] = n  # no such slot
    op, out, h = tree_op(dev, c)
    for _ in range(5):
        out.fill_(99)
        op.run(0)
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy(), want)
    with pytest.raises(B.HardShellError, match="a tree's rows"):
        dev.check()
    dev.check()
    h.close()


@pytest.mark.parametrize("counts,prefixes,n_ctx,hd", [([20], [300], 512, 64), ([20], [1100], 2048, 64), ([9], [600], 1024, 128),
                                                     ([9], [400], 512, 128), ([9], [90], 256, 64)])
@pytest.mark.parametrize("score_m", [2**31 - 1, -2**31 + 1])
@pytest.mark.parametrize("score_s", [31, 32, 48, 51, 52, 53, 54, 61, 62, 63])
def test_tree_scores_of_large_shifts(dev, counts, prefixes, n_ctx, hd, score_m, score_s):
    """The distance in one multiply-add, up to the largest shift, with dots at their extremes."""
    c = tree_case(77, counts, prefixes, n_ctx, hd=hd)
    r = np.random.default_rng(78)
    for name in ("q", "k"):
        c[name][...] = np.where(r.random(c[name].shape[:-1] + (1,)) < 0.5, -128, 127)
    check_tree(dev, c, dict(RULE, score_m=score_m, score_s=score_s, table=np.arange(200, 0, -1)))


# ---- beam selection ----


@pytest.mark.parametrize("alive", [(), (0,), (7,), (3, 4)])
@pytest.mark.parametrize("groups,vocab", [(1, 300), (18, 300), (150, 700)])
def test_beams_that_take_no_time(dev, alive, groups, vocab):
    """Beams that are dead or have ended reach the first block of their cluster at once, whenever it starts:
    one launch after another, each with other blocks that are quick."""
    r = np.random.default_rng(groups + sum(alive))
    c = beam_case(70, groups, 8, vocab)
    c["finished"] = r.integers(0, 2, groups * 8)
    c["base"] = np.where(r.random(groups * 8) < 0.3, -1, c["base"])
    for b in alive:
        c["finished"][b::8], c["base"][b::8] = 0, r.integers(0, 200, groups)
    want = R.beam_select(c["dist"], c["tops"], 7, vocab, 8, 8, c["base"], c["finished"], c["table"])
    rule = B.WeightRule(dev, c["table"])
    dist, tops, base, fin = gpu(c["dist"]), gpu(c["tops"]), gpu(c["base"]), gpu(c["finished"], np.uint8)
    outs = [[torch.full((groups, 8), 7, dtype=t, device="cuda") for t in (torch.int32, torch.int32, torch.int64)]
            for _ in range(20)]
    ops = [B.BeamSelect(rule, dist, tops, vocab, groups, 8, 8, base, *o, fin) for o in outs]
    torch.cuda.synchronize()
    for op in ops:
        op.run(0)
    dev.check()
    for o in outs:
        for got, x in zip(o, want):
            assert np.array_equal(got.cpu().numpy(), x)
    rule.close()


@pytest.mark.parametrize("ended", [0, 1])
@pytest.mark.parametrize("vocab,beams,alive", [(50257, 16, 8), (3000, 32, 5), (1024, 20, 1)])
def test_the_logits_of_dead_and_finished_beams_need_not_be_there(dev, ended, vocab, beams, alive):
    """The last beams of the last group have ended (or are dead), and the distances end, with their allocation,
    at the last living beam's."""
    c = beam_case(73, 1, beams, vocab)
    c["finished"] = np.where(np.arange(beams) < alive, 0, 1) if ended else None
    c["base"][alive:] = 77 if ended else -1
    want = R.beam_select(c["dist"], c["tops"], 7, vocab, beams, beams, c["base"], c["finished"], c["table"])
    ld = c["dist"].shape[1]
    whole = torch.zeros(16 << 20, dtype=torch.int16, device="cuda")  # an allocation of its own
    dist = whole[whole.numel() - alive * ld:].view(alive, ld)
    dist.copy_(gpu(c["dist"][:alive]))
    rule = B.WeightRule(dev, c["table"])
    parent, token = (torch.zeros((1, beams), dtype=torch.int32, device="cuda") for _ in range(2))
    cost = torch.zeros((1, beams), dtype=torch.int64, device="cuda")
    fin = None if c["finished"] is None else gpu(c["finished"], np.uint8)
    op = B.BeamSelect(rule, dist.data_ptr(), gpu(c["tops"]), vocab, 1, beams, beams, gpu(c["base"]), parent, token, cost,
                      fin, ld, c["tops"].shape[1])
    torch.cuda.synchronize()
    for _ in range(3):
        op.run(0)
    dev.check()
    for got, x in zip((parent, token, cost), want):
        assert np.array_equal(got.cpu().numpy(), x)
    rule.close()


@pytest.mark.parametrize("low", [1, 2, 300, 511])
@pytest.mark.parametrize("length", [1, 31, 33, 1025, 16000])
def test_beam_entries_of_one_value(dev, length, low):
    """Many equal entries that only the low bits of their value let pass."""
    vocab, top = 1000, 1 << 40
    c = beam_case(75, 3, 2, vocab)
    c["dist"][:, :vocab] = 0
    c["tops"][...] = 0
    border = top // vocab  # (entries above it pass, as every weight of the rows is the first)
    for value in (border, border + 1, (border >> 9 << 9) + low):
        c["table"] = np.array([top] + [value] * length + [3, 2, 1, 0])
        want = R.norm_of([int(x) for x in c["table"]], vocab * top)
        assert want == (1 + length if value > border else 1)
        got = run_beam(dev, c, 2)[2].reshape(3, 2)
        assert np.array_equal(got, np.sort((c["base"][:, None] + want + np.zeros(2, np.int64)).reshape(3, 4), 1)[:, :2])


def test_beam_time_of_entries_of_one_value(dev):
    """A table with a long run of one value costs what any other of its length does (the run was walked entry by
    entry, a read from global memory each: thousands of them against a few)."""
    vocab, top, n = 1000, 1 << 40, 16000
    c = beam_case(76, 1, 4, vocab)
    c["dist"][:, :vocab] = 0
    c["tops"][...] = 0
    times = []
    for step in (1000, 0):
        c["table"] = np.concatenate([[top], top // vocab + 1 - step * np.arange(n)])
        assert c["table"][-1] > 0
        rule = B.WeightRule(dev, c["table"])
        out = [torch.zeros((1, 4), dtype=t, device="cuda") for t in (torch.int32, torch.int32, torch.int64)]
        op = B.BeamSelect(rule, gpu(c["dist"]), gpu(c["tops"]), vocab, 1, 4, 4, gpu(c["base"]), *out)
        st = torch.cuda.current_stream()
        best = []
        for _ in range(7):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(10):
                op.run(st.cuda_stream)
            b.record()
            b.synchronize()
            best.append(a.elapsed_time(b))
        times.append(min(best))
        dev.check()
        rule.close()
    assert times[1] < 5 * times[0], times


# ---- moves of cache rows ----


@pytest.mark.parametrize("length", [3, 1, 40])
@pytest.mark.parametrize("n_ctx,hd", [(64, 16), (50, 20)])
def test_a_path_is_read_to_its_length(dev, length, n_ctx, hd):
    """path[i * path_stride + 0 .. lengths[i] - 1] is all there is: the last path's row, and with it the
    allocation, ends at its last entry."""
    r = np.random.default_rng(length)
    n, stride = 3, 128
    k = r.integers(-128, 128, (n, 2, n_ctx, hd)).astype(np.int8)
    v = r.integers(-128, 128, (n, 2, hd, n_ctx)).astype(np.int8)
    seqs = np.array([[0, 20, 2, 4], [20, 44, 0, 5], [64, 44, 1, 0]])
    lengths = np.array([0, 30, length])
    path = np.zeros((n, stride), np.int64)
    for i in range(n):
        path[i, :lengths[i]] = np.sort(r.permutation(seqs[i, 1])[:lengths[i]])
    want = R.commit(k, v, seqs, path, lengths)
    size = (n - 1) * stride + length
    whole = torch.zeros(8 << 20, dtype=torch.int32, device="cuda")
    whole[whole.numel() - size:] = gpu(path, np.int32).view(-1)[:size]
    dk, dv = gpu(k), gpu(v)
    B.CacheCommit(dev, B.KvCache(dk, dv, n, 2, n_ctx, hd), gpu(seqs, np.int32), n,
                  whole.data_ptr() + 4 * (whole.numel() - size), stride, gpu(lengths, np.int32)).run()
    dev.check()
    assert np.array_equal(dk.cpu().numpy(), want[0]) and np.array_equal(dv.cpu().numpy(), want[1])


@pytest.mark.parametrize("parents,fault", [([0, -1, 0], False), ([0, 5, 0], True), ([1, 0, 0], True)])
def test_reorder_of_lone_beams(dev, parents, fault):
    """Groups of one beam: nothing moves, and a parent out of range is an error as in any group."""
    r = np.random.default_rng(74)
    k = r.integers(-128, 128, (3, 2, 32, 16)).astype(np.int8)
    v = r.integers(-128, 128, (3, 2, 16, 32)).astype(np.int8)
    dk, dv = gpu(k), gpu(v)
    before = B.launch_count()
    B.CacheReorder(dev, B.KvCache(dk, dv, 3, 2, 32, 16), 3, 1, gpu(np.array(parents), np.int32),
                   gpu(np.array([4, 5, 6]), np.int32)).run()
    assert B.launch_count() == before + 1
    if fault:
        with pytest.raises(B.HardShellError, match="a beam's parent"):
            dev.check()
    dev.check()
    assert np.array_equal(dk.cpu().numpy(), k) and np.array_equal(dv.cpu().numpy(), v)


# ---- offsets past 32 bits ----

FAR = 3 << 30  # bytes from a slot to the next


@pytest.fixture(scope="module")
def far_bytes():
    """Three slots FAR apart; a test's values lie 2^30 bytes behind its keys."""
    x = torch.empty(2 * FAR + (1 << 30) + (64 << 20), dtype=torch.int8, device="cuda")
    yield x
    del x
    torch.cuda.empty_cache()


def far_cache(x, k, v):
    """The caches k, v in x, slots FAR apart, and a function that reads them back."""
    slots, planes, n_ctx, hd = k.shape
    size = planes * n_ctx * hd
    parts = [[x[at + FAR * s:][:size] for s in range(slots)] for at in (0, 1 << 30)]
    for part, y in zip(parts, (k, v)):
        for s in range(slots):
            part[s].copy_(gpu(y[s].reshape(-1)))
    cache = B.KvCache(x, x[1 << 30:], slots, planes, n_ctx, hd, FAR)
    return cache, lambda: [np.stack([p.cpu().numpy() for p in part]).reshape(y.shape) for part, y in zip(parts, (k, v))]


@pytest.mark.parametrize("counts,prefixes,n_ctx,hd", [([20, 9], [300, 80], 512, 64), ([9, 3], [90, 200], 256, 64),
                                                     ([9, 16], [1500, 30], 2048, 128), ([5, 7], [30, 20], 50, 20)])
def test_trees_of_far_slots(dev, far_bytes, counts, prefixes, n_ctx, hd):
    c = tree_case(79, counts, prefixes, n_ctx, hd=hd, slots=3)
    c["seqs"][:, 2] = [2, 1]
    cache, _ = far_cache(far_bytes, c["k"], c["v"])
    out = torch.full(c["q"].shape, 99, dtype=torch.int8, device="cuda")
    h = B.AttnRule(dev, *(RULE[n] for n in ("score_m", "score_s", "out_m", "out_s", "P", "table")))
    B.TreeAttention(h, cache, 2, 2, gpu(c["q"]), out, out.shape[0], gpu(c["seqs"]), 2, c["max_count"], c["max_keys"],
                    gpu(c["mask"]), c["mask"].shape[1]).run()
    dev.check()
    assert np.array_equal(out.cpu().numpy(), want_tree(c))
    h.close()


@pytest.mark.parametrize("n_ctx,hd", [(64, 16), (50, 20)])
def test_moves_of_far_slots(dev, far_bytes, n_ctx, hd):
    r = np.random.default_rng(80)
    k = r.integers(-128, 128, (3, 3, n_ctx, hd)).astype(np.int8)
    v = r.integers(-128, 128, (3, 3, hd, n_ctx)).astype(np.int8)
    parents, rows = np.array([[2, 0, 1]]), np.array([40, 33, 50])
    cache, back = far_cache(far_bytes, k, v)
    B.CacheReorder(dev, cache, 1, 3, gpu(parents, np.int32), gpu(rows, np.int32)).run()
    dev.check()
    k, v = R.reorder(k, v, np.arange(3), parents, rows, 3)
    for got, want in zip(back(), (k, v)):
        assert np.array_equal(got, want)
    seqs, path, lengths = np.array([[0, 30, 2, 15], [30, 9, 1, 0]]), np.array([[3, 8, 21, 29], [1, 2, 0, 0]]), np.array([4, 2])
    B.CacheCommit(dev, cache, gpu(seqs, np.int32), 2, gpu(path, np.int32), 4, gpu(lengths, np.int32)).run()
    dev.check()
    for got, want in zip(back(), R.commit(k, v, seqs, path, lengths)):
        assert np.array_equal(got, want)


@pytest.mark.parametrize("odd", [0, 1])
def test_beams_of_far_rows(dev, far_bytes, odd):
    """Rows of distances 3 GB apart, by vectors and by symbols."""
    c = beam_case(81, 1, 3, 1000)
    stride = FAR // 2 + odd
    x = far_bytes.view(torch.int16)
    for i in range(3):
        x[i * stride:][:1000].copy_(gpu(c["dist"][i, :1000]))
    rule = B.WeightRule(dev, c["table"])
    out = [torch.zeros((1, 5), dtype=t, device="cuda") for t in (torch.int32, torch.int32, torch.int64)]
    B.BeamSelect(rule, x, gpu(c["tops"]), 1000, 1, 3, 5, gpu(c["base"]), *out, dist_stride=stride).run()
    dev.check()
    want = R.beam_select(c["dist"], c["tops"], 7, 1000, 3, 5, c["base"], None, c["table"])
    for got, y in zip(out, want):
        assert np.array_equal(got.cpu().numpy(), y)
    rule.close()


# ---- a batch ----


def test_tables_after_a_truncation(dev):
    """The tables of a tree pass answer as before once its slot went back inside its context."""
    model = B.CudaModel(dev, synth.gpt2_hsm(7, shape=synth.MINI))
    batch = B.CudaBatch(model, 2, 64)
    batch.run_coded([0] * 9, range(1, 10), [0] * 9, range(1, 10))
    asks = ([0, 1, 2, 3, 3], [0, 1, 0, 0, 1], [5, 1 << 31, 9, 2, 77])
    want = batch.run_tree([0] * 4, [11, 12, 13, 14], [-1, 0, 0, 2], *asks)
    batch.truncate(0, 6)
    assert np.array_equal(batch.tree_query(*asks), want)
    batch.run_weights([], [])
    assert np.array_equal(batch.tree_query(*asks), want)
    model.close()


def test_more_queries_than_rows(dev):
    """Queries in several chunks of the batch's rows, over and over on the same nodes: each as if asked alone."""
    model = B.CudaModel(dev, synth.gpt2_hsm(7, shape=synth.MINI))
    batch = B.CudaBatch(model, 1, 16)
    r = np.random.default_rng(82)
    n = 700
    nodes, kinds = r.integers(0, 9, n), r.integers(0, 2, n)
    values = np.where(kinds == 0, r.integers(0, model.vocab_size(), n),
                      r.integers(0, 1 << 32, n))
    got = batch.run_tree([0] * 9, range(20, 29), [-1, 0, 0, 1, 2, 2, -1, 6, 7], nodes, kinds, values)
    for i in r.integers(0, n, 40).tolist() + [127, 128, 255, 256, n - 1]:
        assert batch.tree_query(nodes[i:i + 1], kinds[i:i + 1], values[i:i + 1])[0] == got[i], i
    model.close()
