"""Drafts that branch on a batch (hs_batch_run_tree, hs_batch_tree_query, hs_batch_tree_commit,
hs_batch_beam_step) on a B200.

The defining property of a tree pass: the table after a node is the table of a slot that ran the
context and the node's path, bit for bit (the CPU oracle's, by its fast path). The commit leaves a slot
as if the accepted tokens had run one by one: positions, streams, histories (seen through a context
restart and a truncation) and caches. A beam step equals the definition on the oracle's weights.
Together they decode a range-coded stream: beams draft, a tree pass verifies, the path is committed.
"""

from __future__ import annotations

import numpy as np
import pytest

import tests.draft_ref as R
from oracle import oracle as O
from taco_b200 import backend as B
from taco_b200 import synth

from .common import tiny_bytes

pytestmark = pytest.mark.gpu

MODELS = {"tiny": tiny_bytes, "mini": lambda: synth.gpt2_hsm(7, shape=synth.MINI),
          "wide": lambda: synth.gpt2_hsm(7, shape=synth.MINI, wide=True)}
NONE = B.NO_TOKEN


@pytest.fixture(scope="module")
def dev():
    d = B.CudaDevice(0)
    yield d
    d.close()


@pytest.fixture(scope="module", params=list(MODELS))
def setup(request, dev):
    data = MODELS[request.param]()
    m = B.CudaModel(dev, data)
    yield m, O.Model(data)
    m.close()


@pytest.fixture(scope="module")
def mini(dev):
    data = MODELS["mini"]()
    m = B.CudaModel(dev, data)
    yield m, O.Model(data)
    m.close()


def random_tree(r, n, first=0, reach=4):
    """Parents (indices from `first`; -1: the context) of a tree of n nodes."""
    return [first + int(p) if p >= 0 else -1 for p in (max(i - int(r.integers(1, reach + 1)), -1) for i in range(n))]


def path_of(parents, i):
    out = []
    while i >= 0:
        out.append(i)
        i = parents[i]
    return out[::-1]


def oracle_weights(om, ctx, paths, overlap=0):
    """The oracle's weights after ctx + path for each path of tokens (one slot each)."""
    fb = O.FastBatch(om, len(paths), overlap)
    slots, toks, last = [], [], []
    for s, p in enumerate(paths):
        seq = list(ctx[s]) + list(p)
        slots += [s] * len(seq)
        toks += seq
        last.append(len(slots) - 1)
    out = np.zeros((len(paths), om.vocab), np.uint64)
    for s in range(len(paths)):  # one slot at a time: bounded memory
        seq = list(ctx[s]) + list(paths[s])
        out[s] = fb.run_weights([s] * len(seq), seq)[-1]
    return out


@pytest.mark.parametrize("ctx,nodes", [([0], [5]), ([1, 30, 0], [1, 16, 3]), ([40, 7], [24, 9]), ([20], [40])])
def test_tree_answers_equal_the_paths_run_one_by_one(setup, ctx, nodes):
    model, om = setup
    r = np.random.default_rng(sum(ctx) + sum(nodes))
    batch = B.CudaBatch(model, 4, 256)
    slots = r.permutation(4)[:len(ctx)].tolist()
    contexts = [r.integers(0, om.vocab, n).tolist() for n in ctx]
    for s, t in zip(slots, contexts):
        if t:
            batch.run_coded([s] * len(t), t, [0] * len(t), t)
    ns, nt, parents, starts = [], [], [], []
    for s, n in zip(slots, nodes):
        starts.append(len(ns))
        parents += random_tree(r, n, len(ns))
        ns += [s] * n
        nt += r.integers(0, om.vocab, n).tolist()
    q = r.integers(0, len(ns), 3 * len(ns))
    kinds = r.integers(0, 2, q.size)
    values = np.where(kinds == 0, r.integers(0, om.vocab, q.size), r.integers(0, 1 << 32, q.size))
    got = batch.run_tree(ns, nt, parents, q, kinds, values)
    again = batch.tree_query(q[::-1], kinds[::-1], values[::-1])[::-1]
    assert np.array_equal(got, again)
    w = oracle_weights(om, [contexts[slots.index(ns[i])] for i in range(len(ns))],
                       [[nt[j] for j in path_of(parents, i)] for i in range(len(ns))])
    for i in range(q.size):
        want = O.answer(w[q[i]], 32, int(kinds[i]), int(values[i]))
        assert (int(got[i]["symbol"]), int(got[i]["start"]), int(got[i]["freq"])) == want, i
        assert got[i]["is_last"] == (want[0] == om.vocab - 1)
    for s, t in zip(slots, contexts):
        assert batch.position(s) == len(t) and batch.stream_len(s) == len(t)


@pytest.mark.parametrize("ctx,n", [(100, 128), (384, 128), (0, 128), (511, 1), (250, 77)])
def test_large_trees(mini, ctx, n):
    model, om = mini
    r = np.random.default_rng(ctx + n)
    batch = B.CudaBatch(model, 2, 512)
    context = r.integers(0, om.vocab, ctx).tolist()
    for i in range(0, ctx, 256):
        part = context[i:i + 256]
        batch.run_coded([1] * len(part), part, [0] * len(part), part)
    parents, toks = random_tree(r, n, 0, 9), r.integers(0, om.vocab, n).tolist()
    pick = sorted({0, n - 1, n // 2, n // 3})
    got = batch.run_tree([1] * n, toks, parents, pick, [0] * len(pick), [5] * len(pick))
    w = oracle_weights(om, [context] * len(pick), [[toks[j] for j in path_of(parents, i)] for i in pick])
    for i in range(len(pick)):
        assert (int(got[i]["symbol"]), int(got[i]["start"]), int(got[i]["freq"])) == O.answer(w[i], 32, 0, 5)


def same_state(batch, a, b, om, r, n=12):
    """Slots a and b give the same answers for the next n tokens."""
    toks = r.integers(0, om.vocab, n).tolist()
    x = batch.run_coded([a] * n, toks, [0] * n, toks)
    y = batch.run_coded([b] * n, toks, [0] * n, toks)
    assert np.array_equal(x, y)
    assert batch.position(a) == batch.position(b) and batch.stream_len(a) == batch.stream_len(b)


def test_commit_leaves_the_slots_as_if_the_tokens_had_run(setup):
    model, om = setup
    r = np.random.default_rng(3)
    batch = B.CudaBatch(model, 8, 256)
    n_ctx = model.n_ctx()
    ctx = [0, 9, n_ctx - 20, 33]
    contexts = [r.integers(0, om.vocab, n).tolist() for n in ctx]
    for s, t in enumerate(contexts):
        if t:
            batch.run_coded([s] * len(t), t, [0] * len(t), t)
    for _ in range(2):
        nodes = [16, 9, 7, 20]
        ns, nt, parents, accepted = [], [], [], []
        for s, n in enumerate(nodes):
            first = len(ns)
            parents += random_tree(r, n, first)
            ns += [s] * n
            nt += r.integers(0, om.vocab, n).tolist()
            if s != 1:  # slot 1 accepts nothing
                path = path_of(parents, first + n - 1 - int(r.integers(0, 3)))
                accepted += path
                contexts[s] += [nt[j] for j in path]
        batch.run_tree(ns, nt, parents)
        batch.tree_commit(accepted)
    for s, t in enumerate(contexts):
        assert batch.position(s) == len(t) == batch.stream_len(s)
        if t:
            batch.run_coded([4 + s] * len(t), t, [0] * len(t), t)
        same_state(batch, s, 4 + s, om, r)


def test_commit_then_restart_and_truncation(mini):
    """The committed tokens are in the history (a context restart takes its overlap from it) and in the
    stream (a truncation goes back through them)."""
    model, om = mini
    r = np.random.default_rng(5)
    batch = B.CudaBatch(model, 2, 512)
    batch.set_overlap(40)
    ctx = r.integers(0, om.vocab, 480).tolist()
    parents, toks = random_tree(r, 30, 0, 2), r.integers(0, om.vocab, 30).tolist()
    path = path_of(parents, 29)
    full = ctx + [toks[j] for j in path]
    for s in range(2):
        batch.run_coded([s] * 480, ctx, [0] * 480, ctx)
    batch.run_tree([0] * 30, toks, parents)
    batch.tree_commit(path)
    tail = full[480:]
    batch.run_coded([1] * len(tail), tail, [0] * len(tail), tail)
    more = 512 - len(full) + 25  # past the end of the context
    same_state(batch, 0, 1, om, r, more)
    for keep in (500, 481, 490):
        if keep > batch.stream_len(0):
            continue
        for s in range(2):
            batch.truncate(s, keep)
        same_state(batch, 0, 1, om, r, 3)


def test_a_tree_after_a_restart_spoils_no_older_context(mini):
    """A tree pass writes cache rows behind the position, which may be the old context's: a truncation
    before the restart rebuilds them."""
    model, om = mini
    r = np.random.default_rng(6)
    batch = B.CudaBatch(model, 2, 512)
    batch.set_overlap(10)
    toks = r.integers(0, om.vocab, 530).tolist()
    for i in range(0, 530, 256):
        part = toks[i:i + 256]
        batch.run_coded([0] * len(part), part, [0] * len(part), part)
    tree = r.integers(0, om.vocab, 100).tolist()
    batch.run_tree([0] * 100, tree, random_tree(r, 100))
    batch.tree_commit([])
    assert batch.stream_len(0) == 530
    batch.truncate(0, 400)
    part = toks[:400]
    batch.run_coded([1] * 400, part, [0] * 400, part)
    same_state(batch, 0, 1, om, r)


def test_the_end_of_trees(mini):
    model, om = mini
    batch = B.CudaBatch(model, 3, 64)
    batch.run_coded([0, 0, 1], [1, 2, 3], [0] * 3, [1, 2, 3])

    def dead(code=B.HS_BAD_ARGUMENT, commit=(0,)):
        with pytest.raises(B.HardShellError) as e:
            batch.tree_commit(commit)
        assert e.value.code == code

    def tree():
        batch.run_tree([0, 0, 1], [5, 6, 7], [-1, 0, -1])

    dead()
    batch.tree_commit([])
    for end in (lambda: batch.run_coded([2], [1], [0], [1]), lambda: batch.run_weights([2], [1]),
                lambda: batch.truncate(0, 1), lambda: batch.tree_commit([]),
                lambda: batch.beam_step(1, 1, [2], [1], [0]),
                lambda: batch.decode_blocks([2], [b"\0" * 16], [1])):
        tree()
        end()
        dead()
    tree()
    batch.reset(0)
    dead(commit=(0, 1))
    batch.tree_commit([2])
    assert batch.position(1) == 2 and batch.position(0) == 0
    batch.tree_query([0, 2], [0, 0], [1, 1])  # the tables stay until rows run
    batch.run_coded([2], [1], [0], [1])
    with pytest.raises(B.HardShellError):
        batch.tree_query([0], [0], [1])


def test_tree_refusals(mini):
    model, om = mini
    batch = B.CudaBatch(model, 3, 300)
    batch.run_coded([0] * 5, [1] * 5, [0] * 5, [1] * 5)

    def refused(code, *args, **kw):
        with pytest.raises(B.HardShellError) as e:
            batch.run_tree(*args, **kw)
        assert e.value.code == code
        with pytest.raises(B.HardShellError):
            batch.tree_commit([0])

    refused(B.HS_BAD_SLOT, [3], [1], [-1])
    refused(B.HS_TOKEN_RANGE, [0], [om.vocab], [-1])
    refused(B.HS_BAD_ARGUMENT, [0], [1], [0])
    refused(B.HS_BAD_ARGUMENT, [0, 0], [1, 1], [1, -1])
    refused(B.HS_BAD_ARGUMENT, [0, 1], [1, 1], [-1, 0])        # a parent in another slot
    refused(B.HS_BAD_ARGUMENT, [0, 1, 0], [1] * 3, [-1, -1, 0])
    refused(B.HS_UNSUPPORTED, [0] * 129, [1] * 129, [-1] * 129)
    refused(B.HS_UNSUPPORTED, [0] * 100 + [1] * 100 + [2] * 101, [1] * 301, [-1] * 301)
    refused(B.HS_BAD_ARGUMENT, [0], [1], [-1], [1], [0], [0])
    refused(B.HS_UNSUPPORTED, [0], [1], [-1], [0], [0], [om.vocab])
    refused(B.HS_UNSUPPORTED, [0], [1], [-1], [0], [2], [0])
    refused(B.HS_UNSUPPORTED, [0], [1], [-1], [0], [1], [1 << 20], freq_bits=20)
    refused(B.HS_UNSUPPORTED, [0], [1], [-1], freq_bits=5)
    long = np.random.default_rng(0).integers(0, om.vocab, 500).tolist()
    for i in range(0, 500, 250):
        batch.run_coded([1] * 250, long[i:i + 250], [0] * 250, long[i:i + 250])
    refused(B.HS_UNSUPPORTED, [1] * 13, [1] * 13, [-1] * 13)
    batch.run_tree([1] * 12, [1] * 12, [-1] * 12)
    for nodes in ([12], [0, 1], [1, 1]):
        with pytest.raises(B.HardShellError) as e:
            batch.tree_commit(nodes)
        assert e.value.code == B.HS_BAD_ARGUMENT
    batch.run_tree([0, 0, 1, 1], [1] * 4, [-1, 0, -1, 2])
    for nodes in ([1], [0, 1, 2, 0], [0, 2, 1], [1, 0], [0, 0]):
        with pytest.raises(B.HardShellError):
            batch.tree_commit(nodes)
    batch.tree_commit([2, 0, 1])  # a failed commit left the trees
    assert (batch.position(0), batch.position(1)) == (7, 501)
    batch.run_tree([], [], [])


# ---- beams ----


def beam_reference(w, costs, finished, beams, table):
    """The step by its definition on the weights of the living beams: [(cost, beam, token)] per group."""
    place = {int(t): j for j, t in reversed(list(enumerate(table))) if t}
    out = []
    for g in range(len(costs) // beams):
        found = []
        for b in range(beams):
            i = g * beams + b
            if costs[i] < 0:
                continue
            if finished[i]:
                found.append((costs[i], b, NONE))
                continue
            n = R.norm_of(table, int(w[i].sum()))
            for s in np.argsort(-w[i].astype(np.int64), kind="stable")[:beams + 64]:
                if w[i][s]:
                    found.append((costs[i] + n + place[int(w[i][s])], b, int(s)))
        out.append(sorted(found, key=lambda x: (x[0], x[1], -1 if x[2] == NONE else x[2]))[:beams])
    return out


@pytest.mark.parametrize("groups,beams", [(1, 4), (3, 5), (1, 32), (2, 1), (16, 8)])
def test_beam_search_equals_the_definition(mini, groups, beams):
    model, om = mini
    table = synth.exp_table(synth.LOGITS_EXP_E).astype(np.int64).tolist()
    r = np.random.default_rng(groups * 100 + beams)
    n = groups * beams
    batch = B.CudaBatch(model, n + 2, 256)
    slots = r.permutation(n + 2)[:n]
    # Each group starts with its first beam alone, after a context.
    seqs = [[] for _ in range(n)]
    costs = np.full(n, -1, np.int64)
    tokens = np.zeros(n, np.uint32)
    for g in range(groups):
        i = g * beams
        seqs[i] = r.integers(0, om.vocab, 5 + 3 * g).tolist()
        ctx = seqs[i]
        batch.run_coded([int(slots[i])] * len(ctx), ctx, [0] * len(ctx), ctx)
        costs[i], tokens[i] = 10 * g, r.integers(0, om.vocab)
    finished = np.zeros(n, np.uint8)
    for step in range(5):
        alive = [i for i in range(n) if costs[i] >= 0 and not finished[i]]
        for i in alive:
            seqs[i] = seqs[i] + [int(tokens[i])]
        w = np.zeros((n, om.vocab), np.uint64)
        w[alive] = oracle_weights(om, [seqs[i] for i in alive], [[]] * len(alive))
        want = beam_reference(w, costs.tolist(), finished, beams, table)
        s2, t2, c2, f2, p2 = batch.beam_step(groups, beams, slots, tokens, costs, finished)
        new = [[] for _ in range(n)]
        for g in range(groups):
            for j in range(beams):
                i = g * beams + j
                if j < len(want[g]):
                    cost, b, tok = want[g][j]
                    assert (int(c2[i]), int(p2[i]), int(t2[i])) == (cost, b, tok), (step, g, j)
                    assert f2[i] == (tok == NONE)
                    new[i] = seqs[g * beams + b]
                    assert batch.position(int(s2[i])) == len(new[i]) == batch.stream_len(int(s2[i]))
                else:
                    assert (int(c2[i]), int(p2[i]), int(t2[i]), f2[i]) == (-1, NONE, NONE, 0)
                    assert batch.position(int(s2[i])) == 0
            assert sorted(s2[g * beams:(g + 1) * beams]) == sorted(slots[g * beams:(g + 1) * beams])
        seqs, slots, tokens, costs, finished = new, s2, t2, c2, f2.copy()
        if step == 2:
            finished[beams - 1] = 1  # the caller ends a beam (its token was an end)
    # The states follow the beams: every living beam goes on as its sequence says.
    for i in range(n):
        if costs[i] < 0 or not seqs[i]:
            continue
        toks = r.integers(0, om.vocab, 3).tolist()
        got = batch.run_weights([int(slots[i])] * 3, toks)
        want = oracle_weights(om, [seqs[i]] * 3, [toks[:1], toks[:2], toks])
        assert np.array_equal(got, want), i


@pytest.mark.parametrize("name", ["tiny", "wide"])
def test_beam_search_of_other_models(dev, name):
    """Narrow heads and 64-column logits tiles: the states and costs agree with the model's own tables."""
    data = MODELS[name]()
    model, om = B.CudaModel(dev, data), O.Model(data)
    batch = B.CudaBatch(model, 4, 64)
    slots, tokens, costs = np.arange(4), np.array([3, 0, 0, 0]), np.array([0, -1, -1, -1])
    seqs = [[], None, None, None]
    for _ in range(6):
        seqs = [s + [int(t)] if c >= 0 else None for s, t, c in zip(seqs, tokens, costs)]
        slots, tokens, costs, _, par = batch.beam_step(1, 4, slots, tokens, costs)
        assert (np.diff(costs) >= 0).all() and (costs >= 0).all()
        # The cheapest new beam of a parent is its most likely token.
        for b in set(par.tolist()):
            first = par.tolist().index(b)
            w = oracle_weights(om, [seqs[b]], [[]])[0]
            assert w[tokens[first]] == w.max()
        seqs = [seqs[p] for p in par]
    for i in range(4):
        got = batch.run_weights([int(slots[i])], [7])[0]
        assert np.array_equal(got, oracle_weights(om, [seqs[i]], [[7]])[0])


def test_beam_refusals(mini):
    model, om = mini
    batch = B.CudaBatch(model, 4, 64)

    def refused(code, *args):
        with pytest.raises(B.HardShellError) as e:
            batch.beam_step(*args)
        assert e.value.code == code

    refused(B.HS_UNSUPPORTED, 1, 5, range(5), [0] * 5, [0] * 5)
    refused(B.HS_UNSUPPORTED, 1, 33, range(33), [0] * 33, [0] * 33)
    refused(B.HS_BAD_SLOT, 1, 2, [0, 4], [0, 0], [0, 0])
    refused(B.HS_BAD_ARGUMENT, 1, 2, [1, 1], [0, 0], [0, 0])
    refused(B.HS_BAD_ARGUMENT, 1, 2, [0, 1], [0, 0], [0, 1 << 62])
    refused(B.HS_TOKEN_RANGE, 1, 2, [0, 1], [0, om.vocab], [0, 0])
    refused(B.HS_LENGTH_MISMATCH, 2, 2, [0, 1], [0, 0], [0, 0])
    s, t, c, f, p = batch.beam_step(1, 2, [0, 1], [0, om.vocab], [5, -1])  # a dead beam's token is not looked at
    assert (c >= 5).all() and set(p.tolist()) == {0}
    toks = [1] * 512
    batch.reset(3)
    for i in range(0, 512, 64):
        batch.run_coded([3] * 64, toks[:64], [0] * 64, toks[:64])
    refused(B.HS_UNSUPPORTED, 1, 2, [0, 3], [0, 0], [0, 0])
    assert batch.position(3) == 512
    s, t, c, f, p = batch.beam_step(1, 2, [2, 3], [0, 0], [-1, -1])  # nothing lives
    assert (c == -1).all() and (p == NONE).all()
    s, t, c, f, p = batch.beam_step(1, 2, [0, 1], [0, 0], [7, 9], [1, 1])  # all have ended
    assert c.tolist() == [7, 9] and f.tolist() == [1, 1] and (t == NONE).all() and p.tolist() == [0, 1]


# ---- together ----


@pytest.mark.parametrize("depth,beams", [(1, 3), (3, 4), (4, 2)])
def test_speculative_decode_of_a_coded_stream(mini, depth, beams):
    """A range-coded stream of likely tokens comes back: in each round beams of the model (in slots of
    their own) draft a tree, one pass asks every node, the decoder walks it, and the right path plus
    the token after it are committed."""
    model, om = mini
    r = np.random.default_rng(depth * 10 + beams)
    ref, enc, truth, w = O.Session(om), O.Encoder(), [], None
    w = ref.step(om.eot)
    for _ in range(70):
        order = np.argsort(-w.astype(np.int64), kind="stable")
        t = int(order[min(int(r.geometric(0.6)) - 1, om.vocab - 1)])
        start, freq = O.answer(w, 32, 0, t)[1:]
        enc.interval(start, freq, t == om.vocab - 1, 32)
        truth.append(t)
        w = ref.step(t)
    payload = enc.finish()

    batch = B.CudaBatch(model, 1 + beams, 256)
    dec, out = O.Decoder(payload), []

    def take(iv):
        assert dec.interval(int(iv["start"]), int(iv["freq"]), bool(iv["is_last"]), 32)
        out.append(int(iv["symbol"]))

    pending, rounds = om.eot, 0  # the last token, not yet an input
    while len(out) < len(truth):
        rounds += 1
        # Draft: beams from the slot's state. Their slots start from the committed inputs.
        seq = [om.eot] + out
        for s in range(1, 1 + beams):
            batch.reset(s)
        if len(seq) > 1:
            batch.run_coded([1] * (len(seq) - 1), seq[:-1], [0] * (len(seq) - 1), [0] * (len(seq) - 1))
        slots, costs = np.arange(1, 1 + beams), np.array([0] + [-1] * (beams - 1))
        tokens = np.array([pending] + [0] * (beams - 1))
        trie, chains = {(): 0}, [()] * beams  # the root is the pending token
        for _ in range(depth):
            slots, tokens, costs, _, par = batch.beam_step(1, beams, slots, tokens, costs)
            chains = [chains[p] + (int(t),) if c >= 0 else () for p, t, c in zip(par, tokens, costs)]
            for ch in chains:
                for k in range(len(ch)):
                    trie.setdefault(ch[:k + 1], len(trie))
        toks = [pending] + [ch[-1] for ch in trie if ch]
        parents = [-1] + [trie[ch[:-1]] for ch in trie if ch]
        # Verify: every node's table is asked for each of its drafted children.
        asks = [(trie[ch[:-1]], ch[-1]) for ch in trie if ch]
        ivs = batch.run_tree([0] * len(toks), toks, parents, [a for a, _ in asks], [0] * len(asks),
                             [t for _, t in asks])
        path, at = [0], ()
        while len(out) < len(truth):
            target = dec.target(32)
            hit = None
            for (a, t), iv in zip(asks, ivs):
                if a == trie[at] and int(iv["start"]) <= target and (
                        iv["is_last"] or target < int(iv["start"]) + int(iv["freq"])):
                    hit = (t, iv)
            if hit is None:
                break
            take(hit[1])
            at = at + (hit[0],)
            path.append(trie[at])
        if len(out) < len(truth):  # the token that no draft holds, from the last right table
            iv = batch.tree_query([path[-1]], [1], [dec.target(32)])[0]
            take(iv)
        batch.tree_commit(path)
        pending = out[-1]
        assert out == truth[:len(out)]
        assert batch.position(0) == len(path) + (0 if rounds == 1 else before)
        before = batch.position(0)
    assert out == truth and rounds < len(truth)
