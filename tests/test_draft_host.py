"""The host side of the draft operators without a GPU: the library on a stand-in CUDA runtime (fake_cuda.py), where a
call can be made to fail and the calls are seen."""

from __future__ import annotations

import numpy as np
import pytest

from taco_b200 import backend as B
from tests import fake_cuda
from tests.common import tiny_bytes


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    from taco_b200 import build

    build.build()
    return fake_cuda.build(tmp_path_factory.mktemp("fake"))


def there(fake, function, *args):
    fake_cuda.run(fake, __name__, function.__name__, *args)


# ---- handles ----


def handles_that_are_ready():
    rt = fake_cuda.Runtime()
    dev = B.CudaDevice(0)
    assert rt.in_flight() == 0
    attn = B.AttnRule(dev, 1, 1, 1, 1, 30, np.arange(100, 0, -1))
    assert rt.in_flight() == 0
    weights = B.WeightRule(dev, np.arange(100, 0, -1))
    assert rt.in_flight() == 0
    attn.close()
    weights.close()
    dev.close()


def test_a_new_handle_is_whole_before_it_returns(fake):
    """The tables and the error words are on the GPU when the call that makes them returns: a stream that does not
    wait for the legacy one may use them at once."""
    there(fake, handles_that_are_ready)


def batches_whose_buffers_are_ready():
    rt = fake_cuda.Runtime()
    dev = B.CudaDevice(0)
    model = B.CudaModel(dev, tiny_bytes())
    batch = B.CudaBatch(model, 4, 64)
    batch.run_tree([0, 0], [1, 2], [-1, 0], [1], [0], [3])
    batch.tree_commit([0, 1])
    batch.beam_step(1, 2, [0, 1], [1, 1], [0, -1])
    batch.run_coded([0], [1], [0], [1])
    batch.run_weights([0], [1])
    batch.decode_blocks([2], [b"\0" * 16], [1])
    assert rt.launches() and rt.raced() == 0


def test_a_batch_uses_no_buffer_that_is_being_cleared(fake):
    """Buffers are cleared on the legacy stream and used on the batch's own, the ones made by a first tree pass or beam
    step too."""
    there(fake, batches_whose_buffers_are_ready)


# ---- errors of a batch ----


def beam_steps_that_fail():
    rt = fake_cuda.Runtime()
    batch = B.CudaBatch(B.CudaModel(B.CudaDevice(0), tiny_bytes()), 6, 64)

    def step():
        return batch.beam_step(1, 3, [4, 0, 2], [5, 6, 7], [3, -1, 9], [0, 0, 1])

    def state():
        return [(batch.position(s), batch.stream_len(s)) for s in range(6)]

    batch.run_coded([4, 4, 2], [1, 2, 3], [0] * 3, [1, 2, 3])
    batch.run_coded([4] * 4, [1] * 4, [0] * 4, [1] * 4)
    # (all new beams come from the first one, as kernels that do nothing leave it: the others get copies)
    rt.clear()
    before = state()
    assert before[4] == (6, 6) and before[2] == (1, 1)
    whole = step()
    after = state()
    assert after == [(7, 7), (0, 0), (7, 7), (0, 0), (7, 7), (0, 0)] and whole[0].tolist() == [4, 0, 2]
    calls = rt.calls()
    reorder = next(c for c in calls if "cache_reorder" in c)
    for s in range(6):
        batch.reset(s)
    batch.run_coded([4, 4, 2], [1, 2, 3], [0] * 3, [1, 2, 3])
    batch.run_coded([4] * 4, [1] * 4, [0] * 4, [1] * 4)
    assert state() == before
    for name in ("cudaMemcpyAsync", "cudaMemcpy", "cudaStreamSynchronize", reorder):
        for at in range(calls.count(name) if name != "cudaStreamSynchronize" else 1):
            rt.clear()
            rt.fail(name, at)
            with pytest.raises(B.HardShellError) as e:
                step()
            assert e.value.code == B.HS_CUDA, (name, at)
            rt.clear()
            assert state() == before, (name, at)
    assert [x.tolist() for x in step()] == [x.tolist() for x in whole] and state() == after


def test_a_beam_step_that_fails_changes_nothing(fake):
    """Every copy, wait and the cache move of a step fail once: the positions, streams, slots and tokens stay, and the
    step can be made again."""
    there(fake, beam_steps_that_fail)


def tree_commits_that_fail():
    rt = fake_cuda.Runtime()
    batch = B.CudaBatch(B.CudaModel(B.CudaDevice(0), tiny_bytes()), 3, 64)
    path = [0, 2, 3, 5, 6]

    def trees():
        for s in range(3):
            batch.reset(s)
        batch.run_coded([0] * 5, [1] * 5, [0] * 5, [1] * 5)
        batch.run_tree([0] * 4 + [2] * 3, [1] * 7, [-1, 0, 0, 2, -1, -1, 5])
        rt.clear()

    trees()
    batch.tree_commit(path)
    calls = rt.calls()
    assert (batch.position(0), batch.position(2)) == (8, 2)
    trees()
    for name in {c for c in calls if c.startswith(("cudaMemcpy", "launch"))}:
        for at in range(calls.count(name)):
            rt.clear()
            rt.fail(name, at)
            with pytest.raises(B.HardShellError):
                batch.tree_commit(path)
            assert (batch.position(0), batch.position(2)) == (5, 0) == (batch.stream_len(0), batch.stream_len(2))
    rt.clear()
    batch.tree_commit(path)
    assert (batch.position(0), batch.position(2)) == (8, 2)


def test_a_tree_commit_that_fails_changes_nothing(fake):
    there(fake, tree_commits_that_fail)


# ---- the end of trees and tables ----


def tables_after_calls_that_run_no_rows():
    batch = B.CudaBatch(B.CudaModel(B.CudaDevice(0), tiny_bytes()), 4, 64)

    def trees():
        for s in range(4):
            batch.reset(s)
        batch.run_coded([0] * 5, [1] * 5, [0] * 5, [1] * 5)
        batch.run_tree([0, 0], [1, 2], [-1, 0])

    def gone(f):
        with pytest.raises(B.HardShellError) as e:
            f()
        assert e.value.code == B.HS_BAD_ARGUMENT

    query = lambda: batch.tree_query([0, 1], [0, 0], [1, 2])  # noqa: E731
    for call, trees_end in ((lambda: batch.truncate(0, 3), True), (lambda: batch.truncate(0, 5), True),
                            (lambda: batch.tree_commit([0]), True), (lambda: batch.reset(3), False),
                            (lambda: batch.run_coded([], [], [], []), False), (lambda: batch.run_weights([], []), False),
                            (lambda: batch.decode_blocks([], [], []), False),
                            (lambda: batch.beam_step(1, 2, [1, 2], [0, 0], [5, -1], [1, 0]), True)):
        trees()
        call()
        query()
        if trees_end:
            gone(lambda: batch.tree_commit([0]))
        else:
            batch.tree_commit([0])
    for call in (lambda: batch.run_coded([3], [1], [0], [1]), lambda: batch.run_weights([3], [1]),
                 lambda: batch.decode_blocks([3], [b"\0" * 16], [1]),
                 lambda: batch.beam_step(1, 2, [1, 2], [0, 0], [5, -1])):
        trees()
        call()
        gone(query)
        gone(lambda: batch.tree_commit([0]))


def test_the_tables_of_a_tree_pass_stay_until_rows_run(fake):
    """A truncation inside the context, a commit, a reset, a call without rows and a step without living beams run
    nothing: the tables can still be asked."""
    there(fake, tables_after_calls_that_run_no_rows)


# ---- launches of the device-resident operators ----


def reorders_of_one_beam():
    rt = fake_cuda.Runtime()
    dev = B.CudaDevice(0)
    k, v = (fake_cuda.Tensor(rt, (2, 1, 16, 16), "int8") for _ in range(2))
    ids = fake_cuda.Tensor(rt, (2,), "int32")
    for groups, beams in ((2, 1), (1, 2)):
        rt.clear()
        before = B.launch_count()
        B.CacheReorder(dev, B.KvCache(k, v, 2, 1, 16, 16), groups, beams, ids, ids).run()
        assert len(rt.launches()) == 1 == B.launch_count() - before


def test_a_reorder_of_one_beam_is_checked_by_its_kernel(fake):
    """Groups of one beam have nothing to move, but a parent out of range is reported: the launch is made, as it is
    counted."""
    there(fake, reorders_of_one_beam)


# ---- the tensors of the device-resident operators ----


class Ops:
    """Calls with good tensors on the stand-in device; a test changes one of them."""

    def __init__(self):
        self.rt = rt = fake_cuda.Runtime()
        self.dev = B.CudaDevice(0)
        t = self.t = lambda shape, dtype, strides=None: fake_cuda.Tensor(rt, shape, dtype, strides)
        self.attn = B.AttnRule(self.dev, 1, 1, 1, 1, 30, [3, 2, 1])
        self.weights = B.WeightRule(self.dev, [3, 2, 1])
        # 3 slots of 4 planes of 32 rows of 16; 2 trees of up to 5 nodes; 2 groups of 3 beams over 300 symbols.
        self.cache = dict(k=t((3, 4, 32, 16), "int8"), v=t((3, 4, 16, 32), "int8"), slots=3, planes=4, n_ctx=32, head_dim=16)
        self.tree = dict(heads=8, kv_heads=4, q=t((10, 8, 16), "int8"), out=t((10, 8, 16), "int8"), rows=10,
                         seqs=t((2, 4), "int32"), n_seq=2, max_count=5, max_keys=30, mask=t((10, 1), "int32"), mask_words=1)
        self.beam = dict(dist=t((6, 512), "int16"), tops=t((6, 3), "int64"), vocab=300, groups=2, beams=3, keep=4,
                         base=t((6,), "int64"), parent=t((2, 4), "int32"), token=t((2, 4), "int32"),
                         cost=t((2, 4), "int64"), finished=t((6,), "uint8"))
        self.reorder = dict(groups=1, beams=3, parent=t((1, 3), "int32"), rows=t((1, 3), "int32"), slots=t((1, 3), "int32"))
        self.commit = dict(seqs=t((2, 4), "int32"), n_seq=2, path=t((2, 5), "int32"), path_ld=5, length=t((2,), "int32"))

    def run(self, op, cache=None, **kw):
        """The launches of a call."""
        self.rt.clear()
        c = B.KvCache(**{**self.cache, **(cache or {})})
        if op == "tree":
            call = B.TreeAttention(self.attn, c, **{**self.tree, **kw})
        elif op == "beam":
            call = B.BeamSelect(self.weights, **{**self.beam, **kw})
        elif op == "reorder":
            call = B.CacheReorder(self.dev, c, **{**self.reorder, **kw})
        else:
            call = B.CacheCommit(self.dev, c, **{**self.commit, **kw})
        for _ in range(2):
            call.run()
        return len(self.rt.launches())

    def refused(self, op, cache=None, code=B.HS_BAD_ARGUMENT, **kw):
        with pytest.raises(B.HardShellError) as e:
            self.run(op, cache, **kw)
        assert e.value.code == code, str(e.value)
        assert not self.rt.launches(), kw


def tensors_that_do_not_fit():
    o = Ops()
    t = o.t
    for op in ("tree", "beam", "reorder", "commit"):
        assert o.run(op) == 2
        for name, x in {**o.cache, **getattr(o, op)}.items() if op != "beam" else o.beam.items():
            if not hasattr(x, "shape"):
                continue
            inside = name in ("k", "v")
            wrong = {"int8": ("uint8", "int16", "float16"), "int32": ("int64", "float32", "int16"),
                     "int16": ("int32", "bfloat16"), "int64": ("int32", "float64"), "uint8": ("int32", "float32")}
            bad = [t(x.shape, d) for d in wrong[x.dtype.rsplit(".")[-1]]]           # another type
            if name != "dist":  # (whose rows are longer than the vocabulary)
                bad.append(t(x.shape[:-1] + (x.shape[-1] - 1,), x.dtype[6:]))           # too short
            bad.append(t((0,) + x.shape[1:], x.dtype[6:]))                              # empty
            if len(x.shape) > 1:
                if x.shape[0] > 1:
                    bad.append(t((x.shape[0] - 1,) + x.shape[1:], x.dtype[6:]))
                    if name not in ("dist", "tops"):  # (whose strides are the tensors' own)
                        bad.append(t(x.shape, x.dtype[6:], (x.strides[0] + 16,) + x.strides[1:]))  # a view with gaps
                    bad.append(t(x.shape, x.dtype[6:], (0,) + x.strides[1:]))                 # one row, expanded
                if x.shape[0] > 1 and x.shape[-1] > 1:
                    turned = list(x.strides)
                    turned[0], turned[-1] = 1, x.shape[0] * 700
                    bad.append(t(x.shape, x.dtype[6:], turned))                               # transposed
            else:
                bad.append(t(x.shape, x.dtype[6:], (2,)))                                     # every other element
            for y in bad:
                if inside:
                    o.refused(op, {name: y})
                else:
                    o.refused(op, **{name: y})


def test_tensors_that_do_not_hold_what_a_call_reads_are_refused(fake):
    """Another type, too few elements, gaps, expanded and transposed views of each tensor of each operator: an error,
    and nothing is launched."""
    there(fake, tensors_that_do_not_fit)


def caches_that_do_not_fit():
    o = Ops()
    t = o.t
    for op in ("tree", "reorder", "commit"):
        o.refused(op, dict(v=t((3, 4, 32, 16), "int8")))               # values that are not transposed
        o.refused(op, dict(k=t((3, 4, 16, 32), "int8")))
        o.refused(op, dict(k=t((3, 4, 32, 16), "int8", (2048, 512, 1, 32))))   # a transposed view
        o.refused(op, dict(slots=4))
        o.refused(op, dict(slot_stride=2064))
        # A batch's planes of a larger cache: its slots are slot_stride apart.
        part = {n: t(o.cache[n].shape, "int8", (5 * 512, 512) + o.cache[n].strides[2:]) for n in ("k", "v")}
        o.refused(op, part)
        assert o.run(op, dict(part, slot_stride=5 * 512)) == 2
        flat = {n: t((3 * 2048,), "int8") for n in ("k", "v")}
        assert o.run(op, flat) == 2
        assert o.run(op, {n: o.cache[n].data_ptr() for n in ("k", "v")}) == 2  # addresses are taken as they are


def test_caches_that_do_not_fit_are_refused(fake):
    there(fake, caches_that_do_not_fit)


def views_that_fit():
    o = Ops()
    t = o.t
    # q of a row of q, k and v; outputs with room behind each row.
    assert o.run("tree", q=t((10, 8, 16), "int8", (384, 16, 1)), q_stride=384) == 2
    o.refused("tree", q=t((10, 8, 16), "int8", (384, 16, 1)))
    o.refused("tree", q=t((10, 8, 16), "int8", (384, 16, 1)), q_stride=256)
    assert o.run("tree", out=t((10, 128), "int8", (144, 1)), out_stride=144) == 2
    assert o.run("tree", q=t((40, 128), "int8"), q_stride=512) == 2
    o.refused("tree", q=t((36, 128), "int8"), q_stride=512)
    assert o.run("tree", seqs=t((9, 4), "int32"), mask=t((640,), "uint32")) == 2
    # Logits by group and beam, parts of longer rows, and one row as a vector.
    assert o.run("beam", dist=t((2, 3, 512), "uint16"), tops=t((2, 3, 3), "int64")) == 2
    assert o.run("beam", dist=t((6, 300), "int16", (1000, 1)), tops=t((2, 3, 3), "int64", (12, 4, 1))) == 2
    o.refused("beam", dist=t((2, 3, 300), "int16", (4000, 1000, 1)))   # the groups are not 3 rows apart
    o.refused("beam", dist=t((2, 2, 512), "int16"))
    o.refused("beam", dist=t((6, 512), "int16"), dist_stride=600)
    assert o.run("beam", dist=t((300,), "int16"), tops=t((3,), "int64"), groups=1, beams=1) == 2
    assert o.run("beam", finished=t((2, 3), "bool")) == 2
    assert o.run("beam", finished=None) == 2
    # Nothing to do: nothing is looked at.
    assert o.run("tree", n_seq=0, q=t((1,), "int64")) == 0
    assert o.run("beam", keep=0, dist=None) == 0
    assert o.run("reorder", groups=0, parent=None) == 0
    assert o.run("commit", n_seq=0, path=None) == 0


def test_views_that_hold_what_a_call_reads_are_taken(fake):
    there(fake, views_that_fit)


def two_first_runs():
    o = Ops()
    o.rt.clear()
    call = B.CacheReorder(o.dev, B.KvCache(**o.cache), **o.reorder)
    check, other = call._check_fn, []

    def checked(handle, args):
        if not other:  # another thread's first run comes between, and ends first
            other.append(1)
            call.run()
        return check(handle, args)

    call._check_fn = checked
    call.run()
    assert len(o.rt.launches()) == 2


def test_two_first_runs_of_one_call(fake):
    """Two threads run an operator for the first time at once: both look it over, both launch."""
    there(fake, two_first_runs)


def refusals_of_the_library_first():
    o = Ops()
    # What the library refuses keeps its code, whatever the tensors are.
    small = o.t((1,), "float32")
    o.refused("tree", code=B.HS_UNSUPPORTED, heads=7, q=small)
    o.refused("tree", dict(n_ctx=8193, k=small), code=B.HS_UNSUPPORTED)
    o.refused("beam", code=B.HS_UNSUPPORTED, keep=65)
    o.refused("beam", code=B.HS_UNSUPPORTED, vocab=65537)
    o.refused("reorder", code=B.HS_UNSUPPORTED, beams=33)
    o.refused("reorder", groups=2)
    o.refused("commit", n_seq=4)
    for name in ("q", "out", "seqs", "mask"):
        o.refused("tree", **{name: None})


def test_the_library_refuses_first(fake):
    there(fake, refusals_of_the_library_first)
