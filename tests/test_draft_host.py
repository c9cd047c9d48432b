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
