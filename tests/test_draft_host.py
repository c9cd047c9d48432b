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
