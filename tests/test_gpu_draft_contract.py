"""What the draft operators' documentation promises around the results: entries that are left out, calls
beside one another, and the first and last blocks of a launch. Plain 64-bit implementations as in
test_gpu_draft_ops.py; whole numbers, always equal."""

from __future__ import annotations

import numpy as np
import pytest

import tests.draft_ref as R
from taco_b200 import backend as B
from tests.test_gpu_draft_ops import beam_case, dev, gpu  # noqa: F401  (dev: the fixture)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


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
