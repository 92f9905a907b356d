"""accept and the decision that verify_drafts takes, next to the border between the two."""
import numpy as np
import pytest
import torch

from test_gpu_tokens import DEV, TYPES, softmax64, verify_inputs
from vortex_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("Vn", [1000, 50021])
def test_accept_agrees_with_a_decision_next_to_the_border(dt, Vn, with_draft):
    """u is p / q rounded to fp32, or a neighbour: such a draft is decided from fp64 sums, and accept comes from the same.  One
    rounding to fp32 keeps the order (u < p / q: u <= accept), and is all that accept is off by."""
    B = 60
    target, _, u, draft, _, _ = verify_inputs(B, 1, Vn, dt, 7 * Vn, greedy=0.0)
    p, q = (np.stack([softmax64(r.numpy(), 1.0) for r in t[:, 0].float()]) for t in (target, draft))
    x = (q - p).argmax(1) if with_draft else p.argmax(1)
    ratio = p[np.arange(B), x] / (q[np.arange(B), x] if with_draft else 1.0)
    near = ratio.astype(np.float32)
    u[:, 0] = torch.from_numpy(np.stack([near, np.nextafter(near, np.float32(0)), np.nextafter(near, np.float32(1))])[np.arange(B) % 3, np.arange(B)])
    assert bool((u[:, 0] < 1).all())
    _, cnt, acc, _ = ops.verify_drafts(target.to(DEV), torch.from_numpy(x)[:, None].to(DEV), u.to(DEV), draft.to(DEV) if with_draft else None)
    accepted, acc = cnt.cpu().numpy() == 2, acc[:, 0].cpu().numpy()
    assert (accepted == (u[:, 0].numpy().astype(np.float64) < ratio)).all()
    assert (np.abs(acc - ratio) <= ratio * (2.0 ** -24 + 8 * Vn * 2.0 ** -53)).all(), np.abs(acc / ratio - 1).max()
    assert (acc[accepted] >= u[:, 0].numpy()[accepted]).all() and (acc[~accepted] <= u[:, 0].numpy()[~accepted]).all()
