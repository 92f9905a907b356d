"""The token that verify_drafts draws: it has a weight, whatever the rounding of the running sums does.

h = 2^-53, half a step of fp64 above 1: sums are made here whose value depends on the order of their terms.  The running sums go
by runs of tokens (1024 of fp32, 2048 of the 16-bit types), one to several runs for each of 256 threads."""
import numpy as np
import pytest
import torch

from test_gpu_tokens import DEV, TYPES, gen, softmax64
from vortex_amd import ops

pytestmark = pytest.mark.gpu
RUN = {torch.float32: 1024, torch.float16: 2048, torch.bfloat16: 2048}


def random_rows(dt, Vn, kept, rejected, seed):
    """(target, draft or None, tokens, weights of the draw in 64 bits) of 48 sequences: `kept` of the vocabulary is not masked; with
    `rejected` the only draft is refused by a uniform of 1."""
    B, g = 48, gen(seed)
    target = (torch.randn(B, 1 + rejected, Vn, generator=g) * 2).to(dt)
    target[:, :, int(kept * Vn):] = -float("inf")
    if not rejected:
        w = np.stack([softmax64(t.numpy(), 1.0) for t in target[:, 0].float()])
        return target, None, torch.zeros(B, 0, dtype=torch.int64), w
    draft = (target[:, :1].float() + 0.7 * torch.randn(B, 1, Vn, generator=g)).to(dt)
    p, q = (np.stack([softmax64(t.numpy(), 1.0) for t in rows[:, 0].float()]) for rows in (target, draft))
    return target, draft, torch.from_numpy((q - p).argmax(1))[:, None], np.where(p - q > 1e-12 * p, p - q, 0.0)


@pytest.mark.parametrize("rejected", [False, True])
@pytest.mark.parametrize("kept", [1.0, 0.5])
@pytest.mark.parametrize("dt,Vn", [(torch.float32, 5000), (torch.float32, 50021), (torch.bfloat16, 32000), (torch.float16, 131072)])
def test_a_uniform_of_one_draws_a_token_with_weight(dt, Vn, kept, rejected):
    target, draft, tokens, w = random_rows(dt, Vn, kept, rejected, Vn)
    u = torch.ones(target.size(0), 1 + rejected)
    tok, cnt, _, st = ops.verify_drafts(target.to(DEV), tokens.to(DEV), u.to(DEV), draft.to(DEV) if rejected else None)
    assert cnt.tolist() == [1] * len(w) and st.tolist() == [0] * len(w)
    got = tok[:, 0].tolist()
    assert max(got) < Vn and min(got) >= 0
    assert all(w[b, i] > 0 for b, i in enumerate(got)), [(b, i) for b, i in enumerate(got) if not w[b, i] > 0]


@pytest.mark.parametrize("dt", TYPES)
def test_running_sums_that_pass_the_border_at_a_masked_run(dt):
    """Weights 0.77 h, 0.77 h, 1, nothing, 1 in five runs, the uniform one half: the border is 1.  Summed in pairs, the running sum
    is 1 at the third run, where 1 + 0.77 h + 0.77 h leaves 1, and 1 + 2 h at the fourth, where 1 is added to 1.54 h."""
    run = RUN[dt]
    target = torch.full((1, 1, 5 * run + 100), -float("inf"))
    at = [3, run + 5, 2 * run + 77, 4 * run + 1]
    target[0, 0, at] = torch.tensor([-37.0, -37.0, 0.0, 0.0])
    tok = ops.verify_drafts(target.to(dt).to(DEV), torch.zeros(1, 0, dtype=torch.int64, device=DEV), torch.full((1, 1), 0.5, device=DEV))[0]
    assert tok.item() in at[2:]


@pytest.mark.parametrize("rejected", [False, True])
@pytest.mark.parametrize("u_last", [1.0, float("inf"), float("nan")])
@pytest.mark.parametrize("dt,Vn", [(torch.float32, 5000), (torch.float32, 50021), (torch.bfloat16, 32000), (torch.float16, 131072)])
def test_uniforms_of_one_and_above_draw_the_last_token_with_weight(dt, Vn, u_last, rejected):
    target, draft, tokens, w = random_rows(dt, Vn, 0.7, rejected, Vn + 1)
    u = torch.ones(target.size(0), 1 + rejected)
    u[:, -1] = u_last
    tok = ops.verify_drafts(target.to(DEV), tokens.to(DEV), u.to(DEV), draft.to(DEV) if rejected else None)[0]
    assert tok[:, 0].tolist() == [int(np.nonzero(r)[0][-1]) for r in w]


@pytest.mark.parametrize("u", [1.0, 2.0, float("nan")])
@pytest.mark.parametrize("dt", TYPES)
def test_a_uniform_of_one_is_behind_every_running_sum(dt, u):
    """Weights 0.77 h, 0.77 h, 1, 7e-4 h, 7e-4 h: the sum of all is 1 in its own order, the running sum is 1 + 2 h at the fourth."""
    run = RUN[dt]
    target = torch.full((1, 1, 5 * run + 100), -float("inf"))
    target[0, 0, [3, run + 5, 2 * run + 77, 3 * run + 9, 4 * run + 1]] = torch.tensor([-37.0, -37.0, 0.0, -44.0, -44.0])
    tok = ops.verify_drafts(target.to(dt).to(DEV), torch.zeros(1, 0, dtype=torch.int64, device=DEV), torch.full((1, 1), u, device=DEV))[0]
    assert tok.item() == 4 * run + 1


@pytest.mark.parametrize("dt,Vn", [(torch.float32, 400000), (torch.float16, 800000)])
def test_two_runs_a_thread_and_no_running_sum_that_passes(dt, Vn):
    """From 257 runs on a thread has two.  Weights 1 | v, (a, b) | 1 at three threads with v = 0.496 h, a = 1.018 h, b = 1.787 h, the
    uniform one half: the sum of all is rounded to 2 + 4 h, so the border is 1 + 2 h, which the second thread passes as a whole
    (1 + 3.3 h: 1 + 4 h) and run by run does not (1 + v: 1, and 2.8 h more: 1 + 2 h).  The token is then the thread's last, b; it
    is in exact arithmetic too (v + a < (v + a + b) / 2)."""
    run = RUN[dt]
    target = torch.full((1, 1, Vn), -float("inf"))
    at = [5, 2 * run + 40, 3 * run + 300, 3 * run + 700, 4 * run + 9]
    target[0, 0, at] = torch.tensor([0.0, -37.4375, -36.71875, -36.15625, 0.0])
    w = np.exp(np.array([-37.4375, -36.71875, -36.15625])) * 2.0 ** 53
    assert 256 * run < Vn < 512 * run and w[1] > 1 and w[0] < 1 and w[1] + w[2] < 3 < w.sum() < 5 and 2 * (w[0] + w[1]) < w.sum()
    tok = ops.verify_drafts(target.to(dt).to(DEV), torch.zeros(1, 0, dtype=torch.int64, device=DEV), torch.full((1, 1), 0.5, device=DEV))[0]
    assert tok.item() == at[3]
