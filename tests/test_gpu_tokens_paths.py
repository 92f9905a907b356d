"""Paths of the token-model kernels that only large vocabularies and many tokens take."""
import pytest
import torch

from test_gpu_tokens import DEV, TYPES, check_grad, check_verify, gen, grad_ref, verify_inputs, zipf
from vortex_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,Vn", [(torch.float32, 65536), (torch.float32, 65537), (torch.bfloat16, 131073), (torch.bfloat16, 151936), (torch.float16, 256000),
                                   (torch.float32, 262144), (torch.float32, 262145), (torch.float32, 300007), (torch.bfloat16, 524288), (torch.float16, 524289),
                                   (torch.bfloat16, 600011), (torch.float32, 1048583)])
def test_verify_large_vocabularies(dt, Vn):
    """More than 64 statistics of a row (beyond 65536 fp32 or 131072 16-bit logits), more than 256 runs in the draw and sums of a row
    (beyond 262144 or 524288)."""
    B, K = 4, 2
    target, tokens, u, draft, lens, _ = verify_inputs(B, K, Vn, dt, Vn, greedy=0.0)
    temp = torch.tensor([0.8, 0.0, 1.1, 0.6])
    target[1, 0, Vn - 7] = 30.0                                   # greedy: the last chunk's arg-max, and a tie with it further on
    target[1, 0, Vn - 3] = 30.0
    tokens[1, 0] = Vn - 7
    check_verify(target, tokens, u, draft, None, temp)
    check_verify(target, tokens, u, None, lens, temp)
    target[:, :, Vn // 3:Vn - 100] = -float("inf")                # runs without a weight between those that have one
    u[:, K] = torch.tensor([0.999, 0.5, 0.9, 0.25])
    check_verify(target, tokens, u, draft, torch.tensor([2, 2, 1, 0], dtype=torch.int32), temp)
    check_verify(target[:, :1], tokens[:, :0], u[:, K:], None, None, temp)      # sampling without drafts


@pytest.mark.parametrize("dt,Vn", [(torch.float32, 65537), (torch.bfloat16, 524288), (torch.float32, 300007)])
def test_verify_a_uniform_of_zero_draws_the_first_token_with_a_weight(dt, Vn):
    target = torch.randn(3, 1, Vn, generator=gen(Vn)).to(dt)
    for b, n in enumerate((0, 1, Vn - 2)):
        target[b, :, :n] = -float("inf")
    tok = ops.verify_drafts(target.to(DEV), torch.zeros(3, 0, dtype=torch.int64, device=DEV), torch.zeros(3, 1, device=DEV))[0]
    assert tok[:, 0].tolist() == [0, 1, Vn - 2]


@pytest.mark.parametrize("Vn", [50021, 151936])
@pytest.mark.parametrize("dt", TYPES)
def test_verify_greedy_batches(dt, Vn):
    """A whole batch decoded greedily: the drafts of every second sequence are right for a while."""
    B, K = 7, 3
    target, tokens, u, draft, lens, _ = verify_inputs(B, K, Vn, dt, 3 * Vn)
    best = target[:, :K].float().argmax(-1)
    for b in range(B):
        tokens[b, :b % (K + 1)] = best[b, :b % (K + 1)]
    check_verify(target, tokens, u, draft, None, torch.zeros(B))
    check_verify(target, tokens, u, None, lens, torch.zeros(B))


@pytest.mark.parametrize("dt,ot", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("T,Vr,D", [(524288, 3000, 8), (524289, 3000, 8), (600001, 70001, 3), (1300000, 40, 4), (1100003, 1500000, 2)])
def test_embed_grad_of_several_pieces_a_tile(T, Vr, D, dt, ot):
    """Beyond 524288 tokens a workgroup of the radix sort ranks several pieces of 2048 tokens, one after the other."""
    g = gen(T + Vr)
    ids = zipf(T, Vr, g)
    ids[torch.rand(T, generator=g) < 0.05] = -1
    grad = torch.randn(T, D, generator=g).to(dt)
    I, G = ids.to(DEV), grad.to(DEV)
    ref, err = grad_ref(ids, grad, Vr, 1.0)
    if ot == dt:
        got = ops.embed_tokens_grad(I, G, Vr)
        check_grad(got, ref, err)
        assert torch.equal(got, ops.embed_tokens_grad(I.int(), G, Vr)), "the order of the sums is fixed"
    old = torch.randn(Vr, D, generator=g).to(ot)
    ref, err = grad_ref(ids, grad, Vr, 1.0, old)
    check_grad(ops.embed_tokens_grad(I, G, Vr, out=old.to(DEV)), ref, err)
