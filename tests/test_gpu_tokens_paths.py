"""Paths of the token-model kernels that large vocabularies, many tokens, many drafts, wide rows and strides take."""
import pytest
import torch

from test_gpu_tokens import DEV, TYPES, check_grad, check_verify, gen, grad_ref, quant_ref, verify_inputs, zipf
from vortex_amd import _lib as L
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


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("K", [15, 16, 31, 63, 64])
def test_verify_many_drafts(dt, K):
    """Up to 64 drafts, the first of them right: all of a wave's lanes decide, and all words of the masks are used."""
    B, Vn = 6, 301
    target, tokens, u, draft, _, _ = verify_inputs(B, K, Vn, dt, 10 * K, greedy=0.0)
    draft[:3] = target[:3, :K]                                    # p = q: every draft is accepted
    u[:3, :K] *= 0.999
    lens = torch.tensor([K, K - 1, 1, K, K - 1, 0], dtype=torch.int32)
    check_verify(target, tokens, u, draft, None, torch.ones(B))
    check_verify(target, tokens, u, draft, lens, torch.full((B,), 0.7))
    tokens[:4] = target[:4, :K].float().argmax(-1)
    tokens[1, K - 1], tokens[2, K // 2], tokens[3, 0] = Vn, -1, (tokens[3, 0] + 1) % Vn
    check_verify(target, tokens, u, None, lens, torch.zeros(B))
    check_verify(target, tokens, u, draft, None, torch.tensor([0.0, 0.0, 0.0, 0.0, 1.0, 0.3]))


@pytest.mark.parametrize("dt", TYPES)
def test_embed_widest_rows(dt):
    """1048576 columns, the most that a row may have."""
    Vr, D = 3, 1 << 20
    g = gen(1)
    table, ids = torch.randn(Vr, D, generator=g).to(dt), torch.tensor([2, -1, 0, 2, 2])
    out = ops.embed_tokens(ids.to(DEV), table.to(DEV), 0.5).cpu()
    ref = (table[ids.clamp_min(0)].float() * 0.5).to(dt)
    ref[1] = 0
    assert torch.equal(out, ref)
    check_grad(ops.embed_tokens_grad(ids.to(DEV), table[ids].to(DEV), Vr, 2.0), *grad_ref(ids, table[ids], Vr, 2.0))


@pytest.mark.parametrize("M,K,lead,more", [(1, 5, 0, 1), (3, 64, 1, 37), (300, 100, 3, 28), (300, 2500, 0, 60), (2, 9000, 5, 7000), (257, 1, 2, 130)])
def test_quantize_rows_of_a_wider_matrix(M, K, lead, more):
    """Through the C ABI: columns behind K are zeroed up to the row's end, and nothing around the rows is written."""
    lib, g = L.lib(), gen(M + K)
    for dt, code in zip(TYPES, (L.VX_DTYPE_F32, L.VX_DTYPE_F16, L.VX_DTYPE_BF16)):
        x = torch.randn(M, K + 3, generator=g).to(dt)
        X = x.to(DEV)
        q = torch.full((lead + M * (K + more) + 40,), 99, dtype=torch.int8, device=DEV)
        s = torch.full((M + 2,), 7.0, device=DEV)
        rc = lib.vx_quantize_rows_i8(X.data_ptr() + X.element_size(), code, M, K, K + 3, q.data_ptr() + lead, K + more, s.data_ptr() + 4, L.stream_ptr(DEV))
        assert rc == 0
        qr, sr = quant_ref(x[:, 1:1 + K])
        rows = q[lead:lead + M * (K + more)].view(M, K + more).cpu()
        assert torch.equal(rows[:, :K], qr) and not rows[:, K:].any() and torch.equal(s[1:-1].cpu(), sr)
        assert bool((q[:lead] == 99).all()) and bool((q[lead + M * (K + more):] == 99).all()) and s[[0, -1]].tolist() == [7.0, 7.0]
