"""Token-model operators at the largest sizes: launches of more than 2^24 workgroups (HIP takes fewer than 2^32 threads along an axis),
the most tokens and channels of the 8-bit product."""
import pytest
import torch

from test_gpu_tokens import DEV, gen
from vortex_amd import _lib as L
from vortex_amd import ops

pytestmark = pytest.mark.gpu
MANY = 2 ** 26 + 5                              # tokens: one wave each, four to a workgroup


@pytest.mark.parametrize("dt,D", [(torch.float32, 1), (torch.bfloat16, 8)])
def test_embed_more_tokens_than_one_axis_of_a_launch(dt, D):
    Vr = 100003
    table = torch.randn(Vr, D, generator=gen(D)).to(dt).to(DEV)
    ids = (torch.arange(MANY, device=DEV, dtype=torch.int32) * 7919) % Vr        # wraps around below 0 now and then: padding
    ids[-1] = Vr - 1
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = ops.embed_tokens(ids, table, 2.0, status=st)
    for a in range(0, MANY, 1 << 24):
        i = ids[a:a + (1 << 24)].long()
        ref = torch.where((i >= 0)[:, None], table[i.clamp_min(0)] * 2.0, torch.zeros((), dtype=dt, device=DEV))
        assert torch.equal(got[a:a + (1 << 24)], ref), a
    assert int(st) == 0
    ids[-1] = Vr
    assert not ops.embed_tokens(ids, table, 2.0, status=st)[-1].any() and int(st) == L.VX_STATUS_BAD_TOKEN


@pytest.mark.parametrize("D", [1, 4])
def test_embed_grad_of_more_rows_than_one_axis_of_a_launch(D):
    """2^27 table rows and more, eight to a workgroup.  Whole numbers below 2^24: fp32 sums are exact."""
    T, Vr = 20000, 2 ** 27 + 9
    ids = torch.randint(0, Vr, (T,), generator=gen(D)).to(DEV)
    ids[:3000], ids[3000:4000], ids[4000] = Vr - 1, 2 ** 26 + 1, 0
    grad = torch.randint(-8, 9, (T, D), generator=gen(D + 1)).float().to(DEV)
    ref = torch.zeros(Vr, D, device=DEV).index_put_((ids,), grad, accumulate=True)
    assert torch.equal(ops.embed_tokens_grad(ids, grad, Vr), ref)
    out = torch.ones(Vr, D, device=DEV)
    assert torch.equal(ops.embed_tokens_grad(ids, grad, Vr, out=out), ref + 1)


def test_quantize_more_rows_than_one_axis_of_a_launch():
    x = torch.arange(MANY, device=DEV, dtype=torch.float32)[:, None] - 2 ** 25
    q, s = ops.quantize_rows_i8(x)
    assert torch.equal(q, torch.sign(x).to(torch.int8) * 127) and torch.equal(s.cpu(), x[:, 0].cpu().abs() / 127.0)


@pytest.mark.parametrize("with_draft", [False, True])
def test_verify_more_chunks_than_one_axis_of_a_launch(with_draft):
    """65535 sequences with room for 64 drafts and four chunks of logits, all on the same logits: more than 2^24 chunks of
    rows, of which only the first sequences' and the last ones' have drafts."""
    B, K, Vn, n = 65535, 64, 3 * 4096 + 1, 5
    g = gen(3)
    target, draft = torch.randn(1, K + 1, Vn, generator=g).to(DEV), torch.randn(1, K, Vn, generator=g).to(DEV)
    tokens, u = torch.randint(0, Vn, (B, K), generator=g).to(DEV), torch.rand(B, K + 1, generator=g).to(DEV)
    tokens[:, 0] = target[0, 0].argmax()
    u[::2, 0] = 0.0                                               # accepted
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    lens[:n], lens[-n:] = 3, 64
    got = ops.verify_drafts(target.expand(B, K + 1, Vn), tokens, u, draft.expand(B, K, Vn) if with_draft else None, lens)
    for part in (slice(0, n), slice(B // 2, B // 2 + n), slice(B - n, B)):
        ref = ops.verify_drafts(target.expand(n, K + 1, Vn), tokens[part], u[part], draft.expand(n, K, Vn) if with_draft else None, lens[part])
        assert all(torch.equal(a[part], b) for a, b in zip(got, ref)), part
    assert int(got[1].min()) >= 1 and int(got[1].max()) >= 2 and not got[3].any()
    assert bool((got[0][:, 0] >= 0).all()) and bool((got[0] < Vn).all())


MOST = 4194240                                  # tokens or channels of the 8-bit product


def check_product(q, s, qw, sw, got, two):
    """Few enough terms that fp32 sums them exactly; the scales and the product as the operator rounds them.  In pieces: the library's
    product leaves a result from its 2 GiB on at 0."""
    for a in range(0, got.size(0), 1 << 18):
        for b in range(0, got.size(1), 1 << 20):
            r, c = slice(a, a + (1 << 18)), slice(b, b + (1 << 20))
            ref = (q[r].float() @ qw[c].float().t().contiguous()) * (s[r, None] * sw[None, c])
            assert torch.equal(got[r, c], ref) and torch.equal(two[r, c], ref), (a, b)


@pytest.mark.parametrize("M", [1, 3, 40, 200])
def test_linear_most_channels(M):
    K, g = 16, gen(M)
    x, sw = torch.randn(M, K, generator=g).to(DEV), torch.rand(MOST, generator=g).to(DEV)
    qw = torch.randint(-128, 128, (MOST, K), generator=g, dtype=torch.int8).to(DEV)
    q, s = ops.quantize_rows_i8(x)
    check_product(q, s, qw, sw, ops.linear_w8a8(x, qw, sw), ops.linear_i8(q, s, qw, sw))


@pytest.mark.parametrize("N,odd", [(20, 0), (20, 1), (300, 0)])
def test_linear_most_tokens(N, odd):
    """Few channels (the weights stay on the chip), tiles, and with weights at an odd address the streaming kernel, 64 tokens a workgroup."""
    K, g = 16, gen(N)
    x, sw = torch.randn(MOST, K, generator=g).to(DEV), torch.rand(N, generator=g).to(DEV)
    flat = torch.randint(-128, 128, (N * K + odd,), generator=g, dtype=torch.int8).to(DEV)
    qw = flat[odd:].view(N, K)
    q, s = ops.quantize_rows_i8(x)
    check_product(q, s, qw, sw, ops.linear_w8a8(x, qw, sw), ops.linear_i8(q, s, qw, sw))
