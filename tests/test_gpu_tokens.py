"""Token-model operators on the GPU against plain 64-bit implementations on the CPU: embedding lookup and its gradient,
8-bit product, verification of drafted tokens.

Tolerances (u = 2^-24, the rounding of one fp32 operation; e = half a step of the output type, eps/2):
  embedding      one fp32 product, one rounding: bit-exact against the same two operations on the CPU
  gradient       an fp32 sum of n terms in any order: n u sum|terms|, times the scale; the product, the rounding: (2 u + e) |result|
  quantisation   exact by construction: integers equal, scales equal to the fp32 quotient
  product        integer sum exact; its conversion, the product of the scales, their product: 3 u |before bias|; the bias and the
                 rounding: (u + e) |result|
  verification   whole numbers equal.  accept is a quotient of two probabilities whose normalising sums are fp32: an exponential
                 of the sum is off by 2 u (the instruction) + 3 u ln2 |t| (difference, factor and product in its exponent t to base
                 2), and |t| averages, weighted with the distribution, at most its entropy, log2 V; at most 64 operations follow one
                 another, 64 u.  At V = 2^17: (2 + 3 * 0.7 * 17 + 64) u < 102 u for each sum, 2^-16.3 for the quotient: 2^-15 |value|"""
import numpy as np
import pytest
import torch
import torch.nn as nn

import vortex_amd as V
from vortex_amd import _lib as L
from vortex_amd import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}     # the smallest step near zero
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def zipf(n, V_, g):
    return (torch.exp(torch.rand(n, generator=g, dtype=torch.float64) * np.log(V_ + 1.0)) - 1).long().clamp(0, V_ - 1)


# ------------------------------------------------------------------------------------------------ embedding
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("T,Vr,D", [(1, 1, 1), (1, 7, 8), (3, 50, 7), (64, 1000, 64), (65, 1000, 1027), (500, 333, 1000), (33, 5000, 4096), (7, 11, 8200), (9000, 70, 2048), (9001, 70, 2056)])
def test_embed_rows(dt, T, Vr, D):
    g = gen(T * 31 + D)
    table = torch.randn(Vr, D, generator=g).to(dt)
    ids = torch.randint(-2, Vr, (T,), generator=g)
    for scale in (1.0, 0.37):
        got = ops.embed_tokens(ids.to(DEV), table.to(DEV), scale).cpu()
        ref = (table[ids.clamp_min(0)].float() * scale).to(dt)
        ref[ids < 0] = 0
        assert torch.equal(got, ref)


def test_embed_shapes_strides_and_id_types():
    g = gen(5)
    big = torch.randn(40, 96, generator=g)
    ids = torch.randint(0, 20, (2, 3, 5), generator=g)
    d = big.to(DEV)
    views = [(d[:, :33], big[:, :33]), (d[::2], big[::2]), (d[1:21, 3:50], big[1:21, 3:50]), (d.t().contiguous().t(), big),
             (d.half()[:, 1:], big.half()[:, 1:]), (d[:1].expand(20, 96), big[:1].expand(20, 96))]
    for table, ref in views:
        for i in (ids.to(DEV), ids.int().to(DEV), ids.to(DEV).transpose(0, 2).contiguous().transpose(0, 2)):
            out = ops.embed_tokens(i, table)
            assert out.shape == ids.shape + (table.size(1),) and torch.equal(out.cpu(), ref[ids])
    assert ops.embed_tokens(ids[:0].to(DEV), d).shape == (0, 3, 5, 96)
    assert ops.embed_tokens(torch.tensor(3, device=DEV), d).shape == (96,)


def test_embed_reports_ids_beyond_the_table():
    d = torch.randn(10, 16, device=DEV)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    ok = ops.embed_tokens(torch.tensor([0, 9, -1, -(1 << 40)], device=DEV), d, status=st)
    assert int(st) == 0 and torch.equal(ok[:2], d[[0, 9]]) and not ok[2:].any()
    bad = ops.embed_tokens(torch.tensor([0, 10, 1 << 40], device=DEV), d, status=st)
    assert int(st) == L.VX_STATUS_BAD_TOKEN and torch.equal(bad[0], d[0]) and not bad[1:].any()
    st.zero_()
    gr = ops.embed_tokens_grad(torch.tensor([0, 10, 1 << 40, -3, 9], device=DEV), torch.ones(5, 16, device=DEV), 10, status=st)
    assert int(st) == L.VX_STATUS_BAD_TOKEN and gr.sum().item() == 32.0 and gr[0].sum().item() == 16.0
    with pytest.raises(L.VortexHipError):
        ops.raise_on_status(int(st))


def test_embed_offsets_beyond_32_bits():
    """A table of more than 2^31 elements (bf16, 4.4 GB): the last rows are found."""
    Vr, D = 540000, 4096
    table = torch.zeros(Vr, D, dtype=torch.bfloat16, device=DEV)
    table[-3:] = torch.arange(3, device=DEV)[:, None].to(torch.bfloat16) + 1
    out = ops.embed_tokens(torch.tensor([Vr - 1, 0, Vr - 3], device=DEV), table)
    assert out[:, 0].tolist() == [3.0, 0.0, 1.0] and out[:, -1].tolist() == [3.0, 0.0, 1.0]
    g = torch.ones(3, D, dtype=torch.bfloat16, device=DEV)
    gr = ops.embed_tokens_grad(torch.tensor([Vr - 1, Vr - 1, 5], device=DEV), g, Vr)
    assert gr[Vr - 1].float().sum().item() == 2.0 * D and gr[5].float().sum().item() == D and not gr[Vr - 2].any()


# ------------------------------------------------------------------------------------------------ its gradient
def grad_ref(ids, g, Vr, scale, old=None):
    """(result, error of the fp32 sum) in 64 bits."""
    ok = (ids >= 0) & (ids < Vr)
    i, gg = ids[ok], g.double()[ok]
    s = torch.zeros(Vr, g.size(1), dtype=torch.float64).index_add_(0, i, gg)
    a = torch.zeros(Vr, g.size(1), dtype=torch.float64).index_add_(0, i, gg.abs())
    n = torch.zeros(Vr, dtype=torch.float64).index_add_(0, i, torch.ones_like(i, dtype=torch.float64))[:, None]
    s, a = s * scale, a * abs(scale)
    if old is not None:
        s, a = s + old.double(), a + old.double().abs()
    return s, (n + 2) * U * a


def check_grad(got, ref, err):
    dt = got.dtype
    got = got.cpu().double()
    assert got.shape == ref.shape
    off = (got - ref).abs()
    assert bool((off <= err * (1 + HALF_STEP[dt]) + HALF_STEP[dt] * ref.abs() + TINY[dt]).all()), float((off - err).max())


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("T,Vr,D", [(1, 1, 1), (2, 5, 8), (63, 40, 7), (64, 1000, 64), (1000, 3, 65), (1025, 5000, 100), (4097, 700, 1000),
                                    (5000, 50021, 33), (20000, 300, 16), (3000, 1, 40), (9000, 70001, 24), (64, 3, 520), (65, 3, 520), (255, 1, 24), (2049, 200, 520), (8192, 5, 8), (8191, 511, 8), (16384, 512, 8),
                                    (16385, 512, 8), (20001, 511, 9),
                                    (70000, 2, 12), (200000, 600000, 4), (300, 20000, 1024), (301, 20001, 1028)])
def test_embed_grad(dt, T, Vr, D):
    g = gen(T + Vr)
    ids = zipf(T, Vr, g)
    if T > 2:
        ids[torch.rand(T, generator=g) < 0.1] = -1
    grad = torch.randn(T, D, generator=g).to(dt)
    got = ops.embed_tokens_grad(ids.to(DEV), grad.to(DEV), Vr, 0.7)
    assert got.dtype == dt
    check_grad(got, *grad_ref(ids, grad, Vr, np.float32(0.7).item()))
    again = ops.embed_tokens_grad(ids.int().to(DEV), grad.to(DEV), Vr, 0.7)
    assert torch.equal(got, again), "the order of the sums is fixed"


@pytest.mark.parametrize("ids", ["equal", "distinct", "padding", "sorted", "reversed", "two"])
def test_embed_grad_orders(ids):
    T, Vr, D = 3000, 4000, 72
    g = gen(3)
    i = {"equal": torch.full((T,), 17), "distinct": torch.randperm(Vr, generator=g)[:T], "padding": torch.full((T,), -1),
         "sorted": torch.randint(0, Vr, (T,), generator=g).sort()[0], "reversed": torch.arange(T).flip(0),
         "two": torch.tensor([Vr - 1, 0]).repeat(T // 2)}[ids]
    grad = torch.randn(T, D, generator=g)
    check_grad(ops.embed_tokens_grad(i.to(DEV), grad.to(DEV), Vr), *grad_ref(i, grad, Vr, 1.0))


@pytest.mark.parametrize("dt,ot", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float32),
                                   (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)])
def test_embed_grad_accumulates_into_a_given_gradient(dt, ot):
    T, Vr, D = 700, 900, 130
    g = gen(8)
    ids = zipf(T, Vr, g).view(7, 100)
    grad = torch.randn(7, 100, D, generator=g).to(dt)
    old = torch.randn(Vr, D, generator=g).to(ot)
    old[5, 3] = float("nan")                       # a row that no id points to keeps its bits
    ids[ids == 5] = 6
    out = old.to(DEV)
    got = ops.embed_tokens_grad(ids.to(DEV), grad.to(DEV), Vr, 2.0, out=out)
    assert got.data_ptr() == out.data_ptr()
    untouched = torch.ones(Vr, dtype=torch.bool)
    untouched[ids.flatten()] = False
    assert torch.equal(got.cpu()[untouched].view(torch.uint8), old[untouched].view(torch.uint8))
    ref, err = grad_ref(ids.flatten(), grad.flatten(0, 1), Vr, 2.0, old)
    check_grad(got[~untouched.to(DEV)], ref[~untouched], err[~untouched])


@pytest.mark.parametrize("T,Vr,D", [(1, 2, 1), (3, 7, 5), (40, 300, 8), (70, 140, 1027), (500, 1000, 1000), (501, 1001, 64), (16384, 32768, 40), (16384, 32767, 40),
                                    (300, 40000, 2050), (129, 258, 4097)])
@pytest.mark.parametrize("dt", TYPES)
def test_embed_grad_of_few_tokens_clears_the_other_rows(T, Vr, D, dt):
    """Up to half as many tokens as rows the table is cleared beside the sort: at any address, and nothing around it."""
    lib, g = L.lib(), gen(T + Vr + D)
    ids = zipf(T, Vr, g)
    ids[0], ids[T // 2] = Vr - 1, -1
    grad = torch.randn(T, D, generator=g).to(dt)
    I, G = ids.to(DEV), grad.to(DEV)
    code = {torch.float32: L.VX_DTYPE_F32, torch.float16: L.VX_DTYPE_F16, torch.bfloat16: L.VX_DTYPE_BF16}[dt]
    nb = lib.vx_embed_tokens_grad_workspace_bytes(T, Vr, D)
    ws = torch.empty(nb, dtype=torch.uint8, device=DEV)
    ref, err = grad_ref(ids, grad, Vr, 0.5)
    for lead in (0, 1, 5):
        out = torch.full((lead + Vr * D + 9,), 7.0, dtype=dt, device=DEV)
        rc = lib.vx_embed_tokens_grad(I.data_ptr(), 8, T, G.data_ptr(), code, Vr, D, 0.5, out.data_ptr() + lead * out.element_size(), code, 0, None,
                                      ws.data_ptr(), nb, L.stream_ptr(DEV))
        assert rc == 0
        check_grad(out[lead:lead + Vr * D].view(Vr, D), ref, err)
        assert bool((out[:lead] == 7).all()) and bool((out[lead + Vr * D:] == 7).all())
    assert torch.equal(ops.embed_tokens_grad(I, G, Vr, 0.5), out[lead:lead + Vr * D].view(Vr, D))


@pytest.mark.parametrize("T,Vr", [(10, 40), (30, 40), (20000, 70000)])
def test_embed_grad_rows_without_tokens_are_zero_at_any_scale(T, Vr):
    ids = torch.arange(T, device=DEV) % (Vr // 2)
    for scale in (float("inf"), float("nan"), -1.0):
        got = ops.embed_tokens_grad(ids, torch.ones(T, 24, device=DEV), Vr, scale)
        n = min(T, Vr // 2)
        assert not got[n:].any() and not got[n:].isnan().any()
        assert not got[:n].isfinite().any() if scale != -1.0 else bool((got[:n] < 0).all())


def test_embed_grad_keeps_nan_and_inf_in_their_rows():
    ids = torch.tensor([1, 2, 2, 3], device=DEV)
    grad = torch.ones(4, 9, device=DEV)
    grad[0, 0], grad[1, 1], grad[3, 2] = float("nan"), float("inf"), -float("inf")
    got = ops.embed_tokens_grad(ids, grad, 5).cpu()
    assert got[1, 0].isnan() and got[2, 1] == float("inf") and got[3, 2] == -float("inf")
    keep = torch.ones(5, 9, dtype=torch.bool)
    keep[1, 0] = keep[2, 1] = keep[3, 2] = False
    assert bool(got[keep].isfinite().all()) and not got[0].any() and not got[4].any()


def test_embedding_module_trains():
    """TokenEmbedding's gradient against the 64-bit definition and against differences of the loss."""
    m = V.TokenEmbedding(50, 24, scale=3.0).to(DEV)
    ids = torch.tensor([[4, 4, -1], [49, 0, 4]], device=DEV)
    c = torch.randn(2, 3, 24, device=DEV, generator=torch.Generator(DEV).manual_seed(1))

    def loss():
        return (m(ids) * c).sum()
    loss().backward()
    ref, err = grad_ref(ids.cpu().flatten(), c.cpu().flatten(0, 1), 50, 3.0)
    check_grad(m.weight.grad, ref, err)
    with torch.no_grad():
        for v, k in ((4, 0), (49, 23), (0, 5), (7, 2)):
            w = m.weight.detach().double().cpu()
            d = torch.zeros_like(w)
            d[v, k] = 0.5                                        # the loss is linear in the weights: any step is exact
            hi, lo = [float((((w + s * d) * 3.0)[ids.cpu().clamp_min(0)] * (ids.cpu() >= 0)[..., None] * c.cpu().double()).sum()) for s in (1, -1)]
            assert abs((hi - lo) - float(m.weight.grad[v, k])) <= float(err[v, k]) + U * abs(hi - lo) + 1e-11   # 64-bit sums of 72 values
    first = m.weight.grad.clone()
    loss().backward()                                            # accumulates as every parameter's gradient does
    assert torch.equal(m.weight.grad, first + first)
    m.weight.requires_grad_(False)
    assert not m(ids).requires_grad


def test_embedding_gradient_of_an_expanded_and_of_a_strided_grad():
    m = V.TokenEmbedding(11, 40, scale=0.5, dtype=torch.bfloat16).to(DEV)
    ids = torch.tensor([3, 3, 10, -1, 3], device=DEV)
    m(ids).sum().backward()                                        # grad_out: one value, stride 0
    ref, err = grad_ref(ids.cpu(), torch.ones(5, 40), 11, 0.5)
    check_grad(m.weight.grad, ref, err)
    c = torch.randn(40, 5, device=DEV).to(torch.bfloat16).t()
    (g,) = torch.autograd.grad(m(ids), m.weight, c)
    check_grad(g, *grad_ref(ids.cpu(), c.cpu(), 11, 0.5))


def test_embedding_gradient_in_a_captured_graph():
    """Forward and torch.autograd.grad captured together, replayed with other ids between eager steps."""
    m = V.TokenEmbedding(300, 64).to(DEV)
    ids, c = torch.zeros(90, dtype=torch.int64, device=DEV), torch.randn(90, 64, device=DEV)

    def step():
        return torch.autograd.grad((m(ids) * c).sum(), m.weight)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(4):
        ids.copy_(torch.randint(-1, 300, (90,), generator=gen(k)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, ops.embed_tokens_grad(ids, c, 300)), "replay %d" % k


# ------------------------------------------------------------------------------------------------ 8-bit product
def quant_ref(x):
    x = x.double()
    amax = x.abs().amax(-1, keepdim=True)
    q = torch.where(amax > 0, torch.round(x * 127.0 / amax.where(amax > 0, torch.ones_like(amax))), torch.zeros_like(x))
    return q.to(torch.int8), amax[..., 0].float() / 127.0


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (1, 5), (3, 64), (17, 127), (5, 1000), (64, 1024), (2, 4099), (300, 256), (1, 131072)])
def test_quantize_rows(dt, M, K):
    g = gen(M + K)
    x = (torch.randn(M, K, generator=g) * torch.exp(3 * torch.randn(M, 1, generator=g))).to(dt)
    x[0, 0] = 0
    q, s = ops.quantize_rows_i8(x.to(DEV))
    qr, sr = quant_ref(x)
    assert torch.equal(q.cpu(), qr) and torch.equal(s.cpu(), sr)


def test_quantize_ties_go_to_even_in_every_type():
    for dt in TYPES:
        k = torch.arange(-127, 127).float() + 0.5                # amax 127: every value is a tie
        x = torch.cat((k, torch.tensor([127.0]))).to(dt)[None]
        q, s = ops.quantize_rows_i8(x.to(DEV))
        assert s.item() == 1.0 and torch.equal(q.cpu(), quant_ref(x)[0])
        if dt == torch.float32:
            assert torch.equal(q.cpu()[0, :-1].float(), k.round())


def test_quantize_many_ties_and_short_mantissas():
    """Rows of 16-bit types whose largest value has few bits: many quotients are ties, others as near to one as the type allows;
    also at both ends of the range."""
    g = gen(77)
    for dt, bits in ((torch.bfloat16, 8), (torch.float16, 11), (torch.float32, 11)):
        for e in (0, -8, 8) if dt == torch.float16 else (0, -125, -140, 110, -30):
            rows = []
            for _ in range(48):
                ma = int(torch.randint(1, 256, (), generator=g))
                near = ((torch.randint(0, 127, (256,), generator=g).double() * 2 + 1) * ma / 254).to(dt).double()       # the values next to ties
                rows.append(torch.cat((near.clamp(max=ma), torch.tensor([float(ma)], dtype=torch.float64), torch.randint(-ma, ma + 1, (256,), generator=g).double())))
            x = (torch.stack(rows) * 2.0 ** e).to(dt)
            assert bool(x.isfinite().all())
            q, s = ops.quantize_rows_i8(x.to(DEV))
            qr, sr = quant_ref(x)
            assert torch.equal(q.cpu(), qr) and torch.equal(s.cpu(), sr), (dt, e)


def test_quantize_special_rows():
    x = torch.randn(8, 33)
    x[1] = 0
    x[2, 5], x[3, 32], x[4, 0] = float("nan"), float("inf"), -float("inf")
    x[5] = 1e-44
    x[6] = torch.linspace(-3.4e38, 3.4e38, 33)              # its step overflows: the row is not finite
    x[7] = 3.4e38 * torch.linspace(-1, 1, 33)
    q, s = ops.quantize_rows_i8(x.to(DEV))
    q, s = q.cpu(), s.cpu()
    assert s[1] == 0 and not q[1].any() and s[2:5].isnan().all() and not q[2:5].any()
    qr, sr = quant_ref(x)
    assert not x[6].isfinite().all() and s[6].isnan() and not q[6].any()
    for r in (0, 5, 7):
        assert torch.equal(q[r], qr[r]) and s[r] == sr[r]
    y = ops.linear_i8(q.to(DEV), s.to(DEV), torch.ones(4, 33, dtype=torch.int8, device=DEV), torch.ones(4, device=DEV),
                      torch.full((4,), 2.0, device=DEV))
    assert y[[2, 3, 4, 6]].isnan().all() and (y[1] == 2.0).all() and y[[0, 5]].isfinite().all()


def test_quantize_subnormal_and_unaligned_rows():
    for dt in TYPES:
        tiny = torch.arange(1, 34, dtype=torch.float64) * (2.0 ** -133 if dt != torch.float16 else 2.0 ** -24)
        base = torch.stack((tiny, -tiny.flip(0), tiny * 3)).to(dt)
        for cut in (slice(None), slice(1, None), slice(None, None, 2), slice(5, 6)):      # also at odd addresses and strides
            q, s = ops.quantize_rows_i8(base.to(DEV)[:, cut])
            qr, sr = quant_ref(base[:, cut])
            assert torch.equal(q.cpu(), qr) and torch.equal(s.cpu(), sr)


def product_ref(q, s, qw, sw, bias, dt):
    """(result, allowed error) in 64 bits from the integers and the scales that the operator uses."""
    y0 = (q.double() @ qw.double().t()) * (s.double()[:, None] * sw.double()[None])
    y = y0 if bias is None else y0 + bias.double()[None]
    return y, 3.0 * (1 + 4 * U) * U * y0.abs() + (U + HALF_STEP[dt]) * (1 + 4 * U) * y.abs() + 3 * U * HALF_STEP[dt] * y0.abs() + TINY[dt]


LINEAR_SHAPES = [(1, 1, 1), (1, 3, 16), (1, 1000, 64), (2, 257, 1000), (5, 130, 127), (15, 64, 2048), (16, 1024, 1024), (17, 255, 1024), (31, 1000, 513),
                 (32, 96, 4096), (33, 2048, 96), (64, 64, 64), (65, 129, 192), (100, 300, 1025), (128, 512, 256), (200, 255, 1024), (257, 259, 321),
                 (300, 1000, 4096), (513, 70, 128), (1030, 515, 640),
                 (33, 16400, 64), (9, 16384, 160), (16, 16385, 320), (8, 20000, 100), (17, 16385, 144), (64, 17000, 272), (2049, 2100, 192), (4000, 3000, 16), (130, 12300, 80), (48, 20001, 200)]


@pytest.mark.parametrize("M,N,K", LINEAR_SHAPES)
def test_linear(M, N, K):
    g = gen(M * 7 + N * 3 + K)
    for n, (xt, ot, has_bias) in enumerate([(torch.bfloat16, torch.bfloat16, False), (torch.float32, torch.float32, True), (torch.float16, torch.float16, True),
                                            (torch.bfloat16, torch.float32, True)]):
        x = torch.randn(M, K, generator=g).to(xt)
        qw = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8)
        sw = torch.rand(N, generator=g) * 0.01
        bias = torch.randn(N, generator=g) if has_bias else None
        d = [t.to(DEV) if t is not None else None for t in (x, qw, sw, bias)]
        got = ops.linear_w8a8(*d, out_dtype=ot)
        assert got.dtype == ot and got.shape == (M, N)
        q, s = quant_ref(x)
        ref, tol = product_ref(q, s, qw, sw, bias, ot)
        off = (got.cpu().double() - ref).abs()
        assert bool((off <= tol).all()), "%d of %d off, worst %g of the tolerance" % (int((off > tol).sum()), M * N, float((off / tol).max()))
        two = ops.linear_i8(*ops.quantize_rows_i8(d[0]), d[1], d[2], d[3], out_dtype=ot)
        assert torch.equal(got, two), "one call and two calls give the same bits"


@pytest.mark.parametrize("M", [1, 40, 300])
def test_linear_extreme_integers_are_exact(M):
    """K = 131072 products of -128 and 127 each stay inside 32 bits; a sum of +-1 over them is exact."""
    K, N = 131072, 3
    q = torch.full((M, K), 127, dtype=torch.int8)
    qw = torch.stack((torch.full((K,), -128), torch.full((K,), 127), torch.where(torch.arange(K) % 2 == 0, 1, -1))).to(torch.int8)
    q[0, 0] = 126
    got = ops.linear_i8(q.to(DEV), torch.ones(M, device=DEV), qw.to(DEV), torch.ones(N, device=DEV)).cpu().double()
    ref = q.double() @ qw.double().t()
    assert bool(((got - ref).abs() <= U * ref.abs()).all())       # one conversion to fp32


@pytest.mark.parametrize("M,N,K", [(65, 255, 16), (66, 256, 240), (80, 1, 256), (97, 17, 272), (4097, 100, 512), (1000, 33, 528), (8200, 255, 1008),
                                   (12289, 256, 1024), (16385, 255, 256), (300, 256, 1024), (65, 257, 1024), (65, 256, 1040), (70, 200, 1000)])
def test_linear_of_few_channels(M, N, K):
    """Up to 256 channels the weights stay on the chip and x passes by: one to many tiles of tokens for each workgroup, every type,
    and the sizes behind the last that go this way."""
    g = gen(M + N + K)
    qw = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8)
    sw, bias = torch.rand(N, generator=g) * 0.01, torch.randn(N, generator=g)
    for xt in TYPES:
        x = (torch.randn(M, K, generator=g) * torch.exp(3 * torch.randn(M, 1, generator=g))).to(xt)
        x[3] = 0
        x[M - 1, K - 1] = float("nan")
        q, s = quant_ref(x)
        for ot, b in zip(TYPES, (bias, None, bias)):
            d = [t.to(DEV) if t is not None else None for t in (x, qw, sw, b)]
            got = ops.linear_w8a8(*d, out_dtype=ot)
            ref, tol = product_ref(q, s, qw, sw, b, ot)
            y = got.cpu().double()
            ok = (y - ref).abs() <= tol
            if ot == torch.float16:                               # from 65520 on, half a step above the largest, fp16 rounds to infinity
                ok |= (ref.abs() + tol >= 65520) & (y == torch.sign(ref) * float("inf"))
            finite = x.isfinite().all(1)                          # a few rows of fp16 hold an infinity themselves
            assert bool(ok[finite].all()) and bool(y[~finite].isnan().all()) and not bool(finite[-1])
            two = ops.linear_i8(*ops.quantize_rows_i8(d[0]), d[1], d[2], d[3], out_dtype=ot)
            assert torch.equal(got[finite.to(DEV)], two[finite.to(DEV)])


@pytest.mark.parametrize("N,K", [(1, 1), (17, 63), (255, 64), (4096, 1024), (4097, 512), (5000, 1000), (16385, 2049), (32000, 640), (65536, 70), (65537, 64),
                                 (5, 32768), (7, 32769), (40001, 513)])
def test_linear_of_one_token(N, K):
    """A single token is quantised by every workgroup for itself: one to several tiles of channels each, odd sizes, every type, and
    the sizes behind the last that go this way."""
    g = gen(N + K)
    qw = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8)
    sw, bias = torch.rand(N, generator=g) * 0.01, torch.randn(N, generator=g)
    W, SW, B = qw.to(DEV), sw.to(DEV), bias.to(DEV)
    for xt in TYPES:
        x = torch.randn(1, K, generator=g).to(xt)
        X = x.to(DEV)
        q, s = quant_ref(x)
        for ot, b, bd in zip(TYPES, (None, bias, None), (None, B, None)):
            got = ops.linear_w8a8(X, W, SW, bd, out_dtype=ot)
            ref, tol = product_ref(q, s, qw, sw, b, ot)
            assert bool(((got.cpu().double() - ref).abs() <= tol).all())
            assert torch.equal(got, ops.linear_i8(*ops.quantize_rows_i8(X), W, SW, bd, out_dtype=ot))
        for value in (float("nan"), -float("inf")):
            X[0, K // 2] = value
            assert bool(ops.linear_w8a8(X, W, SW).isnan().all())
        X.zero_()
        assert torch.equal(ops.linear_w8a8(X, W, SW, B, out_dtype=torch.float32), B[None])


@pytest.mark.parametrize("M,N,K", [(2, 1, 1), (2, 15, 64), (64, 100, 512), (3, 2049, 1000), (5, 5000, 513), (8, 9000, 4096), (9, 4097, 4097), (17, 20001, 70),
                                   (33, 33000, 129), (37, 16401, 1000), (48, 66000, 96), (64, 70001, 513), (16, 32769, 2048), (16, 17000, 4096), (4, 131073, 100),
                                   (64, 33000, 2301), (1, 40001, 4097), (32, 200, 1024), (49, 131075, 65)])
def test_linear_of_few_tokens(M, N, K):
    """2 to 64 tokens that a workgroup holds all at once, quantised by itself or before: one to sixteen waves for a tile of channels, one
    to several tiles for a wave, odd sizes, every type, nearly all of the LDS."""
    g = gen(M + N + K)
    qw = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8)
    sw, bias = torch.rand(N, generator=g) * 0.01, torch.randn(N, generator=g)
    W, SW, B = qw.to(DEV), sw.to(DEV), bias.to(DEV)
    for xt, ot, b, bd in zip(TYPES, (torch.float16, torch.bfloat16, torch.float32), (None, bias, None), (None, B, None)):
        x = torch.randn(M, K, generator=g).to(xt)
        if M > 2:
            x[1] = 0
            x[2, K - 1] = float("inf")
        X = x.to(DEV)
        q, s = quant_ref(x)
        ref, tol = product_ref(q, s, qw, sw, b, ot)
        ok = x.isfinite().all(1)
        q8, s8 = ops.quantize_rows_i8(X)
        for got in (ops.linear_w8a8(X, W, SW, bd, out_dtype=ot), ops.linear_i8(q8, s8, W, SW, bd, out_dtype=ot)):
            y = got.cpu().double()
            assert bool(((y - ref).abs() <= tol)[ok].all()) and bool(y[~ok].isnan().all())


def test_linear_of_few_tokens_writes_its_rows_only():
    """The same with strides that are no multiple of 16 bytes, through the C ABI: the columns and rows around the result stay, and the
    last channel's weights end where the allocation ends."""
    lib, g = L.lib(), gen(23)
    for M, N, K in ((5, 77, 130), (13, 40000, 99), (1, 300, 75), (37, 17000, 65)):
        x, w = torch.randn(M, K + 3, generator=g), torch.randint(-128, 128, (N * (K + 5),), generator=g, dtype=torch.int8)
        sw = torch.rand(N, generator=g)
        rows = w.as_strided((N, K), (K + 5, 1), 5)
        q, s = quant_ref(x[:, 1:1 + K])
        for ot, code in ((torch.float32, L.VX_DTYPE_F32), (torch.float16, L.VX_DTYPE_F16)):
            ref, tol = product_ref(q, s, rows, sw, None, ot)
            for quantised in (False, True):
                out = torch.full((M + 2, N + 3), 7.0, dtype=ot, device=DEV)
                size = lib.vx_linear_i8_workspace_bytes if quantised else lib.vx_linear_w8a8_workspace_bytes
                nb = size(M, N, K)
                ws, X, W, SW = torch.empty(nb, dtype=torch.uint8, device=DEV), x.to(DEV), w.to(DEV), sw.to(DEV)
                to = out.data_ptr() + (N + 3) * out.element_size()
                if quantised:
                    Q, S = q.to(DEV), s.to(DEV)
                    rc = lib.vx_linear_i8(Q.data_ptr(), K, S.data_ptr(), M, W.data_ptr() + 5, K + 5, SW.data_ptr(), N, K, None, to, code, N + 3,
                                          ws.data_ptr(), nb, L.stream_ptr(DEV))
                else:
                    rc = lib.vx_linear_w8a8(X.data_ptr() + 4, L.VX_DTYPE_F32, K + 3, M, W.data_ptr() + 5, K + 5, SW.data_ptr(), N, K, None, to, code, N + 3,
                                            ws.data_ptr(), nb, L.stream_ptr(DEV))
                assert rc == 0
                got = out.cpu().double()
                assert bool(((got[1:-1, :N] - ref).abs() <= tol).all())
                assert bool((got[0] == 7).all()) and bool((got[-1] == 7).all()) and bool((got[:, N:] == 7).all())


def test_linear_of_few_channels_writes_its_rows_only():
    """Strides of every operand, none a multiple of 16 bytes, through the C ABI: the columns and rows around the result stay."""
    lib, g = L.lib(), gen(19)
    M, N, K = 1003, 77, 144
    x, w = torch.randn(M, 151, generator=g), torch.randint(-128, 128, (N, 150), generator=g, dtype=torch.int8)
    sw = torch.rand(N, generator=g)
    for ot, code in ((torch.float32, L.VX_DTYPE_F32), (torch.bfloat16, L.VX_DTYPE_BF16)):
        out = torch.full((M + 2, 83), 7.0, dtype=ot, device=DEV)
        nb = lib.vx_linear_w8a8_workspace_bytes(M, N, K)
        ws, X, W, SW = torch.empty(nb, dtype=torch.uint8, device=DEV), x.to(DEV), w.to(DEV), sw.to(DEV)
        rc = lib.vx_linear_w8a8(X.data_ptr() + 4, L.VX_DTYPE_F32, 151, M, W.data_ptr() + 3, 150, SW.data_ptr(), N, K, None,
                                out.data_ptr() + 83 * out.element_size(), code, 83, ws.data_ptr(), nb, L.stream_ptr(DEV))
        assert rc == 0
        q, s = quant_ref(x[:, 1:1 + K])
        ref, tol = product_ref(q, s, w[:, 3:3 + K], sw, None, ot)
        got = out.cpu().double()
        assert bool(((got[1:-1, :N] - ref).abs() <= tol).all())
        assert bool((got[0] == 7).all()) and bool((got[-1] == 7).all()) and bool((got[:, N:] == 7).all())


def test_linear_offsets_beyond_32_bits():
    """More than 2^31 weights: the last channels are found by the streaming and by the tile kernel."""
    N, K = 530000, 4096
    qw = torch.zeros(N, K, dtype=torch.int8, device=DEV)
    qw[-2:] = torch.tensor([[3], [-5]], dtype=torch.int8, device=DEV)
    for M in (1, 130):
        y = ops.linear_i8(torch.ones(M, K, dtype=torch.int8, device=DEV), torch.ones(M, device=DEV), qw, torch.ones(N, device=DEV), out_dtype=torch.bfloat16)
        assert y[:, -2].tolist() == [3.0 * K] * M and y[:, -1].tolist() == [-5.0 * K] * M and not y[:, :-2].any()


def test_linear_through_the_c_abi_with_unaligned_rows():
    """What ops copies first, a C caller may pass: weights at an odd address and stride, M beyond the streaming kernel's sizes."""
    lib, g = L.lib(), gen(6)
    M, N, K = 150, 70, 64
    q = torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int8)
    s, sw = torch.rand(M, generator=g), torch.rand(N, generator=g)
    wide = torch.randint(-128, 128, (N, 75), generator=g, dtype=torch.int8)
    out = torch.empty(M, N, device=DEV)
    nb = lib.vx_linear_i8_workspace_bytes(M, N, K)
    ws = torch.empty(nb, dtype=torch.uint8, device=DEV)
    Q, S, W, SW = (t.to(DEV) for t in (q, s, wide, sw))
    rc = lib.vx_linear_i8(Q.data_ptr(), K, S.data_ptr(), M, W.data_ptr() + 3, 75, SW.data_ptr(), N, K, None, out.data_ptr(), L.VX_DTYPE_F32, N,
                          ws.data_ptr(), nb, L.stream_ptr(DEV))
    assert rc == 0
    ref, tol = product_ref(q, s, wide[:, 3:3 + K], sw, None, torch.float32)
    assert bool(((out.cpu().double() - ref).abs() <= tol).all())


def test_linear_strides_and_leading_shapes():
    g = gen(12)
    x = torch.randn(4, 6, 80, generator=g)
    qw = torch.randint(-127, 128, (40, 96), generator=g, dtype=torch.int8)
    sw = torch.rand(80, generator=g)[::2] * 0.01
    bias = torch.randn(2, 40, generator=g)
    X, W, S, B = (t.to(DEV) for t in (x, qw, sw, bias))
    S = sw.to(DEV).repeat_interleave(2)[::2]                      # scales with a stride of two
    for xv, wv, K in ((X[:, :, :64], W[:, :64], 64), (X[:, ::2, 3:53], W[:, 7:57], 50), (X.transpose(0, 1), W[:, :80], 80),
                      (X.transpose(1, 2).contiguous().transpose(1, 2), W[:, 16:], 80), (X[:1].expand(4, 6, 80), W[:, :80], 80)):
        got = ops.linear_w8a8(xv, wv, S, B[1])
        q, s = quant_ref(xv.cpu().reshape(-1, K))
        ref, tol = product_ref(q, s, wv.cpu(), sw, bias[1], torch.float32)
        assert got.shape == xv.shape[:-1] + (40,)
        assert bool(((got.cpu().double().reshape(-1, 40) - ref).abs() <= tol).all())
    assert ops.linear_w8a8(X[:0], W[:, :80], S).shape == (0, 6, 40)
    assert ops.linear_w8a8(X[0, 0], W[:, :80], S).shape == (40,)


def test_linear_refuses_what_does_not_fit():
    x, w, s = torch.zeros(2, 8, device=DEV), torch.zeros(4, 8, dtype=torch.int8, device=DEV), torch.ones(4, device=DEV)
    for call in (lambda: ops.linear_w8a8(x[:, :7], w, s), lambda: ops.linear_w8a8(x, w.float(), s), lambda: ops.linear_w8a8(x, w, s[:3]),
                 lambda: ops.linear_w8a8(x, w, s.double()), lambda: ops.linear_w8a8(x, w, s, s[:3]), lambda: ops.linear_w8a8(x.int(), w, s),
                 lambda: ops.linear_w8a8(x, w, s, out_dtype=torch.float64), lambda: ops.linear_w8a8(x, w.cpu(), s),
                 lambda: ops.linear_i8(w, s[:3], w, s), lambda: ops.linear_w8a8(x, w[:0], s[:0])):
        with pytest.raises(L.VortexHipError):
            call()


def test_int8_head_stands_in_for_linear_layers_and_yolo_convolutions():
    g = gen(2)
    lin = nn.Linear(96, 50)
    x = torch.randn(3, 5, 96, generator=g)
    h = V.Int8Head.from_module(lin.to(DEV))
    q, s = quant_ref(x.reshape(-1, 96))
    qw, sw = quant_ref(lin.weight.detach().cpu())
    ref, tol = product_ref(q, s, qw, sw, lin.bias.detach().cpu(), torch.float32)
    assert bool(((h(x.to(DEV)).cpu().double().reshape(-1, 50) - ref).abs() <= tol).all())
    conv = nn.Conv2d(64, 3 * 12, 1).to(DEV)
    y = torch.randn(2, 64, 13, 13, generator=g)
    layer = V.YoloV3Layer(416, (13, 13), [6, 7, 8], ops.COCO_ANCHORS, 7).to(DEV).eval()
    raw = V.Int8Head.from_module(conv)(y.to(DEV))
    q, s = quant_ref(y.permute(0, 2, 3, 1).reshape(-1, 64))
    qw, sw = quant_ref(conv.weight.detach().cpu().flatten(1))
    ref, tol = product_ref(q, s, qw, sw, conv.bias.detach().cpu(), torch.float32)
    assert raw.shape == (2, 36, 13, 13) and bool(((raw.permute(0, 2, 3, 1).cpu().double().reshape(-1, 36) - ref).abs() <= tol).all())
    assert torch.equal(layer(raw), layer(raw.contiguous()))


# ------------------------------------------------------------------------------------------------ draft verification
def softmax64(row, t):
    row = row.astype(np.float64)
    with np.errstate(invalid="ignore"):
        e = np.where(np.isneginf(row), 0.0, np.exp((row - row.max()) / t))
    return e / e.sum()


def verify_ref(target, tokens, u, draft, lens, temp):
    """The definition, sequence by sequence, in 64 bits: (tokens, counts, accept, status, distance of each draw from a border)."""
    B, K = tokens.shape
    Vn = target.shape[2]
    out, counts, accept, status, margin = np.full((B, K + 1), -1), np.zeros(B, int), np.zeros((B, K)), np.zeros(B, int), np.ones(B)
    for b in range(B):
        n = K if lens is None else min(max(int(lens[b]), 0), K)
        t = float(temp[b])
        greedy = not t > 0

        def state(row):
            if np.isnan(row).any() or np.isposinf(row).any():
                return L.VX_STATUS_NAN
            return L.VX_STATUS_EMPTY_ROW if np.isneginf(row).all() else 0
        ts = [state(target[b, j]) for j in range(n + 1)]
        ds = [state(draft[b, j]) if draft is not None and not greedy else 0 for j in range(n)]
        acc, going = 0, True
        dist = [None] * n
        for j in range(n):
            x = int(tokens[b, j])
            ok, ratio = False, 0.0
            inside = 0 <= x < Vn
            if not inside:
                status[b] |= L.VX_STATUS_BAD_TOKEN
            if greedy:
                ok = not ts[j] and inside and int(np.argmax(target[b, j])) == x
                ratio = float(ok)
            elif not ts[j] and not ds[j]:
                q = softmax64(draft[b, j], t) if draft is not None else np.eye(1, Vn, x if inside else Vn)[0]
                dist[j] = q
                if inside:
                    p = softmax64(target[b, j], t)
                    ok = float(u[b, j]) * q[x] < p[x]
                    ratio = (1.0 if p[x] > 0 else 0.0) if p[x] >= q[x] else p[x] / q[x]
                    margin[b] = min(margin[b], abs(float(u[b, j]) * q[x] - p[x]) / max(p[x], 1e-300)) if p[x] > 0 else margin[b]
            accept[b, j] = ratio
            going = going and ok
            acc += going
        status[b] |= int(np.bitwise_or.reduce(ts + ds + [0]))
        out[b, :acc] = tokens[b, :acc]
        counts[b] = acc + 1
        if ts[acc] or (acc < n and ds[acc]):
            continue
        if greedy:
            out[b, acc] = int(np.argmax(target[b, acc]))
            continue
        r = softmax64(target[b, acc], t)
        if acc < n:
            r2 = np.maximum(r - dist[acc], 0.0)
            r = r2 if r2.sum() > 0 else r
        c = np.cumsum(r)
        goal = float(u[b, K]) * c[-1]
        out[b, acc] = min(int((c <= goal).sum()), int(np.nonzero(r)[0][-1]))
        near = np.abs(c[:-1][r[1:] > 0] - goal) / c[-1] if Vn > 1 else np.array([])
        margin[b] = min([margin[b]] + near.tolist())
    return out, counts, accept, status, margin


def check_verify(target, tokens, u, draft, lens, temp, dev_args=None):
    d = dev_args or {}
    got = ops.verify_drafts(d.get("target", target.to(DEV)), tokens.to(DEV), u.to(DEV),
                            draft_logits=d.get("draft", draft.to(DEV) if draft is not None else None),
                            draft_lens=lens.to(DEV) if lens is not None else None, temperature=temp.to(DEV))
    ref = verify_ref(target.float().numpy(), tokens.numpy(), u.numpy(), draft.float().numpy() if draft is not None else None,
                     lens.numpy() if lens is not None else None, temp.numpy())
    # the inputs are not next to a border (fp64 sums of V terms are within V 2^-53 of each other)
    clear = ref[4] > 4 * max(target.shape[2], 64) * 2.0 ** -53
    tok, cnt, acc, st = (t.cpu().numpy() for t in got)
    assert clear.all(), "an input next to a border"
    assert (cnt == ref[1]).all() and (st == ref[3]).all() and (tok == ref[0]).all()
    assert (np.abs(acc - ref[2]) <= 2.0 ** -15 * ref[2] + 2.0 ** -149).all()
    return tok, cnt


def verify_inputs(B, K, Vn, dt, seed, drift=0.7, greedy=0.3):
    g = gen(seed)
    target = (torch.randn(B, K + 1, Vn, generator=g) * 2).to(dt)
    draft = (target[:, :K].float() + drift * torch.randn(B, K, Vn, generator=g)).to(dt)
    temp = torch.where(torch.rand(B, generator=g) < greedy, torch.zeros(B), 0.4 + torch.rand(B, generator=g))
    t = temp.clamp_min(0.05)[:, None, None]
    noise = -torch.log(-torch.log(torch.rand(B, K, Vn, generator=g).clamp(1e-9, 1 - 1e-7)))
    tokens = (draft.float() / t + noise).argmax(-1) if K else torch.zeros(B, 0, dtype=torch.int64)
    return target, tokens, torch.rand(B, K + 1, generator=g), draft, torch.randint(0, K + 1, (B,), generator=g, dtype=torch.int32), temp


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("B,K,Vn", [(1, 0, 1), (3, 0, 50), (2, 1, 2), (5, 1, 63), (7, 3, 64), (4, 8, 257), (9, 4, 1000), (3, 5, 4097), (6, 2, 8191), (2, 3, 16384), (3, 2, 50021)])
def test_verify(dt, B, K, Vn):
    target, tokens, u, draft, lens, temp = verify_inputs(B, K, Vn, dt, B * 100 + K * 10 + Vn)
    check_verify(target, tokens, u, draft, None, temp)
    check_verify(target, tokens, u, draft, lens, temp)
    check_verify(target, tokens, u, None, lens, temp)
    check_verify(target, tokens, u, draft, torch.tensor([K + 5, -3] * B)[:B].int(), torch.full((B,), 0.9))


def test_verify_masks_and_the_types_lowest_value():
    for dt in TYPES:
        target, tokens, u, draft, _, _ = verify_inputs(6, 3, 700, dt, 77, greedy=0.0)
        temp = torch.tensor([0.0, 1.0, 0.6, 1.3, 1.0, 0.8])
        target[:, :, 100:] = -float("inf")                  # masked in the target, not in the draft
        draft[1:3, :, :50] = -float("inf")                  # and the other way round
        target[3:, :, 50:100] = torch.finfo(dt).min
        target[4, 1] = torch.finfo(dt).min                  # a flat row
        draft[5, 0] = torch.finfo(dt).min
        draft[5, 0, 7] = torch.finfo(dt).max
        tokens[3:] = tokens[3:] % 100
        check_verify(target, tokens, u, draft, None, temp)
        check_verify(target, tokens, u, None, None, temp)


def test_verify_one_token_left_and_unused_rows():
    """A single token with weight is drawn whatever the uniform; NaN behind n_b is not looked at."""
    Vn = 5000
    target = torch.full((4, 3, Vn), -float("inf"))
    for b, i in enumerate((0, Vn - 1, 1234, 4096)):
        target[b, :, i] = -50.0 + b
    target[:, 2] = float("nan")
    tokens = torch.tensor([[0, 9], [3, 9], [1234, 9], [4095, 9]])
    tokens[:, 1] = 1 << 40
    u = torch.tensor([[0.0, 0.5, 0.0], [0.999999, 0.1, 0.0], [0.5, 0.5, 0.99999994], [0.1, 0.2, 0.99999994]])
    for dt in TYPES:
        tok, cnt, acc, st = ops.verify_drafts(target.to(dt).to(DEV), tokens.to(DEV), u.to(DEV), draft_lens=torch.ones(4, dtype=torch.int32, device=DEV))
        assert tok.tolist() == [[0, 0, -1], [Vn - 1, -1, -1], [1234, 1234, -1], [4096, -1, -1]] and cnt.tolist() == [2, 1, 2, 1]
        assert acc.tolist() == [[1, 0], [0, 0], [1, 0], [0, 0]] and st.tolist() == [0, 0, 0, 0]


def test_verify_reports_invalid_rows():
    Vn, inf, nan = 300, float("inf"), float("nan")
    target, tokens, u, draft, _, _ = verify_inputs(10, 2, Vn, torch.float32, 5, greedy=0.0)
    temp = torch.ones(10)
    temp[8:] = 0.0
    target[0, 0, 17] = nan
    target[1, 1, 299] = inf
    target[2, 2] = -inf
    draft[3, 0, 0] = nan
    draft[4, 1] = -inf
    tokens[5, 0] = Vn
    tokens[6, 1] = -1
    target[7, 0] = nan
    target[8, 1, 3] = nan
    draft[9] = nan                                            # greedy: the draft's logits are not used
    check_verify(target, tokens, u, draft, None, temp)
    st = ops.verify_drafts(target.to(DEV), tokens.to(DEV), u.to(DEV), draft.to(DEV), None, temp.to(DEV))[3].tolist()
    assert st == [1, 1, 64, 1, 64, 32, 32, 1, 1, 0]
    post = V.DraftVerifyPostProcess()
    with pytest.raises(ValueError, match="nan"):
        post(target[:1].to(DEV), tokens[:1].to(DEV), u[:1].to(DEV), draft[:1].to(DEV))
    with pytest.raises(ValueError, match="masked"):
        post(target[2:3].to(DEV), tokens[2:3].to(DEV), u[2:3].to(DEV), draft[2:3].to(DEV))
    with pytest.raises(L.VortexHipError):
        post(target[5:6].to(DEV), tokens[5:6].to(DEV), u[5:6].to(DEV), draft[5:6].to(DEV))
    assert len(post(target[9:].to(DEV), tokens[9:].to(DEV), u[9:].to(DEV), draft[9:].to(DEV), temperature=0.0)) == 1


def test_verify_the_same_distribution_accepts_everything():
    target, _, u, _, _, _ = verify_inputs(4, 5, 999, torch.float32, 6, greedy=0.0)
    tokens = torch.randint(0, 999, (4, 5), generator=gen(1))
    _, cnt, acc, _ = ops.verify_drafts(target.to(DEV), tokens.to(DEV), u.to(DEV), target[:, :5].to(DEV))
    assert cnt.tolist() == [6] * 4 and (acc == 1).all()


def test_verify_uniforms_next_to_the_border():
    """u is p / q to the last bit of fp32 and its neighbours: fp32 sums cannot tell on which side it lies."""
    B, K, Vn = 12, 3, 3000
    target, tokens, u, draft, _, _ = verify_inputs(B, K, Vn, torch.float32, 55, greedy=0.0)
    temp = torch.full((B,), 0.8)
    for b in range(B):
        for j in range(K):
            p = softmax64(target[b, j].numpy(), np.float64(np.float32(0.8)))
            q = softmax64(draft[b, j].numpy(), np.float64(np.float32(0.8)))
            x = int(np.argmax(q - p)) if j != b % K else int(tokens[b, j])
            tokens[b, j] = x
            r = np.float32(p[x] / q[x])
            u[b, j] = min(float(r if b % 3 == 0 else np.nextafter(r, np.float32(b % 3 - 1.5) * 2)), 0.9999)
    check_verify(target, tokens, u, draft, None, temp)
    lone = target.clone()
    for b in range(B):
        for j in range(K):
            u[b, j] = float(np.float32(softmax64(lone[b, j].numpy(), np.float64(np.float32(0.8)))[int(tokens[b, j])]))
    check_verify(lone, tokens, u, None, None, temp)


def test_verify_uniforms_outside_their_range():
    """1 and NaN are not asked for, but end in a token all the same: a rejection, and the last token with a weight."""
    target = torch.full((3, 2, 6000), -float("inf"))
    target[:, :, 17], target[1, :, 5000] = 0.0, 0.0
    u = torch.tensor([[1.0, 1.0], [float("nan"), float("nan")], [2.0, 0.5]])
    for dt in TYPES:
        tok, cnt, _, _ = ops.verify_drafts(target.to(dt).to(DEV), torch.full((3, 1), 17, device=DEV), u.to(DEV))
        assert cnt.tolist() == [1, 1, 1] and tok[:, 0].tolist() == [17, 5000, 17]
        tok, cnt, _, _ = ops.verify_drafts(target.to(dt).to(DEV), torch.full((3, 1), 17, device=DEV), u.to(DEV), target[:, :1].to(dt).to(DEV))
        assert cnt.tolist() == [1, 1, 1] and tok[:, 0].tolist() == [17, 5000, 17]


def test_verify_extreme_temperatures():
    target, tokens, u, draft, _, _ = verify_inputs(4, 2, 400, torch.float32, 9, greedy=0.0)
    target[3, :, 100:] = -float("inf")
    check_verify(target, tokens, u, draft, None, torch.tensor([1e-3, 1e30, 50.0, 1e6]))
    # so cold that only the largest logit weighs; an infinite temperature is flat over what is not masked; NaN is greedy
    cold = ops.verify_drafts(target.to(DEV), tokens.to(DEV), u.to(DEV), None, None, torch.full((4,), 1e-42, device=DEV))
    gr = ops.verify_drafts(target.to(DEV), tokens.to(DEV), u.to(DEV), None, None, torch.tensor([0.0, -1.0, float("nan"), 0.0], device=DEV))
    assert torch.equal(cold[0], gr[0]) and torch.equal(cold[1], gr[1])
    hot = ops.verify_drafts(target[:, :1].to(DEV), tokens[:, :0].to(DEV), u[:, :1].to(DEV), None, None, torch.full((4,), float("inf"), device=DEV))
    n = [400, 400, 400, 100]
    assert hot[0][:, 0].tolist() == [int(float(u[b, 0]) * n[b]) for b in range(4)]


def test_verify_greedy_takes_the_first_of_equal_logits():
    target = torch.zeros(3, 2, 9000)
    target[0, 0, [5000, 7, 8999]] = 1.0
    target[1] = -3.0
    target[2, :, 8192] = 2.0
    tokens = torch.tensor([[7], [1], [8192]])
    tok, cnt, acc, _ = ops.verify_drafts(target.to(DEV), tokens.to(DEV), torch.rand(3, 2, device=DEV), temperature=0)
    assert tok.tolist() == [[7, 0], [0, -1], [8192, 8192]] and cnt.tolist() == [2, 1, 2] and acc.tolist() == [[1], [0], [1]]
    signed = torch.zeros(1, 1, 70)
    signed[0, 0, :3] = -0.0                                   # -0 equals 0: the first index
    assert ops.verify_drafts(signed.to(DEV), tokens[:1, :0].to(DEV), torch.rand(1, 1, device=DEV), temperature=0.0)[0].item() == 0


def test_verify_strided_logits():
    """Slices of padded logits, transposed batches, rows shared by all sequences, a stride along the vocabulary."""
    target, tokens, u, draft, lens, temp = verify_inputs(4, 3, 515, torch.bfloat16, 21)
    pad = torch.full((4, 6, 600), float("nan"), dtype=torch.bfloat16, device=DEV)
    pad[:, 1:5, 3:518] = target.to(DEV)
    check_verify(target, tokens, u, draft, lens, temp, {"target": pad[:, 1:5, 3:518]})
    check_verify(target, tokens, u, draft, lens, temp, {"target": target.to(DEV).transpose(0, 1).contiguous().transpose(0, 1),
                                                         "draft": draft.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)})
    one = draft[:1].expand(4, 3, 515)
    check_verify(target, tokens, u, one.contiguous(), lens, temp, {"draft": draft[:1].to(DEV).expand(4, 3, 515)})


def test_verify_offsets_beyond_32_bits():
    """Rows more than 2^31 elements apart (a view of 4.4 GB)."""
    target, tokens, u, draft, _, temp = verify_inputs(2, 1, 777, torch.bfloat16, 91, greedy=0.0)
    far = torch.empty(2 ** 31 + 4 * 777, dtype=torch.bfloat16, device=DEV)
    view = far.as_strided((2, 2, 777), (2 ** 31 + 777, 777, 1))
    view.copy_(target)
    check_verify(target, tokens, u, draft, None, temp, {"target": view})


def test_verify_calls_at_once_on_two_streams():
    target, tokens, u, draft, lens, temp = (t.to(DEV) for t in verify_inputs(6, 4, 30011, torch.float16, 92))
    ref = ops.verify_drafts(target, tokens, u, draft, lens, temp)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for k in range(6):
        with torch.cuda.stream(streams[k % 2]):
            got.append(ops.verify_drafts(target, tokens, u, draft, lens, temp))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, ref))


def test_verify_draws_follow_the_target():
    """Drafts from q, verified against p: the first new token is distributed as p (total variation of n draws from p itself is
    below sqrt(V / n) with probability > 1 - 1e-6 here)."""
    n, Vn = 60000, 12
    g = gen(4)
    p, q = torch.randn(1, 1, Vn, generator=g), torch.randn(1, 1, Vn, generator=g)
    x = torch.multinomial(torch.softmax(q[0, 0], 0), n, replacement=True, generator=g)[:, None]
    u = torch.rand(n, 2, generator=g)
    tok = ops.verify_drafts(p.expand(n, 2, Vn).to(DEV), x.to(DEV), u.to(DEV), q.expand(n, 1, Vn).to(DEV))[0][:, 0].cpu()
    freq = torch.bincount(tok, minlength=Vn).double() / n
    assert 0.5 * float((freq - torch.softmax(p[0, 0].double(), 0)).abs().sum()) < (Vn / n) ** 0.5


# ------------------------------------------------------------------------------------------------ together
class Net(nn.Module):
    """Stands for the network between the two ends."""
    task = "detection"
    output_format = {}

    def __init__(self, D, head):
        super().__init__()
        self.w = nn.Parameter(torch.randn(D, D, generator=gen(0)) * D ** -0.5)
        self.head = head

    def forward(self, h):
        return self.head(torch.tanh(h @ self.w))




def test_drafted_decoding_step_through_the_pipeline():
    """ids -> TokenEmbedding -> network -> Int8Head -> DraftVerifyPostProcess, step after step, as Pipeline composes them;
    each end against its definition on what it was given."""
    D, Vn, B, K = 64, 777, 3, 4
    emb = V.TokenEmbedding(Vn, D, scale=8.0).to(DEV)
    lin = nn.Linear(D, Vn, bias=False).to(DEV)
    with torch.no_grad():
        lin.weight.mul_(8)
    net = Net(D, V.Int8Head.from_module(lin)).to(DEV)
    post = V.DraftVerifyPostProcess(0.8)
    pipe = V.predictor.Pipeline(net, preprocess=emb, postprocess=post)
    g = gen(33)
    last = torch.randint(0, Vn, (B, 1), generator=g)
    for step in range(3):
        drafts = torch.randint(0, Vn, (B, K), generator=g)
        ids = torch.cat((last, drafts), 1).to(DEV)
        logits = net(emb(ids)).detach()
        drafts[:, 0] = logits[:, 0].argmax(-1).cpu()               # so that something is accepted
        ids = torch.cat((last, drafts), 1).to(DEV)
        u = torch.rand(B, K + 1, generator=g)
        new = pipe(ids, drafts.to(DEV), u.to(DEV))
        with torch.no_grad():
            h = torch.tanh(emb(ids) @ net.w)
            logits = net.head(h)
        assert torch.equal(emb(ids).detach().cpu(), emb.weight.detach().cpu()[ids.cpu()] * 8.0)
        q, s = quant_ref(h.cpu().reshape(-1, D))
        ref, tol = product_ref(q, s, net.head.qweight.cpu(), net.head.weight_scale.cpu(), None, torch.float32)
        assert bool(((logits.cpu().double().reshape(-1, Vn) - ref).abs() <= tol).all())
        tok, cnt = check_verify(logits.cpu(), drafts, u, None, None, torch.full((B,), 0.8))
        assert [t.tolist() for t in new] == [tok[b, :cnt[b]].tolist() for b in range(B)]
        last = torch.tensor([[int(t[-1])] for t in new])


def test_captured_step_replays_with_new_inputs():
    """One captured graph of all three operators and the gradient, replayed with other inputs between eager work."""
    D, Vn, B, K = 96, 1500, 4, 3
    g = gen(9)
    table = torch.randn(Vn, D, generator=g).to(DEV)
    qw, sw = ops.quantize_rows_i8(torch.randn(Vn, D, generator=g).to(DEV))
    ids, drafts, u = torch.zeros(B, K + 1, dtype=torch.int64, device=DEV), torch.zeros(B, K, dtype=torch.int64, device=DEV), torch.zeros(B, K + 1, device=DEV)
    temp = torch.tensor([0.7, 0.0, 1.0, 1.2], device=DEV)

    def step():
        h = ops.embed_tokens(ids, table, 2.0)
        logits = ops.linear_w8a8(h, qw, sw)
        return (h, logits) + ops.verify_drafts(logits, drafts, u, None, None, temp) + (ops.embed_tokens_grad(ids, h, Vn),)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for gr in graphs:
        with torch.cuda.graph(gr):
            outs.append(step())
    for k in range(5):
        ids.copy_(torch.randint(-1, Vn, (B, K + 1), generator=g))
        drafts.copy_(torch.randint(0, Vn, (B, K), generator=g))
        u.copy_(torch.rand(B, K + 1, generator=g))
        graphs[0].replay()
        graphs[1].replay()
        eager = step()
        torch.cuda.synchronize()
        for o in outs:
            for a, b in zip(o, eager):
                assert torch.equal(a, b), "replay %d" % k


def test_operators_on_another_stream_than_their_tensors():
    side = torch.cuda.Stream()
    g = gen(14)
    table, ids = torch.randn(3000, 512, generator=g).to(DEV), torch.randint(0, 3000, (4000,), generator=g).to(DEV)
    ref = ops.embed_tokens(ids, table)
    gref = ops.embed_tokens_grad(ids, ref, 3000)
    torch.cuda.synchronize()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.embed_tokens(ids, table)
        grad = ops.embed_tokens_grad(ids, got, 3000)
    here = ops.embed_tokens_grad(ids, ref, 3000)                  # at the same time on the first stream
    torch.cuda.synchronize()
    assert torch.equal(got, ref) and torch.equal(grad, gref) and torch.equal(here, gref)
