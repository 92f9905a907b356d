"""Token-model operators (embedding and its gradient, 8-bit product, draft verification): host-side refusals of the C ABI
and of the functional layer.  No GPU: nothing is launched."""
import pytest
import torch

import vortex_amd as V
from vortex_amd import _lib as L
from vortex_amd import ops

P = 1 << 20                                   # a fake, aligned, non-null address; never dereferenced on the host
BIG = 1 << 50


def test_embed_refusals():
    f = L.lib().vx_embed_tokens
    ok = [P, 8, 4, P, 10, 16, 16, 2, 1.0, P, None, None]

    def rc(**kw):
        a = list(ok)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return f(*a)
    for i in (0, 3, 9):
        assert rc(**{"a%d" % i: None}) == -1
    assert rc(a1=2) == -1 and rc(a2=0) == -1 and rc(a4=0) == -1 and rc(a5=0) == -1 and rc(a6=15) == -1 and rc(a7=3) == -1
    assert rc(a2=1 << 30) == -2 and rc(a4=1 << 30) == -2 and rc(a5=(1 << 20) + 1, a6=1 << 21) == -2
    assert rc(a0=P + 4) == -5 and rc(a3=P + 1) == -5 and rc(a9=P + 1) == -5 and rc(a10=P + 2) == -5


def test_embed_grad_refusals():
    lib = L.lib()
    nb = lib.vx_embed_tokens_grad_workspace_bytes(4, 10, 16)
    assert nb > 0 and lib.vx_embed_tokens_grad_workspace_bytes(0, 10, 16) == 0
    assert lib.vx_embed_tokens_grad_workspace_bytes(1 << 30, 10, 16) == 0
    ok = [P, 8, 4, P, 2, 10, 16, 1.0, P, 2, 0, None, P, nb, None]

    def rc(**kw):
        a = list(ok)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return lib.vx_embed_tokens_grad(*a)
    for i in (0, 3, 8, 12):
        assert rc(**{"a%d" % i: None}) == -1
    assert rc(a1=3) == -1 and rc(a2=0) == -1 and rc(a4=7) == -1 and rc(a5=0) == -1 and rc(a6=0) == -1 and rc(a9=-1) == -1
    assert rc(a2=1 << 30, a13=BIG) == -2 and rc(a5=1 << 30, a13=BIG) == -2
    assert rc(a4=1, a9=2) == -2 and rc(a4=0, a9=2) == -2              # f16 -> bf16 and f32 -> bf16 tables
    assert rc(a13=nb - 1) == -3
    assert rc(a3=P + 1) == -5 and rc(a8=P + 1) == -5 and rc(a12=P + 128) == -5 and rc(a0=P + 4) == -5


def test_linear_refusals():
    lib = L.lib()
    assert lib.vx_quantize_rows_i8(None, 0, 1, 4, 4, P, 4, P, None) == -1
    assert lib.vx_quantize_rows_i8(P, 0, 1, 4, 3, P, 4, P, None) == -1
    assert lib.vx_quantize_rows_i8(P, 0, 1, 4, 4, P, 3, P, None) == -1
    assert lib.vx_quantize_rows_i8(P, 5, 1, 4, 4, P, 4, P, None) == -1
    assert lib.vx_quantize_rows_i8(P, 0, 1, 131073, 131073, P, 131073, P, None) == -2
    assert lib.vx_quantize_rows_i8(P + 2, 0, 1, 4, 4, P, 4, P, None) == -5
    nb = lib.vx_linear_w8a8_workspace_bytes(3, 5, 7)
    n8 = lib.vx_linear_i8_workspace_bytes(3, 5, 7)
    assert nb > n8 > 0 and lib.vx_linear_i8_workspace_bytes(3, 5, 131073) == 0 and lib.vx_linear_w8a8_workspace_bytes(0, 5, 7) == 0
    ok = [P, 7, P, 3, P, 7, P, 5, 7, None, P, 0, 5, P, nb, None]

    def i8(**kw):
        a = list(ok)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return lib.vx_linear_i8(*a)
    for i in (0, 2, 4, 6, 10, 13):
        assert i8(**{"a%d" % i: None}) == -1
    assert i8(a1=6) == -1 and i8(a5=6) == -1 and i8(a12=4) == -1 and i8(a11=3) == -1 and i8(a3=0) == -1 and i8(a7=0) == -1 and i8(a8=0) == -1
    assert i8(a8=131073, a1=131073, a5=131073, a14=BIG) == -2 and i8(a3=1 << 23, a14=BIG) == -2 and i8(a7=1 << 23, a12=1 << 23, a14=BIG) == -2
    assert i8(a14=n8 - 1) == -3 and i8(a6=P + 2) == -5 and i8(a9=P + 2) == -5 and i8(a10=P + 2) == -5 and i8(a2=P + 1) == -5 and i8(a13=P + 8) == -5
    w = [P, 2, 7, 3, P, 7, P, 5, 7, None, P, 0, 5, P, nb, None]
    assert lib.vx_linear_w8a8(*(w[:14] + [nb - 1, None])) == -3
    assert lib.vx_linear_w8a8(*([P, 9] + w[2:])) == -1 and lib.vx_linear_w8a8(*([P + 1] + w[1:])) == -5


def test_verify_refusals():
    lib = L.lib()
    nb = lib.vx_verify_drafts_workspace_bytes(2, 3, 100)
    assert nb > 0 and lib.vx_verify_drafts_workspace_bytes(2, 65, 100) == 0 and lib.vx_verify_drafts_workspace_bytes(0, 3, 100) == 0
    assert lib.vx_verify_drafts_workspace_bytes(65536, 3, 100) == 0 and lib.vx_verify_drafts_workspace_bytes(2, 0, 100) > 0
    ok = [P, 400, 100, P, 300, 100, 2, P, None, P, P, 1.0, 2, 3, 100, P, P, P, P, P, nb, None]

    def rc(**kw):
        a = list(ok)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return lib.vx_verify_drafts(*a)
    for i in (0, 7, 9, 15, 16, 17, 18, 19):
        assert rc(**{"a%d" % i: None}) == -1
    assert rc(a6=4) == -1 and rc(a12=0) == -1 and rc(a13=-1) == -1 and rc(a14=0) == -1 and rc(a2=-1) == -1 and rc(a5=-1) == -1
    assert rc(a12=65536, a20=BIG) == -2 and rc(a13=65, a20=BIG) == -2 and rc(a14=1 << 30, a20=BIG) == -2
    assert rc(a20=nb - 1) == -3
    assert rc(a0=P + 1) == -5 and rc(a3=P + 1) == -5 and rc(a7=P + 4) == -5 and rc(a15=P + 4) == -5 and rc(a8=P + 2) == -5 and rc(a19=P + 64) == -5


def test_functional_layer_refuses_cpu_tensors():
    ids, table = torch.zeros(3, dtype=torch.int64), torch.zeros(5, 4)
    q, s = torch.zeros(3, 4, dtype=torch.int8), torch.zeros(3)
    for call in (lambda: ops.embed_tokens(ids, table), lambda: ops.embed_tokens_grad(ids, torch.zeros(3, 4), 5),
                 lambda: ops.quantize_rows_i8(torch.zeros(3, 4)), lambda: ops.linear_i8(q, s, q, s),
                 lambda: ops.linear_w8a8(torch.zeros(3, 4), q, s),
                 lambda: ops.verify_drafts(torch.zeros(1, 2, 4), ids[None, :1], torch.zeros(1, 2)),
                 lambda: V.TokenEmbedding(5, 4)(ids), lambda: V.Int8Head.from_module(torch.nn.Linear(4, 3)),
                 lambda: V.DraftVerifyPostProcess()(torch.zeros(1, 2, 4), ids[None, :1], torch.zeros(1, 2)),
                 lambda: ops.embed_tokens([1, 2], table), lambda: ops.embed_tokens(ids.float(), table)):
        with pytest.raises(L.VortexHipError):
            call()


def test_int8_head_takes_linear_layers_and_1x1_convolutions_only():
    for m in (torch.nn.Conv2d(4, 4, 3), torch.nn.Conv2d(4, 4, 1, stride=2), torch.nn.Conv2d(4, 4, 1, groups=2),
              torch.nn.Conv2d(4, 4, 1, padding=1), torch.nn.ReLU()):
        with pytest.raises(RuntimeError, match="Int8Head takes"):
            V.Int8Head.from_module(m)


def test_int8_head_keeps_fp32_scales_when_the_network_is_halved():
    h = V.Int8Head(torch.zeros(3, 4, dtype=torch.int8), torch.full((3,), 1.0001), torch.ones(3))
    h.half()
    assert torch.equal(h.weight_scale, torch.full((3,), 1.0001))
    assert h.qweight.dtype == torch.int8 and h.weight_scale.dtype == torch.float32 and h.bias.dtype == torch.float32
    assert set(h.state_dict()) == {"qweight", "weight_scale", "bias"}


def test_status_bits_become_errors():
    with pytest.raises(ValueError):
        ops.raise_on_status(L.VX_STATUS_NAN)
    with pytest.raises(ValueError):
        ops.raise_on_status(L.VX_STATUS_EMPTY_ROW)
    with pytest.raises(L.VortexHipError):
        ops.raise_on_status(L.VX_STATUS_BAD_TOKEN)
    assert not ops.status_ok(L.VX_STATUS_BAD_TOKEN) and not ops.status_ok(L.VX_STATUS_EMPTY_ROW)
