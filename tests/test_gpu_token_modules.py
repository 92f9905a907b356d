"""The modules of the token-model operators: what they report."""
import pytest
import torch

import vortex_amd as V
from test_gpu_tokens import DEV
from vortex_amd import _lib as L
from vortex_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("train", [False, True])
def test_token_embedding_reports_ids_beyond_its_table(train):
    m = V.TokenEmbedding(10, 16).to(DEV).requires_grad_(train)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ok = m(torch.tensor([0, 9, -1], device=DEV), status=status)
    ops.raise_on_status(int(status))
    assert torch.equal(ok[:2], m.weight[[0, 9]]) and ok.requires_grad == train
    bad = m(torch.tensor([[3, 10], [1 << 40, 9]], device=DEV), status=status)
    assert int(status) == L.VX_STATUS_BAD_TOKEN and not bad[0, 1].any() and not bad[1, 0].any()
    with pytest.raises(L.VortexHipError, match="vocabulary"):
        ops.raise_on_status(int(status))
    if train:
        bad.sum().backward()
        ref = torch.zeros(10, 16, device=DEV)
        ref[[3, 9]] = 1.0
        assert torch.equal(m.weight.grad, ref)


def test_token_embedding_refuses_a_status_that_is_no_word_on_its_device():
    m, ids = V.TokenEmbedding(10, 16).to(DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    for status in (torch.zeros(1, dtype=torch.int64, device=DEV), torch.zeros(1, dtype=torch.int32), torch.zeros(0, dtype=torch.int32, device=DEV), 0):
        with pytest.raises(L.VortexHipError, match="status"):
            m(ids, status=status)


@pytest.mark.parametrize("padding", ["same", "valid"])
def test_int8_head_of_a_1x1_convolution_whose_padding_is_none_by_name(padding):
    conv = torch.nn.Conv2d(64, 20, 1, padding=padding).to(DEV)
    plain = torch.nn.Conv2d(64, 20, 1).to(DEV)
    plain.load_state_dict(conv.state_dict())
    x = torch.randn(2, 64, 5, 7, device=DEV)
    assert torch.equal(V.Int8Head.from_module(conv)(x), V.Int8Head.from_module(plain)(x))
