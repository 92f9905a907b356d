"""Calls of the token-model operators that need no GPU to be seen through: layers that are taken, arguments by name."""
import pytest
import torch

import vortex_amd as V
from vortex_amd import _lib as L
from vortex_amd import ops


def test_int8_head_takes_1x1_convolutions_whose_padding_is_none_by_name():
    """"same" and "valid" add nothing to a 1x1 kernel: such layers get as far as the GPU they need."""
    for padding in ("same", "valid"):
        with pytest.raises(L.VortexHipError, match="must live on"):
            V.Int8Head.from_module(torch.nn.Conv2d(4, 4, 1, padding=padding))
    with pytest.raises(RuntimeError, match="Int8Head takes"):
        V.Int8Head.from_module(torch.nn.Conv2d(4, 4, 3, padding="same"))


def test_functional_layer_takes_its_arguments_by_name():
    """As far as a call gets without a GPU: the refusal of tensors on the CPU."""
    ids, table = torch.zeros(3, dtype=torch.int64), torch.zeros(5, 4)
    q, s = torch.zeros(3, 4, dtype=torch.int8), torch.zeros(3)
    for call in (lambda: ops.embed_tokens(ids=ids, table=table), lambda: ops.embed_tokens(scale=2.0, table=table, ids=ids),
                 lambda: ops.embed_tokens_grad(ids=ids, grad_out=torch.zeros(3, 4), n_rows=5), lambda: ops.quantize_rows_i8(x=table),
                 lambda: ops.linear_i8(q=q, scale=s, qw=q, w_scale=s), lambda: ops.linear_w8a8(x=table, qw=q, w_scale=s),
                 lambda: ops.verify_drafts(target_logits=torch.zeros(1, 2, 4), draft_tokens=ids[None, :1], uniforms=torch.zeros(1, 2))):
        with pytest.raises(L.VortexHipError, match="must live on"):
            call()
