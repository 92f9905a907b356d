"""Drop-in for the reference's networks/modules/preprocess/normalizer.py (Normalize :63-77,
FlipNormalize :79-95, get_preprocess :102-121) and preprocess/__init__.py:47-55 (names
`normalizer`, `normalize`, `flip_normalizer`, `flip_normalize`).  The arithmetic runs in the
HIP kernel vx_preprocess_u8hwc_f32nchw; same constructor arguments, buffers, annotations and
assertions as the reference."""
from typing import Optional

import torch
import torch.nn as nn

from . import ops


class Normalize(nn.Module):
    """uint8 NHWC -> float NCHW, ((x / scaler) - mean) / std.  Returns a contiguous NCHW tensor
    (the reference returns an NCHW-shaped view of NHWC memory; values are identical)."""
    __constants__ = ["mean", "std", "scaler"]

    def __init__(self, mean=[0.485, 0.456, 0.406], std=[0.229, 0.224, 0.225], scaler=255):
        super(Normalize, self).__init__()
        self.register_buffer("mean", torch.as_tensor(mean, dtype=torch.float))
        self.register_buffer("std", torch.as_tensor(std, dtype=torch.float))
        self.register_buffer("scaler", torch.as_tensor(scaler, dtype=torch.int))
        self._flip = False
        self._host = None

    def _consts(self):
        # host copies of the (tiny) buffers, read once: they are kernel arguments
        if self._host is None:
            self._host = (self.mean.detach().cpu().tolist(), self.std.detach().cpu().tolist(),
                          int(self.scaler.item()))
        return self._host

    def _apply(self, fn, *a, **k):
        self._host = None
        return super()._apply(fn, *a, **k)

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        # reference to_tensor asserts (normalizer.py:23-26)
        assert len(input.size()) == 4, "to_tensor only support 4-dimension tensor (NHWC) as input, "\
            "got size of %s" % list(input.size())
        assert input.size(3) == 3 or input.size(3) == 1, "to_tensor only support NHWC input layout, "\
            "got size of %s" % list(input.size())
        if self._flip:
            assert input.size(3) == 3, "only supports 3 color channels with HWC format"
        if input.size(3) != 3:
            raise NotImplementedError("libvortex_hip pre-process handles 3-channel images")
        mean, std, scaler = self._consts()
        return ops.preprocess(input, mean, std, scaler, flip=self._flip)


class FlipNormalize(Normalize):
    """Channel reversal (RGB<->BGR) in front of Normalize (normalizer.py:79-95)."""

    def __init__(self, mean=[0.485, 0.456, 0.406], std=[0.229, 0.224, 0.225], scaler=255, flip_dim=-1):
        super(FlipNormalize, self).__init__(mean, std, scaler)
        if flip_dim not in (-1, 3):
            raise NotImplementedError("only the channel dimension can be flipped")
        self.flip_dim = flip_dim
        self._flip = True

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        return super().forward(input)


class _EmbedTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, status):
        ctx.save_for_backward(ids)
        ctx.n_rows, ctx.scale = weight.size(0), scale
        return ops.embed_tokens(ids, weight, scale, status)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        ids, = ctx.saved_tensors
        return None, ops.embed_tokens_grad(ids, grad, ctx.n_rows, ctx.scale), None, None


class TokenEmbedding(nn.Module):
    """The pre-process of a token model: integer ids -> the network's input vectors, scale * weight[ids] (what Normalize
    is for images).  An id below 0 is padding: a row of zeros that gets no gradient.  The gradient of `weight` is summed in
    fp32 over the tokens in a fixed order (vx_embed_tokens_grad), dense, in the type of `weight`.

    An id at or beyond n_rows gives zeros and no gradient as well, since a call does not wait for the GPU to say so.  Where such ids
    can occur, hand over a word for them and look at it when the host waits anyway:

        status = torch.zeros(1, dtype=torch.int32, device=ids.device)
        h = embed(ids, status=status)
        ops.raise_on_status(int(status))               # VortexHipError; VX_STATUS_BAD_TOKEN is ORed in, nothing clears it

    In a captured HIP graph, take the gradient with torch.autograd.grad: a captured backward() accumulates into `weight.grad`
    on the stream of whatever eager graph of `weight` is still alive, which torch answers by ending the process."""

    def __init__(self, n_rows: int, dim: int, scale: float = 1.0, dtype=None, device=None):
        super(TokenEmbedding, self).__init__()
        self.scale = float(scale)
        self.weight = nn.Parameter(torch.empty(n_rows, dim, dtype=dtype, device=device))
        nn.init.normal_(self.weight, std=dim ** -0.5)

    def forward(self, input: torch.Tensor, status: Optional[torch.Tensor] = None) -> torch.Tensor:
        if torch.is_grad_enabled() and self.weight.requires_grad:
            return _EmbedTokens.apply(input, self.weight, self.scale, status)
        return ops.embed_tokens(input, self.weight, self.scale, status)


preproc_map = dict(
    normalizer=Normalize, normalize=Normalize,
    flip_normalizer=FlipNormalize, flip_normalize=FlipNormalize,
)


def get_preprocess(preprocess: str, **kwargs):
    assert preprocess in preproc_map, "unsupported preproc f{preprocess}"
    normalizer = preproc_map[preprocess]
    normalization_args = kwargs["input_normalization"] if "input_normalization" in kwargs else kwargs
    return normalizer(**normalization_args)
