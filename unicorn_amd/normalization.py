"""Layer normalisation of latents and tokens on the HIP kernels `ur_layer_norm_forward / _backward`: the networks that
predict shape, texture and candidate poses (the reference's heads, unicorn.py:246-304) normalise what they read.

    layer_norm(x, weight=None, bias=None, eps=1e-5)     y = (x - mean) / sqrt(var + eps) * weight + bias, last dimension
    LayerNorm(dim, eps=1e-5, affine=True, bias=True)     the same as a module

x: float32, float16 or bfloat16, any shape and strides (rows with a dense last dimension and an even spacing are read where
they lie, others are copied first); weight and bias have x's type or float32.  Statistics and sums are float32, the
result is rounded once.  The gradients of weight and bias are summed in a fixed order, at most 128 rows one after the other in
float32 and those sums in 64 bits: the same call gives the same bits.
No rows give an empty result and zero parameter gradients.  A row that holds an infinity or a NaN becomes NaN; one whose
squares pass float32's range (numbers beyond 1e19) has no variance: NaN, or the bias.
"""
import torch
from torch import nn

from . import native


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Normalises the last dimension of x.  -> a contiguous tensor of x's shape and type."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"layer_norm needs a last dimension of at least 1, got shape {tuple(x.shape)}")
    native.check_type(x, "x")
    dtype = None
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.dim() != 1 or p.shape[0] != x.shape[-1]:
            raise ValueError(f"{name} must have shape ({x.shape[-1]},), got {tuple(p.shape)}")
        if p.dtype is not x.dtype and p.dtype is not torch.float32:
            raise ValueError(f"{name} must be {x.dtype} or float32, got {p.dtype}")
        if dtype is not None and p.dtype is not dtype:
            raise ValueError("weight and bias must have the same type")
        dtype = p.dtype
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    native.on_gpu(x)
    weight = weight if weight is None or weight.is_contiguous() else weight.contiguous()
    bias = bias if bias is None or bias.is_contiguous() else bias.contiguous()
    return native.nodes().layer_norm(x, weight, bias, eps)


class LayerNorm(nn.Module):
    """layer_norm over the last dimension of size `dim`, with its parameters (weight 1, bias 0 at the start)."""

    def __init__(self, dim, eps=1e-5, affine=True, bias=True, device=None, dtype=None):
        super().__init__()
        if dim < 1:
            raise ValueError(f"dim must be at least 1, got {dim}")
        self.dim, self.eps = int(dim), float(eps)
        self.weight = nn.Parameter(torch.ones(dim, device=device, dtype=dtype)) if affine else None
        self.bias = nn.Parameter(torch.zeros(dim, device=device, dtype=dtype)) if affine and bias else None

    def forward(self, x):
        if x.shape[-1] != self.dim:
            raise ValueError(f"expected a last dimension of {self.dim}, got {tuple(x.shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return f"{self.dim}, eps={self.eps}, affine={self.weight is not None}, bias={self.bias is not None}"
