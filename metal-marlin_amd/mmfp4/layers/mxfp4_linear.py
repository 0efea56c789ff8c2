"""Linear layer on MXFP4 weights, the counterpart of MMFP4Linear (metal_marlin/layers/
mmfp4_linear.py:600-960) whose activations are quantized as well."""

from __future__ import annotations

import torch
import torch.nn as nn

from .. import autograd, mxfp4

__all__ = ["MXFP4Linear"]


class MXFP4Linear(nn.Module):
    """y = q(x) @ W^T (+ bias) in x's type, W MXFP4: packed_weights [out, in/8] words and scales
    uint8 [out, in/32].  As in MMFP4Linear the bias is added to the product in its type: two
    roundings.  Differentiable in x, straight through its rounding; the weights are
    frozen, and a bias that requires a gradient gets it."""

    def __init__(self, packed_weights: torch.Tensor, scales: torch.Tensor,
                 bias: torch.Tensor | None = None) -> None:
        super().__init__()
        words, scales = mxfp4._weights(packed_weights, scales, 2, "packed_weights")
        out_f = words.shape[0]
        if bias is not None and (bias.dim() != 1 or bias.shape[0] != out_f):
            raise ValueError(f"bias must be shape [{out_f}], got shape={tuple(bias.shape)}")
        self.register_buffer("packed_weights", words.contiguous())
        self.register_buffer("scales", scales.contiguous())
        self.register_buffer("bias", None if bias is None else bias.contiguous())
        self.in_features = 8 * words.shape[1]
        self.out_features = out_f

    @classmethod
    def from_linear(cls, linear: nn.Linear, device: torch.device | str | None = None):
        """Quantizes the weight of an nn.Linear; the bias stays as it is."""
        dev = torch.device(device) if device is not None else (
            linear.weight.device if linear.weight.is_cuda else torch.device("cuda"))
        bias = None if linear.bias is None else linear.bias.detach().to(dev)
        return cls(*mxfp4.mxfp4_quantize(linear.weight.detach().to(dev)), bias)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.in_features:
            raise ValueError(f"Expected input last dim={self.in_features}, got {x.shape[-1]}")
        out = mxfp4.mxfp4_gemm(x, self.packed_weights, self.scales)
        if self.bias is not None:
            if self.bias.requires_grad and torch.is_grad_enabled():
                autograd.refuse_foreign_leaf(self.bias)
            out = out + self.bias.to(out.dtype)
        return out

    def input_grad(self, dy: torch.Tensor, dtype: torch.dtype | None = None) -> torch.Tensor:
        """The gradient of the input for dy [*, out] -> [*, in], in dy's type or `dtype`."""
        return mxfp4.mxfp4_gemm_backward(dy, self.packed_weights, self.scales, out_dtype=dtype)
