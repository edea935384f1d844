"""Linear layers in microscaled 4-bit floating point, beside the bit-sliced ones.

The bit-sliced layer keeps 7- and 6-bit integers and the reference's exact arithmetic; here both sides are e2m1 (4 bits) under block
scales, which the tensor cores multiply directly: about half the weight bytes, four times the rate of 16-bit products.

* ``mxfp4``: blocks of 32 with a power-of-two scale, 4.25 bits an element;
* ``nvfp4``: blocks of 16 with an e4m3 scale, 4.5 bits, and a power of two per row, so that a row's values depend on that row alone.

``quantize_fp4`` packs a matrix, ``fp4_linear`` multiplies activations (packed on the fly) with a packed weight, ``FP4Linear`` is the
layer, and ``quantize_model_fp4`` swaps a model's linears for it by the rules of ``quantize_model_bsi``. Nothing is recorded for
gradients, as with the bit-sliced layer. There is no CPU path.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch
from torch import nn

from .linear import _ops, quantize_model_bsi

FORMATS = {"mxfp4": 0, "nvfp4": 1}
_BLOCK = {"mxfp4": 32, "nvfp4": 16}


def _format(name: str) -> int:
    if name not in FORMATS:
        raise ValueError(f"format must be 'mxfp4' or 'nvfp4', got {name!r}")
    return FORMATS[name]


class FP4Matrix(NamedTuple):
    """A packed matrix [rows, features]; see include/bsi_b200.h for the layout of its bytes."""
    codes: torch.Tensor                  # uint8 [rows, bytes]
    scales: torch.Tensor                 # uint8, tiles of 128 rows x 4 blocks
    row_scale: Optional[torch.Tensor]    # float32 [rows], nvfp4 only
    features: int
    format: str
    dtype: torch.dtype                   # of the matrix that was packed

    @property
    def shape(self):
        return torch.Size((self.codes.shape[0], self.features))

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel() + (0 if self.row_scale is None else 4 * self.row_scale.numel())

    def dequantize(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """The values that the codes stand for, in ``dtype`` (the packed matrix's own by default)."""
        return _ops().fp4_dequantize(self.codes, self.scales, self.row_scale, self.features, _format(self.format), dtype or self.dtype)

    def _scale_tiles(self) -> torch.Tensor:
        """A view of the scales: row tile, group of blocks, row % 32, row % 128 / 32, block of the group."""
        return self.scales.view(-(-self.codes.shape[0] // 128), -(-self.features // 256) * (64 // _BLOCK[self.format]), 32, 4, 4)

    def block_scales(self) -> torch.Tensor:
        """The block scales as float32 [rows, blocks], without the row scale."""
        rows, blocks = self.codes.shape[0], -(-self.features // _BLOCK[self.format])
        t = self._scale_tiles()
        t = t.permute(0, 3, 2, 1, 4).reshape(t.shape[0] * 128, t.shape[1] * 4)[:rows, :blocks].contiguous()
        return t.view(torch.float8_e8m0fnu if self.format == "mxfp4" else torch.float8_e4m3fn).float()


def quantize_fp4(x: torch.Tensor, format: str = "nvfp4") -> FP4Matrix:
    """Packs ``x`` [..., features] (float32, float16 or bfloat16), leading dimensions as rows. A block (mxfp4) or row (nvfp4) that
    holds an infinity or a NaN stands for NaN. The matrix's tensors share one allocation, and the scales' last tile is only written
    where there are rows."""
    return FP4Matrix(*_ops().fp4_quantize(x, _format(format)), x.shape[-1], format, x.dtype)


def fp4_linear(x: Union[torch.Tensor, FP4Matrix], weight: FP4Matrix, bias: Optional[torch.Tensor] = None, relu: bool = False,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``act(x @ weight.T + bias)`` with ``x`` packed in the weight's format, float32 sums and one rounding to ``out_dtype`` (x's type
    by default). ``x`` may be packed already (``quantize_fp4``): one packing then serves several weights."""
    f = _format(weight.format)
    if isinstance(x, FP4Matrix):
        return _ops().fp4_linear_packed(x.codes, x.scales, x.row_scale, weight.codes, weight.scales, weight.row_scale, x.features,
                                        weight.features, _format(x.format), f, bias, relu, out_dtype or x.dtype)
    return _ops().fp4_linear(x, weight.codes, weight.scales, weight.row_scale, weight.features, f, bias, relu, out_dtype)


class FP4Linear(nn.Module):
    """``nn.Linear`` with a packed weight and activations packed on the fly; its buffers are all that a state dict needs."""

    def __init__(self, original_linear: nn.Linear, format: str = "nvfp4"):
        super().__init__()
        self.in_features, self.out_features, self.format = original_linear.in_features, original_linear.out_features, format
        with torch.no_grad():
            packed = quantize_fp4(original_linear.weight.detach(), format)
        # a copy each, as the packer's outputs share one allocation, and zeros for the scales of rows that are not there, which it
        # leaves as they were: a buffer can be kept or saved by itself, and equal weights have equal state dicts
        packed = FP4Matrix(*(t.clone() if isinstance(t, torch.Tensor) else t for t in packed))
        row = torch.arange(32, device=packed.scales.device)[:, None] + 32 * torch.arange(4, device=packed.scales.device)
        packed._scale_tiles()[-1:][:, :, row > (self.out_features - 1) % 128] = 0
        self.register_buffer("codes", packed.codes)
        self.register_buffer("scales", packed.scales)
        self.register_buffer("row_scale", packed.row_scale)
        bias = original_linear.bias
        self.register_buffer("bias", None if bias is None else bias.detach().to(torch.float32))
        self.weight_dtype = packed.dtype

    @property
    def weight(self) -> FP4Matrix:
        return FP4Matrix(self.codes, self.scales, self.row_scale, self.in_features, self.format, self.weight_dtype)

    def _apply(self, fn, recurse=True):
        # .half() and .to(dtype) are for activations: a row scale and a bias in 16 bits would be other numbers
        kept = {n: b for n, b in self._buffers.items() if n in ("row_scale", "bias") and b is not None}
        super()._apply(fn, recurse)
        for n, b in kept.items():
            if self._buffers[n].dtype != torch.float32:
                self._buffers[n] = b.to(self._buffers[n].device)
        return self

    def forward(self, x):
        return _ops().fp4_linear(x, self.codes, self.scales, self.row_scale, self.in_features, FORMATS[self.format], self.bias, False)

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, format={self.format}"


def quantize_model_fp4(model: nn.Module, format: str = "nvfp4", skip_lm_head: bool = True, scope: str = "all", verbose: bool = True) -> nn.Module:
    """Swaps a model's ``nn.Linear`` modules (on the GPU already) for ``FP4Linear``, picked as ``quantize_model_bsi`` picks them."""
    _format(format)
    quantize_model_bsi(model, skip_lm_head=skip_lm_head, scope=scope, verbose=False, layer_factory=lambda linear, **_: FP4Linear(linear, format))
    if verbose:
        print(f"Quantized {sum(isinstance(m, FP4Linear) for m in model.modules())} linear layers to {format} (scope={scope})")
    return model
