"""Products with 4-bit weights: group scales and zero points, for single tokens up to whole prompts.

The reference quotes its figures on models whose weights are 4-bit and leaves their products to its
host engine; these are extensions with no reference counterpart:

* :class:`QuantizedLinear` — a weight [out_features, in_features] in codes of 4 bits with a 16-bit scale
  and a zero point per group of inputs, laid out once for the kernels;
* :func:`quantized_linear` — ``x @ weight.T + bias``;
* ``triton_kernels.qkv_projection_paged`` and ``partial_prefill_layer_paged`` take a
  :class:`QuantizedLinear` where they take a weight.

A server's calls without a backward pass, as in :mod:`semblend_amd.paged_cache`.
"""

from __future__ import annotations

import functools

import torch

from . import _lib
from .paged_cache import _device, _recorded

__all__ = ["QuantizedLinear", "quantized_linear"]

_ROW_STRIDE_MAX = 1 << 22  # elements (the C ABI's limit, and that of in_features)
_16BIT = (torch.bfloat16, torch.float16)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(*sizes: int) -> int:
    return _lib.size_query("sb_w4_linear_workspace_size", *sizes)


class QuantizedLinear:
    """w[n, k] = (code[n, k] - zero[n, k // group]) * scale[n, k // group].

    codes: [out_features, in_features] uint8 of 0 to 15; scales: [out_features, in_features / group]
    bf16 or fp16; zeros: like scales, uint8 of 0 to 15 (None: 8, symmetric weights). The group is what
    the shapes say: a multiple of 32 that divides in_features (one group a row included). The inputs
    are copied into the kernels' own layout (0.53 bytes a weight with groups of 128) and not kept."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None):
        if codes.dtype != torch.uint8 or (zeros is not None and zeros.dtype != torch.uint8):
            raise TypeError("codes and zeros must be uint8")
        if scales.dtype not in _16BIT:
            raise TypeError("scales must be bf16 or fp16")
        if codes.dim() != 2 or scales.dim() != 2 or 0 in codes.shape or 0 in scales.shape:
            raise ValueError("codes must be [out_features, in_features] and scales [out_features, "
                             "in_features / group]")
        n, k = codes.shape
        groups = scales.shape[1]
        if scales.shape[0] != n or k % groups or k // groups % 32:
            raise ValueError("scales must be [out_features, in_features / group] with a group that "
                             "is a multiple of 32")
        if zeros is not None and zeros.shape != scales.shape:
            raise ValueError("zeros must have the shape of scales")
        dev = _device(codes, (scales, zeros))
        for name, t in (("codes", codes), ("zeros", zeros)):
            if t is not None and int(t.max()) > 15:
                raise ValueError(f"{name} must lie in 0 .. 15")
        self.out_features, self.in_features, self.group = n, k, k // groups
        self.device, self.scale_dtype = dev, scales.dtype
        self.shape = (n, k)
        self._code = _lib.SB_DTYPE[scales.dtype]
        self._packed = torch.empty(_lib.size_query("sb_w4_codes_size", n, k), dtype=torch.uint8,
                                   device=dev)
        self._table = torch.empty(_lib.size_query("sb_w4_table_size", n, k, self.group),
                                  dtype=torch.uint8, device=dev)
        codes, scales = (t if t.stride(1) == 1 else t.contiguous() for t in (codes, scales))
        if zeros is not None and zeros.stride(1) != 1:
            zeros = zeros.contiguous()
        _lib.launch(dev, "sb_w4_pack", self._packed.data_ptr(), self._table.data_ptr(),
                    codes.data_ptr(), scales.data_ptr(), _lib.ptr(zeros), n, k, self.group,
                    codes.stride(0), scales.stride(0), zeros.stride(0) if zeros is not None else 0)

    @classmethod
    def quantize(cls, weight: torch.Tensor, group: int = 128, symmetric: bool = False,
                 scale_dtype: torch.dtype | None = None) -> "QuantizedLinear":
        """The nearest codes to a weight [out_features, in_features]: per group the range from its
        smallest to its largest value and 0 (symmetric: plus and minus the largest magnitude) in 15
        steps of a scale that is rounded to ``scale_dtype`` first (the weight's own, bf16 for fp32)."""
        if weight.dim() != 2 or 0 in weight.shape:
            raise ValueError("weight must be [out_features, in_features]")
        n, k = weight.shape
        if group < 1 or group % 32 or k % group:
            raise ValueError("group must be a multiple of 32 that divides in_features")
        if scale_dtype is None:
            scale_dtype = weight.dtype if weight.dtype in _16BIT else torch.bfloat16
        if scale_dtype not in _16BIT:
            raise TypeError("scale_dtype must be bf16 or fp16")
        _device(weight, ())
        w = weight.detach().float().unflatten(1, (-1, group))
        if not bool(w.isfinite().all()):
            raise ValueError("weight holds values that are not finite")
        if symmetric:
            low = -w.abs().amax(-1)
            scale = (low / -7.5)
        else:
            low = w.amin(-1).clamp(max=0)
            scale = (w.amax(-1).clamp(min=0) - low) / 15
        scale = scale.to(scale_dtype)
        step = scale.float()
        if not bool(step.isfinite().all()):
            raise ValueError("a group's scale is past the range of scale_dtype")
        step = torch.where(step > 0, step, torch.ones_like(step))
        zero = torch.full_like(step, 8.0) if symmetric else (-low / step).round().clamp(0, 15)
        codes = ((w / step[..., None]).round() + zero[..., None]).clamp(0, 15)
        return cls(codes.flatten(1).to(torch.uint8), scale,
                   None if symmetric else zero.to(torch.uint8))

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The weight [out_features, in_features] itself, rounded once to dtype."""
        if dtype not in _lib.SB_DTYPE:
            raise TypeError(f"unsupported dtype {dtype}")
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        _lib.launch(self.device, "sb_w4_dequantize", out.data_ptr(), self._packed.data_ptr(),
                    self._table.data_ptr(), *self.shape, self.group, out.stride(0), self._code,
                    _lib.SB_DTYPE[dtype])
        return out


def quantized_linear(
    x: torch.Tensor,
    weight: QuantizedLinear,
    bias: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``x @ weight.T + bias`` with the exact 4-bit weights, fp32 sums and one rounding.

    x: [..., in_features] bf16 or fp16, any number of rows; bias: [out_features] of x's type; ``out``:
    [..., out_features] of x's type with a unit last stride and rows at one stride (a new tensor by
    default; returned). Range: x finite and below 2^116 in magnitude, scales below 2^122, and an output's
    sum of |x| |scale| below 2^120 (those of fp16 inputs and scales always are): the fp32 sums of a group of
    inputs are up to 31 times as large. A row that holds an infinity or a NaN gives NaN (or infinities), other rows
    are not affected. ``out`` must not overlap x.
    Groups of 128 in bf16: one row of 3584 -> 4608 6.6 us, 8 of 3584 -> 37888 14 (18 where the weights
    are in no cache), 2458 of 3584 -> 4608 91; one of 4096 -> 131072 in fp16 44. Extension with no reference counterpart.
    """
    if not isinstance(weight, QuantizedLinear):
        raise TypeError("weight must be a QuantizedLinear")
    dev = _device(x, (weight._packed, bias, out))
    dtype, shape = x.dtype, x.shape
    if dtype not in _16BIT:
        raise TypeError("x must be bf16 or fp16")
    n, k = weight.shape
    if len(shape) == 0 or shape[-1] != k:
        raise ValueError(f"x must be [..., {k}]")
    if bias is not None and (bias.shape != (n,) or bias.dtype != dtype):
        raise ValueError(f"bias must be [{n}] of x's dtype")
    rows = x if len(shape) == 2 else x.reshape(-1, k)
    num = rows.shape[0]
    new = out is None
    if new:
        out = torch.empty((*shape[:-1], n), dtype=dtype, device=dev)
        out_rows = n
    else:
        if out.shape != (*shape[:-1], n) or out.dtype != dtype or out.stride(-1) != 1:
            raise ValueError("out must be [..., out_features] of x's dtype, with a unit last stride")
        flat = out if out.dim() == 2 else out.view(-1, n)
        out_rows = flat.stride(0)
    if num:
        step = rows.stride(0)
        if rows.stride(1) != 1 or step % 8 or step > _ROW_STRIDE_MAX or rows.data_ptr() % 16:
            rows = rows.clone(memory_format=torch.contiguous_format)
            step = k
        if bias is not None and bias.stride(0) != 1:
            bias = bias.contiguous()
        dt = _lib.SB_DTYPE[dtype]
        ws_bytes = _workspace_bytes(num, n, k, weight.group, dt)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
        _lib.launch(dev, "sb_w4_linear", out.data_ptr(), rows.data_ptr(), weight._packed.data_ptr(),
                    weight._table.data_ptr(), _lib.ptr(bias), num, n, k, weight.group, step, out_rows,
                    _lib.ptr(ws), ws_bytes, weight._code, dt)
    if new and (x.requires_grad or bias is not None and bias.requires_grad):
        return _recorded("quantized_linear", out, x, *(() if bias is None else (bias,)))
    return out
