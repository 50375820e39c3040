"""Products of a few tokens with 4-bit weights: the dense matrices around the routed experts (projections,
shared expert, output head) in a decode step.

    w[n, k] = scale[n, k // group] * (code[n, k] - zero[n, k // group])       codes and zero points 0..15

`W4Weight` lays a matrix out once for the kernels; `linear` and `gated` (gate and up with the routed experts'
SwiGLU, one launch) multiply fp16 or bf16 tokens with it, in fp32 sums of unrounded products. `shared_expert`
adds a shared expert's output to the routed layer's. All work runs on the current CUDA stream, nothing
synchronises the host and nothing but the outputs is allocated, so the calls can be captured in a CUDA graph.
The kernels are made for decode batches: every 32 tokens stream the weights once.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib

_X_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
_OUT_DTYPES = {**_X_DTYPES, torch.float32: _lib.DTYPE_F32}


class W4Weight:
    """A 4-bit matrix [n, k] on the GPU, laid out for the kernels.

    codes: uint8 [n, k / 2], two codes a byte, even k in the low nibble. scales: fp16 or bf16 [n, k / group]
    (group 32, 64 or 128). zeros: uint8 [n, k / group] zero points 0..15, or None: 8 everywhere."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None):
        if codes.dim() != 2 or codes.dtype != torch.uint8:
            raise ValueError("codes must be uint8 [n, k / 2]")
        n, k = codes.shape[0], 2 * codes.shape[1]
        if scales.dim() != 2 or scales.shape[0] != n or scales.dtype not in _X_DTYPES or scales.shape[1] == 0:
            raise ValueError("scales must be fp16 or bf16 [n, k / group]")
        group = k // scales.shape[1]
        if group not in (32, 64, 128) or group * scales.shape[1] != k:
            raise ValueError(f"{scales.shape[1]} scales per row of {k} inputs: groups must be 32, 64 or 128 inputs")
        if not codes.is_cuda or scales.device != codes.device:
            raise ValueError("codes and scales must live on one CUDA device")
        if zeros is not None:
            if zeros.shape != scales.shape or zeros.dtype != torch.uint8 or zeros.device != codes.device:
                raise ValueError("zeros must be uint8 of the scales' shape, on their device")
            if zeros.numel() and int(zeros.max()) > 15:
                raise ValueError("zero points must be 0..15")
            zeros = zeros.contiguous()
        codes, scales = codes.contiguous(), scales.contiguous()
        L = _lib.load()
        size = C.c_size_t()
        _lib.check(L.dsv41_w4_layout_size(n, k, group, int(zeros is not None), C.byref(size)), "dsv41_w4_layout_size")
        self.n, self.k, self.group, self.device = n, k, group, codes.device
        self.data = torch.empty(size.value, dtype=torch.uint8, device=codes.device)
        _lib.call(self.device, L.dsv41_w4_pack, codes.data_ptr(), scales.data_ptr(),
                  zeros.data_ptr() if zeros is not None else None, n, k, group, self.data.data_ptr(), size.value,
                  _lib.current_stream(self.device))
        self._c = _lib.W4WeightC(n, k, group, int(zeros is not None), _X_DTYPES[scales.dtype], self.data.data_ptr())
        self._ref = C.byref(self._c)

    @classmethod
    def quantize(cls, weight: torch.Tensor, group: int = 128, symmetric: bool = True) -> "W4Weight":
        """Round a dense [n, k] matrix to 4 bits: symmetric scales so that the largest magnitude of a group
        lands on code 15 or 1 of 8 +- 7, or asymmetric ones that span the group's range (with zero)."""
        if weight.dim() != 2 or group not in (32, 64, 128) or weight.shape[1] % group:
            raise ValueError("weight must be [n, k] with k a multiple of a group of 32, 64 or 128")
        w = weight.float().reshape(weight.shape[0], -1, group)
        dtype = weight.dtype if weight.dtype in _X_DTYPES else torch.float16
        if symmetric:
            scale = (w.abs().amax(2) / 7.0).clamp_min(1e-6).to(dtype)
            zero = torch.full_like(scale, 8.0, dtype=torch.float32)
        else:
            lo, hi = w.amin(2).clamp_max(0.0), w.amax(2).clamp_min(0.0)
            scale = ((hi - lo) / 15.0).clamp_min(1e-6).to(dtype)
            zero = torch.round(-lo / scale.float()).clamp(0, 15)
        code = torch.round(w / scale.float()[:, :, None] + zero[:, :, None]).clamp(0, 15).to(torch.uint8).view(weight.shape)
        return cls(code[:, 0::2] | (code[:, 1::2] << 4), scale, None if symmetric else zero.to(torch.uint8))


def _rows(x: torch.Tensor, w: W4Weight) -> torch.Tensor:
    """x as [tokens, k] rows the kernels can read: contiguous inputs, 16-byte aligned rows."""
    if x.dtype not in _X_DTYPES:
        raise TypeError(f"unsupported activation dtype {x.dtype} (fp16 or bf16)")
    if x.dim() < 1 or x.shape[-1] != w.k:
        raise ValueError(f"x must be [..., {w.k}]")
    if x.device != w.device:
        raise ValueError("x must live on the weight's device")
    if x.dim() != 2:
        x = x.reshape(-1, w.k)
    if not x.is_contiguous() and (x.stride(1) != 1 or x.stride(0) % 8 or x.stride(0) < w.k):
        x = x.contiguous()
    if x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def _product(fn, weights, x: torch.Tensor, w: W4Weight, out: torch.Tensor | None, out_dtype: torch.dtype | None,
             tail) -> torch.Tensor:
    rows = _rows(x, w)
    n, tokens = w.n, rows.shape[0]
    stride = n
    if out is None:
        out_dtype = out_dtype or x.dtype
        if out_dtype not in _OUT_DTYPES:
            raise TypeError(f"unsupported output dtype {out_dtype}")
        out = x.new_empty((tokens, n) if x.dim() == 2 else (*x.shape[:-1], n), dtype=out_dtype)
    else:
        if out.shape != (*x.shape[:-1], n) or out.dtype not in _OUT_DTYPES or out.device != w.device:
            raise ValueError("out must be a fp32, fp16 or bf16 tensor of x's leading shape and n columns on the weight's device")
        if out_dtype is not None and out.dtype != out_dtype:
            raise ValueError("out and out_dtype differ")
        if not out.is_contiguous():
            if out.dim() != 2 or out.stride(1) != 1 or out.stride(0) < n:
                raise ValueError("out must have contiguous rows")
            stride = out.stride(0)
    _lib.call(w.device, fn, *weights, rows.data_ptr(), _X_DTYPES[rows.dtype], max(rows.stride(0), w.k) if tokens > 1 else w.k,
              tokens, *tail[0], out.data_ptr(), _OUT_DTYPES[out.dtype], stride, *tail[1], _lib.current_stream(w.device))
    return out


def linear(x: torch.Tensor, weight: W4Weight, *, out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
           accumulate: bool = False) -> torch.Tensor:
    """x [..., k] (fp16 or bf16) times the transposed 4-bit matrix -> [..., n] in out_dtype (default x's; fp32,
    fp16 or bf16). accumulate adds into a given fp32 `out`."""
    if accumulate and (out is None or out.dtype != torch.float32):
        raise ValueError("accumulate needs an fp32 out")
    return _product(_lib.load().dsv41_w4_linear, (weight._ref,), x, weight, out, out_dtype, ((), (int(accumulate),)))


def gated(x: torch.Tensor, gate: W4Weight, up: W4Weight, limit: float | None = None, *,
          out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """min(silu(x gate^T), limit) * clamp(x up^T, -limit, limit) -> [..., n] in out_dtype (default x's): the
    routed experts' SwiGLU (limit None or 0: no clamp)."""
    if up.device != gate.device:
        raise ValueError("gate and up must live on one device")
    lim = float(limit) if limit is not None and limit > 0 else 0.0
    return _product(_lib.load().dsv41_w4_gated, (gate._ref, up._ref), x, gate, out, out_dtype, ((lim,), ()))


def shared_expert(x: torch.Tensor, gate: W4Weight, up: W4Weight, down: W4Weight, limit: float | None = None, *,
                  out: torch.Tensor) -> torch.Tensor:
    """out [T, H] fp32 (the routed experts' sum, exl3.apply_exl3_fused_moe) += down(gated(x)); the activations
    between the two products have x's type."""
    return linear(gated(x, gate, up, limit), down, out=out, accumulate=True)
