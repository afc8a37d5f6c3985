"""Quantisation of weights: e4m3 with a scale per row, and 4 bits with a scale per group of columns.

Row-wise e4m3 of an LM-head weight is the storage format of the fp8 sampling path.

``weight[v, :] ≈ q[v, :] * scale[v]`` with ``q`` in ``torch.float8_e4m3fn`` and
``scale[v] = max|weight[v, :]| / 448`` (448 is the largest finite e4m3 value).  The sampling
kernels quantise the hidden states the same way, per row, on the way in; this module is what a
user runs once on the weight.

4-bit codes with group scales, ``weight[v, k] ≈ (q[v, k] - zero[v, g]) * scale[v, g]`` with ``g = k // group_size`` and
``q`` in 0..15, are what ``flashsampling_b200.Int4Weight`` holds and ``int4_linear`` multiplies with.

Plain torch: works on CPU and CUDA tensors.
"""

from __future__ import annotations

import torch

E4M3_MAX = 448.0


def round_to_e4m3(y: torch.Tensor) -> torch.Tensor:
    """fp32 values rounded to the nearest e4m3 value, ties to the even mantissa, saturating at +-448 - the
    rounding of the CUDA conversion the kernels use for the hidden states (``torch``'s own cast resolves exact
    ties differently).  Returns fp32 holding exactly representable values."""
    a = y.float().abs()
    _, ex = torch.frexp(a)  # a = m * 2^ex, m in [0.5, 1)
    e = (ex - 1).clamp_min(-6)  # exponent of the value; below 2^-6 the format is denormal with a fixed step
    step = torch.ldexp(torch.ones_like(a), e - 3)  # three mantissa bits
    q = (torch.round(a / step) * step).clamp_max(E4M3_MAX)  # torch.round: half to even
    return torch.copysign(q, y.float())


def quantize_rows_e4m3(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q [R, C] float8_e4m3fn, scale [R] fp32)`` of a 2-D floating-point tensor, processed in
    blocks of rows so that a 1e9-element weight needs no fp32 copy of itself."""
    if x.ndim != 2:
        raise ValueError("expected a [rows, columns] tensor")
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scale = torch.empty(x.shape[0], dtype=torch.float32, device=x.device)
    step = 8192
    for r0 in range(0, x.shape[0], step):
        blk = x[r0:r0 + step].float()
        amax = blk.abs().amax(dim=1).clamp_min(1e-12)
        # one correctly rounded fp32 division, then one fp32 multiply: the operations of the CUDA quantiser
        # (tensor / tensor on purpose: `scalar / tensor` is evaluated as reciprocal-times-scalar)
        inv = torch.full_like(amax, E4M3_MAX) / amax
        q[r0:r0 + step] = round_to_e4m3(blk * inv[:, None]).to(torch.float8_e4m3fn)  # exact: no second rounding
        scale[r0:r0 + step] = amax / torch.full_like(amax, E4M3_MAX)
    return q, scale


def dequantize_rows(q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """fp32 values that the quantised rows stand for."""
    return q.float() * scale[:, None].float()


def int4_group_ok(group_size: int, cols: int) -> bool:
    """Groups of 32 or 64 columns or of a multiple of 128 (up to the whole row), that divide the columns."""
    return group_size > 0 and (group_size in (32, 64) or group_size % 128 == 0) and cols % group_size == 0


def quantize_groups_int4(
    w: torch.Tensor, group_size: int = 128, symmetric: bool = True, scale_dtype: torch.dtype | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """``(q [R, C] uint8 in 0..15, scales [R, C / group_size], zeros [R, C / group_size] uint8 or None)`` of a 2-D
    floating-point tensor, rounded to the nearest code.

    Symmetric: the zero point is 8 everywhere (``zeros`` is ``None``) and the group's largest magnitude becomes +-7.
    Otherwise the group's range, widened to hold 0, is spread over the 16 codes.  ``scale_dtype`` is bf16 or fp16
    (default: the weight's own type if it is one of them, else bf16); codes are chosen for the rounded scale.  A weight that is not
    finite, or whose scales ``scale_dtype`` cannot hold, is refused (which waits for the GPU, once)."""
    if w.ndim != 2 or not w.is_floating_point():
        raise ValueError("expected a floating-point [rows, columns] tensor")
    if not int4_group_ok(group_size, w.shape[1]):
        raise ValueError(f"group_size must be 32, 64 or a multiple of 128 and divide the number of columns ({w.shape[1]})")
    if scale_dtype is None:
        scale_dtype = w.dtype if w.dtype in (torch.bfloat16, torch.float16) else torch.bfloat16
    if scale_dtype not in (torch.bfloat16, torch.float16):
        raise TypeError("scale_dtype must be bfloat16 or float16")
    rows, cols = w.shape
    groups = cols // group_size
    q = torch.empty((rows, cols), dtype=torch.uint8, device=w.device)
    scales = torch.empty((rows, groups), dtype=scale_dtype, device=w.device)
    zeros = None if symmetric else torch.empty((rows, groups), dtype=torch.uint8, device=w.device)
    finite = torch.ones((), dtype=torch.bool, device=w.device)
    step = 8192
    for r0 in range(0, rows, step):
        blk = w[r0:r0 + step].float().view(-1, groups, group_size)
        if symmetric:
            s = blk.abs().amax(-1) / 7
        else:
            lo, hi = blk.amin(-1).clamp_max(0), blk.amax(-1).clamp_min(0)
            s = (hi - lo) / 15
        s = s.to(scale_dtype)
        finite &= s.isfinite().all()
        s = torch.where(s > 0, s, torch.ones_like(s))  # an all-zero group, or one whose scale rounds to zero
        z = torch.full_like(s, 8.0) if symmetric else torch.round(-lo / s.float()).clamp(0, 15).to(s.dtype)
        code = torch.round(blk / s.float()[..., None]) + z.float()[..., None]
        q[r0:r0 + step] = code.clamp(0, 15).to(torch.uint8).view(-1, cols)
        scales[r0:r0 + step] = s
        if zeros is not None:
            zeros[r0:r0 + step] = z.to(torch.uint8)
    if not bool(finite):
        raise ValueError(f"the weight holds values that are not finite, or too large for a scale in {scale_dtype}")
    return q, scales, zeros
