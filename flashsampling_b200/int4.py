"""Products with 4-bit weights and group scales: ``int4_linear(x, Int4Weight)``.

For the few rows of a decode step a linear layer, above all the LM head, costs what streaming its weight costs; four
bits per element are a quarter of the bf16 stream.  The result is that of the dequantised weight, accumulated in fp32;
``fused_mm_sample`` samples from bf16 and e4m3 heads, ``int4_linear`` gives the logits of a 4-bit one, for instance to
``beam_search_step``.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _lib
from .core import _refuse_gradients, _status_word
from .quant import int4_group_ok, quantize_groups_int4

__all__ = ["Int4Weight", "int4_linear"]

_DTYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16, torch.float32: _lib.F32}
_ws_bytes: dict[tuple, int] = {}


class Int4Weight:
    """A ``[rows, cols]`` weight in 4 bits, laid out for ``int4_linear``.

    ``qweight`` uint8 ``[tiles, chunks, 512]``: a tile is 16 rows, a chunk 64 columns, both rounded up; the bytes of a
    (tile, chunk) are indexed ``[g 8][t 4][j 4][b1 2][b0 2]``, and a byte holds rows ``16 tile + g`` (low nibble) and
    ``16 tile + 8 + g`` (high nibble) of column ``64 chunk + 16 j + 8 b0 + 2 t + b1``.  ``scales`` (bf16 or fp16) and
    ``zeros`` (uint8, or ``None``: 8 everywhere) are ``[tiles, groups, 8, 2]``, row ``g`` and row ``8 + g`` next to
    each other.  A weight is ``(q - zero) * scale``.  What rows and columns beyond the weight hold does not matter.
    The tensors' contents may change, the tensors themselves may not: a call refuses a weight whose tensors have moved.

    ``Int4Weight.from_rows`` lays out plain codes, ``Int4Weight.quantize`` rounds a floating-point weight.
    """

    __slots__ = ("qweight", "scales", "zeros", "rows", "cols", "group_size", "_args")

    def __init__(self, qweight: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None, rows: int, cols: int):
        if rows < 1 or cols < 1:
            raise ValueError("an Int4Weight needs at least one row and one column")
        if rows > (1 << 31) - 16 or cols > 1 << 30:
            raise ValueError("an Int4Weight has at most 2^31 - 16 rows and 2^30 columns")
        tiles, chunks = -(-rows // 16), -(-cols // 64)
        if qweight.dtype != torch.uint8 or qweight.shape != (tiles, chunks, 512):
            raise ValueError(f"qweight must be uint8 [{tiles}, {chunks}, 512] for a [{rows}, {cols}] weight")
        if scales.ndim != 4 or scales.shape[1] < 1 or cols % scales.shape[1] or not int4_group_ok(cols // scales.shape[1], cols):
            raise ValueError(f"scales must be [{tiles}, groups, 8, 2] with groups of 32, 64 or a multiple of 128 columns")
        if scales.shape != (tiles, scales.shape[1], 8, 2):
            raise ValueError(f"scales must be [{tiles}, {scales.shape[1]}, 8, 2]")
        if scales.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError("scales must be bfloat16 or float16")
        if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape):
            raise ValueError("zeros must be uint8 of the scales' shape")
        for name, t in (("qweight", qweight), ("scales", scales), ("zeros", zeros)):
            if t is not None and (not t.is_contiguous() or t.data_ptr() % 16 or t.device != qweight.device):
                raise ValueError(f"{name} must be contiguous, start on a 16-byte boundary and lie on qweight's device")
        rows, cols, group = int(rows), int(cols), cols // scales.shape[1]
        # what every call passes on: the tensors are kept and no attribute changes, so their addresses stay
        args = (
            qweight.data_ptr(), scales.data_ptr(), _DTYPES[scales.dtype], zeros.data_ptr() if zeros is not None else None,
            rows, cols, group,
        )
        for name, value in zip(self.__slots__, (qweight, scales, zeros, rows, cols, group, args)):
            object.__setattr__(self, name, value)
        if qweight.is_cuda:
            _status_word(qweight.device)  # here, for the first product may be inside a capture

    def __setattr__(self, name, value):
        raise AttributeError("an Int4Weight keeps its tensors: make a new one")

    def __reduce__(self):
        return (Int4Weight, (self.qweight, self.scales, self.zeros, self.rows, self.cols))

    def _call_args(self) -> tuple:
        """What a call passes on, if the tensors still lie where they did (``t.data = ...`` and ``t.resize_`` move them)."""
        args = self._args
        if (self.qweight.data_ptr() != args[0] or self.scales.data_ptr() != args[1]
                or (self.zeros is not None and self.zeros.data_ptr() != args[3])):
            raise RuntimeError("a tensor of this Int4Weight has got other memory since: make a new Int4Weight")
        return args

    @property
    def shape(self) -> tuple[int, int]:
        return (self.rows, self.cols)

    @property
    def device(self) -> torch.device:
        return self.qweight.device

    def __repr__(self) -> str:
        kind = "zero points" if self.zeros is not None else "symmetric"
        return f"Int4Weight([{self.rows}, {self.cols}], group_size={self.group_size}, {kind}, {self.device})"

    @classmethod
    def from_rows(cls, q: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None) -> "Int4Weight":
        """From codes ``q`` uint8 ``[rows, cols]`` in 0..15 and ``scales`` / ``zeros`` ``[rows, groups]``."""
        if q.ndim != 2 or q.dtype != torch.uint8:
            raise ValueError("q must be uint8 [rows, cols] with one code per element")
        if scales.ndim != 2 or scales.shape[0] != q.shape[0]:
            raise ValueError(f"scales must be [{q.shape[0]}, groups]")
        if zeros is not None and zeros.shape != scales.shape:
            raise ValueError("zeros must have the scales' shape")
        rows, cols = q.shape
        tiles, chunks = -(-rows // 16), -(-cols // 64)
        q = torch.nn.functional.pad(q & 15, (0, chunks * 64 - cols, 0, tiles * 16 - rows))
        v = q.view(tiles, 2, 8, chunks, 4, 2, 4, 2)  # tile h g chunk j b0 t b1
        v = v.permute(0, 3, 2, 6, 4, 7, 5, 1)  # tile chunk g t j b1 b0 h
        packed = (v[..., 0] | (v[..., 1] << 4)).reshape(tiles, chunks, 512)

        def by_tile(t: torch.Tensor) -> torch.Tensor:  # [rows, groups] -> [tiles, groups, 8, 2]
            t = torch.nn.functional.pad(t, (0, 0, 0, tiles * 16 - rows))
            return t.view(tiles, 2, 8, -1).permute(0, 3, 2, 1).contiguous()

        return cls(packed.contiguous(), by_tile(scales), None if zeros is None else by_tile(zeros), rows, cols)

    @classmethod
    def quantize(cls, w: torch.Tensor, group_size: int = 128, symmetric: bool = True,
                 scale_dtype: torch.dtype | None = None) -> "Int4Weight":
        """The nearest codes of a floating-point ``[rows, cols]`` weight (``quant.quantize_groups_int4``)."""
        return cls.from_rows(*quantize_groups_int4(w, group_size, symmetric, scale_dtype))

    def to(self, device) -> "Int4Weight":
        return Int4Weight(self.qweight.to(device), self.scales.to(device),
                          None if self.zeros is None else self.zeros.to(device), self.rows, self.cols)

    def codes(self) -> torch.Tensor:
        """The codes as plain uint8 ``[rows, cols]``."""
        tiles, chunks, _ = self.qweight.shape
        v = self.qweight.view(tiles, chunks, 8, 4, 4, 2, 2)  # tile chunk g t j b1 b0
        v = torch.stack((v & 15, v >> 4), dim=-1)  # ... h
        v = v.permute(0, 7, 2, 1, 4, 6, 3, 5)  # tile h g chunk j b0 t b1
        return v.reshape(tiles * 16, chunks * 64)[:self.rows, :self.cols].contiguous()

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values that the weight stands for, ``[rows, cols]``."""
        def by_row(t):
            return t.permute(0, 3, 2, 1).reshape(-1, t.shape[1])[:self.rows]

        q = self.codes().to(dtype).view(self.rows, -1, self.group_size)
        z = 8 if self.zeros is None else by_row(self.zeros).to(dtype)[..., None]
        return ((q - z) * by_row(self.scales).to(dtype)[..., None]).view(self.rows, self.cols)


def int4_linear(x: torch.Tensor, weight: Int4Weight, *, out_dtype: torch.dtype | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ weight.T`` for bf16 or fp16 ``x [..., cols]``: ``[..., rows]`` in ``out_dtype`` (bf16, fp16 or fp32; default
    the type of ``x``), or into ``out``, which must not share memory with ``x``.

    Made for the few rows of a decode step.  In times of the weight's stream (at the rate of a plain copy) a large weight costs 1.1 for
    one row and 1.2 for eight, with zero points and groups of 64 1.8 for five; 16 rows cost 1.7, 32 rows 2 (with groups
    of 64 both above 3), 64 rows 3.4 to 5, and more than 64 (32 for groups of 32 columns) read the weight again for every 64.

    Rows of ``x`` may be strided.  They are multiplied as fp16 after an exact power of two per row: bf16 values below 2^-28 of
    their row's largest are rounded to 2^-39 of it, in batches of more than eight rows values below 2^-24 (fp16: 2^-21) to 2^-32
    of it.  Sums are fp32 and their order is fixed: a row of ``x`` gives the same bits in every batch of up to eight rows, and in every
    larger one.  No gradients: the weight is for serving."""
    if not isinstance(weight, Int4Weight):
        raise TypeError("weight must be an Int4Weight")
    if not (x.is_cuda and weight.qweight.is_cuda):
        raise RuntimeError("int4_linear requires CUDA tensors (there is no CPU path)")
    if x.dtype is not torch.bfloat16 and x.dtype is not torch.float16:
        raise TypeError("x must be bfloat16 or float16")
    if x.ndim < 1 or x.shape[-1] != weight.cols:
        raise ValueError(f"x must be [..., {weight.cols}], got {list(x.shape)}")
    dev = weight.qweight.device
    if x.device != dev:
        raise ValueError(f"x is on {x.device}, the weight on {dev}")
    if x.requires_grad or forward_ad._current_level >= 0:
        _refuse_gradients("int4_linear", x)
    x2 = x if x.ndim == 2 else x.reshape(-1, weight.cols)
    if x2.stride(1) != 1 or x2.stride(0) < weight.cols:
        x2 = x2.contiguous()
    b = x2.shape[0]
    if b >= 1 << 31:
        raise ValueError("int4_linear takes fewer than 2^31 rows of x")
    shape = x.shape[:-1] + (weight.rows,)
    given = out is not None
    if not given:
        out_dtype = out_dtype or x.dtype
        if out_dtype not in _DTYPES:
            raise TypeError("out_dtype must be bfloat16, float16 or float32")
        out = torch.empty(shape, dtype=out_dtype, device=dev)
        out_stride = weight.rows
    else:
        if out.shape != shape or out.device != dev or out.dtype not in _DTYPES or (out_dtype or out.dtype) != out.dtype:
            raise ValueError(f"out must be {list(shape)} in bfloat16, float16 or float32 on {dev}")
        if out.ndim == 2 and out.stride(1) == 1 and (out.stride(0) >= weight.rows or b <= 1):
            out_stride = max(out.stride(0), weight.rows)
        elif out.is_contiguous():
            out_stride = weight.rows
        else:
            raise ValueError("out must have consecutive rows of consecutive elements")
        if out.requires_grad:
            raise RuntimeError("out must not require gradients")
        if forward_ad._current_level >= 0:
            _refuse_gradients("int4_linear", out)
    if b == 0:
        return out
    stride = x2.stride(0) if b > 1 else max(x2.stride(0), weight.cols)
    if given and _rows_meet(x2, stride, out, out_stride, b, weight):
        raise ValueError("out must not share memory with x: rows of x are still read while others are written")
    index = dev.index
    if torch._C._cuda_getDevice() == index:
        rc = _launch(x2, stride, weight, b, out, out_stride, index)
    else:
        with torch.cuda.device(dev):
            rc = _launch(x2, stride, weight, b, out, out_stride, index)
    if rc:
        raise _lib.FmmsError(rc, "fmms_int4_linear")
    if given:
        increment_version(out)
    return out


def _rows_meet(x, stride, out, out_stride, b, weight) -> bool:
    """Whether the rows that are read and those that are written have bytes in common (side by side in one buffer: no)."""
    ex, eo = x.element_size(), out.element_size()
    pitch, pitch_out, width, width_out = stride * ex, out_stride * eo, weight.cols * ex, weight.rows * eo
    apart = out.data_ptr() - x.data_ptr()
    if apart >= (b - 1) * pitch + width or -apart >= (b - 1) * pitch_out + width_out:
        return False
    if b == 1 or pitch != pitch_out:
        return True
    apart %= pitch
    return apart < width or apart + width_out > pitch


def _launch(x, stride, weight, b, out, out_stride, index):
    qw, scales, scale_dtype, zeros, rows, cols, group = weight._call_args()
    key = (rows, cols, group, b)
    nbytes = _ws_bytes.get(key)
    if nbytes is None:
        nbytes = _ws_bytes[key] = _lib.query_int4_workspace(*key)
    # from torch's allocator on every call: calls on several streams, or in several captured graphs, share nothing
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
    status = None
    if b > 8:  # up to eight rows there are no waits between warps
        status = _status_word(x.device)
        if status is None:
            raise RuntimeError("int4_linear has no status word yet, and cannot make one in a capture: make an Int4Weight on the device before it")
    return _lib.load().fmms_int4_linear(
        x.data_ptr(), _DTYPES[x.dtype], stride, qw, scales, scale_dtype, zeros, rows, cols, group, b,
        out.data_ptr(), _DTYPES[out.dtype], out_stride, ws.data_ptr() if nbytes else None, nbytes,
        status.data_ptr() if status is not None else None,
        torch._C._cuda_getCurrentRawStream(index))
