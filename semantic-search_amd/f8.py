"""8-bit rows: quantisation, the norm that ends in them, and their product (libssmi.so, csrc/f8_*.hip).

A row is e4m3 codes with one power-of-two scale for every 128 of them, kept as its biased exponent:
value = code * 2**(scale - 127).  `IndexFlatIP(d, storage="f8")` keeps such rows: `add` and `search` quantise what they are given,
or take an `F8Rows` as it is - for instance what `rms_norm_f8(..., unit=True)` makes of a model's last hidden states, which is
what the reference's embedder does in fp32 before it hands rows to FAISS (core/qwen3_vl_embedding.py:447-448).

All calls work on tensors of a ROCm device, enqueue on its current torch stream, wait for nothing and may be captured into a
graph; none of them records a gradient.  What they write into counts as changed in place (a backward pass that saved it raises), must not
require a gradient outside of torch.no_grad(), and may overlap an input only where that is said.  Argument errors raise ValueError or
TypeError, errors of the engine RuntimeError.
"""
from typing import Optional

import torch

from . import _lib

BLOCK = 128
_SRC = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def _blocks(d: int) -> int:
    return (d + BLOCK - 1) // BLOCK


# handle of the current torch stream of device i (the Stream object around it costs more than a launch)
_stream = torch._C._cuda_getCurrentRawStream


# autograd's notice that a tensor has been written through its pointer
_changed = torch.autograd.graph.increment_version


def _writable(t: torch.Tensor, what: str) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} is written without a gradient but requires one: detach it, or call under torch.no_grad()")


def _rows_arg(x, what: str) -> torch.Tensor:
    """A 2-D device tensor of a known type whose rows are contiguous (other layouts are copied)."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what}: expected a torch tensor, got {type(x).__name__}")
    if not x.is_cuda:
        raise ValueError(f"{what}: the tensor must live on a ROCm device")
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"{what}: expected a 2-D tensor with at least one column, got shape {tuple(x.shape)}")
    if x.dtype not in _SRC:
        raise TypeError(f"{what}: expected float32, float16 or bfloat16, got {x.dtype}")
    return x if x.stride(1) == 1 and (x.shape[0] <= 1 or x.stride(0) >= x.shape[1]) else x.contiguous()


def _stride(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _layout_error(codes, scales, d: int) -> Optional[str]:
    """What keeps the kernels from reading the tensors as rows of d elements, or None."""
    for t, name, dtype in ((codes, "codes", torch.float8_e4m3fn), (scales, "scales", torch.uint8)):
        if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.dim() != 2:
            return f"{name} must be a 2-D tensor of {dtype}"
    ld, ls = _blocks(d) * BLOCK, (_blocks(d) + 3) // 4 * 4
    if d < 1 or codes.shape[1] != ld or scales.shape[1] < ls or codes.shape[0] != scales.shape[0] or codes.device != scales.device:
        return f"{d} elements need {ld} codes and {ls} scales a row, as many rows of both on one device, got {tuple(codes.shape)} and {tuple(scales.shape)}"
    for t, name, width, unit in ((codes, "codes", ld, 16), (scales, "scales", ls, 4)):
        if t.stride(1) != 1 or t.data_ptr() % unit or (t.shape[0] > 1 and (t.stride(0) % unit or t.stride(0) < width)):
            return f"rows of {name} must be contiguous, {unit}-byte aligned and a multiple of {unit} bytes apart"
    return None


class F8Rows:
    """n rows of d elements in 8 bits: `codes` (n, whole blocks of 128) float8_e4m3fn, `scales` (n, >= blocks) uint8."""

    __slots__ = ("n", "d", "device_index", "_args", "_buffer", "_codes", "_scales")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, d: int):
        """The tensors as they are, in the layout that the kernels read: rows of whole blocks of codes, zero behind d, and of scales in words of
        four; `from_parts` takes others."""
        d = int(d)
        what = _layout_error(codes, scales, d)
        if what:
            raise ValueError(f"F8Rows: {what}")
        self._set(codes, scales, d)

    def _set(self, codes: torch.Tensor, scales: torch.Tensor, d: int) -> None:
        self.n, self.d, self._codes, self._scales, self._buffer = codes.shape[0], d, codes, scales, None
        self.device_index = codes.get_device()
        # codes, their stride, scales, their stride: as the C entry points take them
        self._args = (codes.data_ptr(), codes.stride(0) if self.n > 1 else codes.shape[1],
                      scales.data_ptr(), scales.stride(0) if self.n > 1 else (scales.shape[1] + 3) // 4 * 4)

    @classmethod
    def empty(cls, n: int, d: int, device) -> "F8Rows":
        """Rows to be written by quantize_f8 / rms_norm_f8 (`out=`): one allocation, the codes and behind them the scales."""
        blocks = _blocks(d)
        ld, ls = blocks * BLOCK, (blocks + 3) // 4 * 4
        self = cls.__new__(cls)
        self.n, self.d, self._codes, self._scales = n, d, None, None
        self._buffer = buf = torch.empty(n * (ld + ls), dtype=torch.uint8, device=device)
        self.device_index = buf.get_device()
        p = buf.data_ptr()
        self._args = (p, ld, p + n * ld, ls)
        return self

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            ld = _blocks(self.d) * BLOCK
            self._codes = self._buffer[:self.n * ld].view(self.n, ld).view(torch.float8_e4m3fn)
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            blocks = _blocks(self.d)
            self._scales = self._buffer[self.n * blocks * BLOCK:].view(self.n, (blocks + 3) // 4 * 4)
        return self._scales

    @classmethod
    def from_parts(cls, codes: torch.Tensor, scales: torch.Tensor, d: Optional[int] = None) -> "F8Rows":
        """Rows from codes (n, d or whole blocks; float8_e4m3fn or uint8) and scale exponents (n, blocks; uint8).  The tensors are used as they are
        where their layout allows and are never written; whole blocks whose codes behind d are not all zero are copied (to look waits for them)."""
        if codes.dim() != 2 or scales.dim() != 2 or codes.shape[0] != scales.shape[0]:
            raise ValueError(f"F8Rows: expected 2-D codes and scales of as many rows, got {tuple(codes.shape)} and {tuple(scales.shape)}")
        if not codes.is_cuda or codes.device != scales.device:
            raise ValueError("F8Rows: codes and scales must live on the same ROCm device")
        if codes.dtype not in (torch.float8_e4m3fn, torch.uint8) or scales.dtype != torch.uint8:
            raise TypeError(f"F8Rows: expected float8_e4m3fn or uint8 codes and uint8 scales, got {codes.dtype} and {scales.dtype}")
        d = int(codes.shape[1] if d is None else d)
        blocks = _blocks(d)
        if d < 1 or codes.shape[1] not in (d, blocks * BLOCK) or scales.shape[1] < blocks:
            raise ValueError(f"F8Rows: {d} elements need {d} or {blocks * BLOCK} codes and {blocks} scales a row, got {codes.shape[1]} and {scales.shape[1]}")
        raw, whole = codes.view(torch.uint8), blocks * BLOCK
        copy = raw.shape[1] != whole or raw.stride(1) != 1 or raw.stride(0) % 16 or raw.data_ptr() % 16 or raw.stride(0) < whole
        if not copy and d < whole:   # (a stream that is captured cannot be waited for)
            copy = torch.cuda.is_current_stream_capturing() or bool((raw[:, d:] & 0x7F).any())
        if copy:
            fresh = torch.zeros((raw.shape[0], whole), dtype=torch.uint8, device=raw.device)
            fresh[:, :d] = raw[:, :d]
            raw = fresh
        if scales.stride(1) != 1 or scales.stride(0) % 4 or scales.data_ptr() % 4 or min(scales.shape[1], scales.stride(0)) < (blocks + 3) // 4 * 4:
            fresh = torch.zeros((scales.shape[0], (blocks + 3) // 4 * 4), dtype=torch.uint8, device=scales.device)
            fresh[:, :blocks] = scales[:, :blocks]
            scales = fresh
        return cls(raw.view(torch.float8_e4m3fn), scales, d)

    @property
    def device(self) -> torch.device:
        return torch.device("cuda", self.device_index)

    def __len__(self) -> int:
        return self.n

    def __getitem__(self, rows: slice) -> "F8Rows":
        """A contiguous range of the rows (a view)."""
        if not isinstance(rows, slice) or rows.step not in (None, 1):
            raise TypeError("F8Rows: only plain slices of rows")
        part = F8Rows.__new__(F8Rows)
        part._set(self.codes[rows], self.scales[rows], self.d)   # (the layout is its whole's)
        return part

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values the rows stand for, (n, d); exact in float32 and bfloat16 (four significant bits times a power of two)."""
        if dtype not in _SRC:
            raise TypeError(f"dequantize: expected float32, float16 or bfloat16, got {dtype}")
        i = self.device_index
        out = torch.empty((self.n, self.d), dtype=dtype, device=i)
        _lib.check(_lib.load().ssmi_f8_dequantize(i, self.n, self.d, *self._args, out.data_ptr(), _SRC[dtype], self.d, _stream(i)))
        return out


def _rows_changed(out: F8Rows) -> None:
    _changed(out._buffer if out._buffer is not None else (out._codes, out._scales))


def _out_rows(out: Optional[F8Rows], n: int, d: int, device_index: int, what: str) -> F8Rows:
    if out is None:
        return F8Rows.empty(n, d, device_index)
    if not isinstance(out, F8Rows) or out.n != n or out.d != d or out.device_index != device_index:
        raise ValueError(f"{what}: out must be F8Rows of {n} rows of {d} elements on cuda:{device_index}")
    return out


def quantize_f8(x: torch.Tensor, out: Optional[F8Rows] = None) -> F8Rows:
    """8-bit rows of x (n, d): per 128 elements the smallest power of two s with max|x| <= 448 s, codes x / s to nearest even."""
    x = _rows_arg(x, "quantize_f8")
    n, d = x.shape
    i = x.get_device()
    rows = _out_rows(out, n, d, i, "quantize_f8")
    _lib.check(_lib.load().ssmi_f8_quantize(i, n, d, x.data_ptr(), _SRC[x.dtype], _stride(x), *rows._args, _stream(i)))
    if out is not None:
        _rows_changed(rows)
    return rows


def rms_norm_f8(x: torch.Tensor, weight: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                residual_out: Optional[torch.Tensor] = None, eps: float = 1e-6, unit: bool = False, out: Optional[F8Rows] = None) -> F8Rows:
    """8-bit rows of the root-mean-square norm of h = x + residual: h / sqrt(mean(h^2) + eps) * weight, in 64 bits.

    The sum is rounded to x's type and stored in `residual_out` (default: back into `residual`; it may be `x` or `residual`, and else shares no
    memory with them).  unit=True: rows of unit length,
    ready for an inner-product index."""
    x = _rows_arg(x, "rms_norm_f8")
    n, d = x.shape
    i = x.get_device()
    w = r = ro = None
    if weight is not None:
        if not isinstance(weight, torch.Tensor) or weight.shape != (d,) or weight.device != x.device:
            raise ValueError(f"rms_norm_f8: weight must be a tensor of {d} elements on {x.device}")
        if weight.dtype not in _SRC:
            raise TypeError(f"rms_norm_f8: weight must be float32, float16 or bfloat16, got {weight.dtype}")
        w = weight.contiguous()
    if residual is not None:
        r = residual
        ro = residual if residual_out is None else residual_out
        for t, name in ((r, "residual"), (ro, "residual_out")):
            if not isinstance(t, torch.Tensor) or t.shape != x.shape or t.dtype != x.dtype or t.device != x.device:
                raise ValueError(f"rms_norm_f8: {name} must be like x: shape {tuple(x.shape)}, {x.dtype}, {x.device}")
        if d > 1 and ro.stride(1) != 1 or n > 1 and ro.stride(0) < d:
            raise ValueError("rms_norm_f8: residual_out must have contiguous rows")
        _writable(ro, "rms_norm_f8: residual" if residual_out is None else "rms_norm_f8: residual_out")
        if d > 1 and r.stride(1) != 1 or n > 1 and r.stride(0) < d:
            r = r.contiguous()
    elif residual_out is not None:
        raise ValueError("rms_norm_f8: residual_out without a residual")
    rows = _out_rows(out, n, d, i, "rms_norm_f8")
    _lib.check(_lib.load().ssmi_f8_rms_norm(
        i, n, d, x.data_ptr(), _SRC[x.dtype], _stride(x), r.data_ptr() if r is not None else None, _stride(r) if r is not None else 0,
        ro.data_ptr() if ro is not None else None, _stride(ro) if ro is not None else 0, w.data_ptr() if w is not None else None,
        _SRC[w.dtype] if w is not None else 0, float(eps), 1 if unit else 0, *rows._args, _stream(i)))
    if ro is not None:
        _changed(ro)
    if out is not None:
        _rows_changed(rows)
    return rows


def matmul_f8(a: F8Rows, b: F8Rows, out_dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """(a.n, b.n): inner products of the rows of a (activations) with the rows of b (weights, or a table of embeddings), exact products
    summed in float32 and rounded once to the output's type."""
    if not isinstance(a, F8Rows) or not isinstance(b, F8Rows):
        raise TypeError("matmul_f8: expected two F8Rows")
    if a.d != b.d:
        raise ValueError(f"matmul_f8: rows of {a.d} and {b.d} elements")
    i = a.device_index
    if i != b.device_index:
        raise ValueError(f"matmul_f8: operands on {a.device} and {b.device}")
    if out is not None:
        if not isinstance(out, torch.Tensor):
            raise TypeError(f"matmul_f8: out must be a tensor, got {type(out).__name__}")
        out_dtype = out.dtype
    if out_dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"matmul_f8: the output is float16 or bfloat16, not {out_dtype}")
    given = out is not None
    if not given:
        out = torch.empty((a.n, b.n), dtype=out_dtype, device=i)
    elif out.shape != (a.n, b.n) or out.get_device() != i or (b.n > 1 and out.stride(1) != 1) or (a.n > 1 and out.stride(0) < b.n):
        raise ValueError(f"matmul_f8: out must be ({a.n}, {b.n}) with contiguous rows on {a.device}")
    else:
        _writable(out, "matmul_f8: out")
    _lib.check(_lib.load().ssmi_f8_matmul(i, a.n, b.n, a.d, *a._args, *b._args, out.data_ptr(), _SRC[out_dtype],
                                          out.stride(0) if a.n > 1 else b.n, _stream(i)))
    if given:
        _changed(out)
    return out
