"""Projections whose weights are held in 4 bits with group scales, on libftk (csrc/ftk_w4.hip).

``W[n, k] = s[n, k // group] * (q[n, k] - z[n, k // group])`` with codes q in 0..15, scales s in BF16 or FP16
and zero points z in 0..15 (8 everywhere where none are given). A checkpoint's codes are laid out once by
``pack_w4`` (``quantize_w4`` makes codes and scales of a BF16 weight first); the ``W4Weight`` it returns stands
where a weight tensor does in the BF16 functions:

    linear_w4(x, weight)                                x W^T
    linear_residual_w4(x, weight, residual)             x W^T + residual
    rms_norm_linear_w4(x, norm_weight, eps, weight)     rms_norm(x) W^T (+ residual)
    gate_up_swiglu_w4(x, weight, norm_weight, eps)      silu(xn Wg^T) * (xn Wu^T), W = cat(Wg, Wu)

BF16 activations, FP32 sums, one rounding of the result to BF16 (SwiGLU included: its gate and up sums stay
FP32, and the norm rounds nothing on the way: x gain meets the weights as two BF16 addends that hold it exactly).
An infinite or NaN activation gives what the products with s (q - z) give. Up to ``linear.MAX_ROWS`` rows run on
the 4-bit kernels; more rows (a prompt) take ``dequantize_w4`` and the native GEMM, as ``linear`` sends them there.
No counterpart in the reference, whose weights are BF16.
"""

import ctypes

import torch
from torch.nn import functional as F

from kernels import _native
from kernels.rmsnorm import rms_norm
from kernels.swiglu import swiglu

#: Weight rows of a tile and columns of a chunk of the packed layout.
TILE, CHUNK = 16, 128
_calls = _native.calls
#: Group sizes the kernels take; longer groups (multiples of 128, or whole rows) repeat their scale per chunk.
GROUPS = (32, 64, 128)
#: Weight elements laid out at a time: bounds the memory ``pack_w4`` needs beside its result.
_SLAB = 1 << 26


class W4Weight:
    """A [rows, columns] weight in the kernels' layout: ``codes`` int32 [tiles, chunks, 64, 4], ``scales`` [tiles,
    chunks, 16, 128 / group], ``zeros`` uint8 of the same shape or None. ``gate_up``: the rows are cat(Wg, Wu) and
    the product ends in SwiGLU. Made by ``pack_w4``; its tensors must not be replaced."""

    def __init__(self, codes, scales, zeros, rows, columns, group, gate_up):
        half = TILE // 2 if gate_up else TILE
        blocks = (-(-(rows // 2 if gate_up else rows) // half), -(-columns // CHUNK))  # tiles, chunks
        if group not in GROUPS or rows < 1 or columns < 1 or (gate_up and rows % 2):
            raise ValueError(f"no packed weight of {rows} x {columns} in groups of {group}")
        if codes.dtype != torch.int32 or codes.shape != (*blocks, 64, 4) or not codes.is_contiguous():
            raise ValueError(f"codes must be contiguous int32 {(*blocks, 64, 4)}, got {codes.dtype} {tuple(codes.shape)}")
        shape = (*blocks, TILE, CHUNK // group)
        for name, t, types in (("scales", scales, (torch.bfloat16, torch.float16)), ("zeros", zeros, (torch.uint8,))):
            if t is not None and (t.dtype not in types or t.shape != shape or not t.is_contiguous() or
                                  t.device != codes.device):
                raise ValueError(f"{name} must be contiguous {shape} beside the codes, got {t.dtype} {tuple(t.shape)}")
        if any(t is not None and t.data_ptr() % 16 for t in (codes, scales, zeros)):
            raise ValueError("packed tensors must be 16-byte aligned")
        self.codes, self.scales, self.zeros = codes, scales, zeros
        self.rows, self.columns, self.group, self.gate_up = rows, columns, group, gate_up
        self.outputs = rows // 2 if gate_up else rows
        self.device = codes.device
        # (The kernels' rows have at least 8 columns; codes past the weight's own meet zeros.)
        self._handle = _native.W4(codes.data_ptr(), scales.data_ptr(), _native.ptr(zeros), rows, max(columns, 8), group,
                                  _native.W4_SCALE_FP16 if scales.dtype == torch.float16 else _native.W4_SCALE_BF16,
                                  _native.W4_GATE_UP if gate_up else _native.W4_ROWS)
        self._ref = ctypes.byref(self._handle)
        #: What the direct calls take: the handle's address for the products this weight is for (else None), its device.
        address = ctypes.addressof(self._handle)
        self._rows, self._gate_up = (None, address) if gate_up else (address, None)
        self._index = codes.get_device()

    def __repr__(self):
        return f"W4Weight({self.rows} x {self.columns}, group {self.group}{', gate_up' if self.gate_up else ''})"


def _tiles(t, gate_up, fill):
    """Rows of ``t`` [N, ...] in tile order [tiles, 16, ...], the missing ones ``fill``."""
    if not gate_up:
        return F.pad(t, (0, 0, 0, -t.shape[0] % TILE), value=fill).unflatten(0, (-1, TILE))
    half = TILE // 2
    gate, up = (F.pad(p, (0, 0, 0, -p.shape[0] % half), value=fill).unflatten(0, (-1, half)) for p in t.chunk(2))
    return torch.cat((gate, up), dim=1)


def pack_w4(codes, scales, zeros=None, group=128, gate_up=False):
    """A ``W4Weight`` of ``codes`` [N, K] uint8 (0..15), ``scales`` [N, ceil(K / group)] (BF16 or FP16) and optional
    ``zeros`` of the scales' shape (uint8, 0..15). ``group`` is 32, 64, a multiple of 128, or at least K. With
    ``gate_up`` N is even and the rows are cat(Wg, Wu). Reads the codes back once to check them."""
    n, k = codes.shape
    if codes.dtype != torch.uint8 or n < 1 or k < 1:
        raise ValueError("codes must be a [N, K] uint8 tensor")
    if group < 1 or not (group in GROUPS or group % CHUNK == 0 or group >= k):
        raise ValueError(f"group {group}: the kernels take 32, 64, multiples of 128 or whole rows")
    if scales.dtype not in (torch.bfloat16, torch.float16) or scales.shape != (n, -(-k // group)):
        raise ValueError(f"scales must be BF16 or FP16 [{n}, {-(-k // group)}], got {scales.dtype} {tuple(scales.shape)}")
    if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape):
        raise ValueError("zeros must be uint8 and have the scales' shape")
    if gate_up and n % 2:
        raise ValueError("gate_up stacks gate and up rows: an even row count")
    if scales.device != codes.device or (zeros is not None and zeros.device != codes.device):
        raise ValueError("codes, scales and zeros must be on one device")
    if int(codes.max()) > 15 or (zeros is not None and int(zeros.max()) > 15):
        raise ValueError("codes and zeros must be 0..15")
    chunks = -(-k // CHUNK)
    unit = group if group in GROUPS else CHUNK  # columns of a stored scale
    subs = CHUNK // unit

    def spread(t, fill):
        # One entry per `unit` columns: a longer group's is repeated, entries past K are `fill`.
        entry = torch.arange(chunks * subs, device=t.device) * unit
        wide = t[:, (entry.clamp(max=k - 1) // group)]
        wide = torch.where(entry < k, wide, torch.full_like(wide, fill))
        return _tiles(wide, gate_up, fill).unflatten(2, (chunks, subs)).transpose(1, 2).contiguous()

    shift = torch.tensor([4 * (e // 2) + 16 * (e % 2) for e in range(8)], device=codes.device, dtype=torch.int32)
    half = TILE // 2 if gate_up else TILE
    tiles = -(-(n // 2 if gate_up else n) // half)
    packed = torch.empty((tiles, chunks, 64, 4), dtype=torch.int32, device=codes.device)
    step = max(1, _SLAB // (chunks * CHUNK * TILE))
    for t in range(0, tiles, step):
        if gate_up:
            rows = torch.cat([codes[o + t * half : o + min(n // 2, (t + step) * half)] for o in (0, n // 2)])
        else:
            rows = codes[t * half : (t + step) * half]
        part = _tiles(F.pad(rows, (0, chunks * CHUNK - k), value=8), gate_up, 8)
        # [tile, row, chunk, step, lane group, element] -> lane (row + 16 group), dword (step)
        part = part.view(-1, TILE, chunks, 4, 4, 8).permute(0, 2, 4, 1, 3, 5)
        packed[t : t + part.shape[0]] = (part.to(torch.int32) << shift).sum(dim=-1, dtype=torch.int32).flatten(2, 3)
    return W4Weight(packed, spread(scales, 0.0), None if zeros is None else spread(zeros, 8), n, k, unit, gate_up)


def quantize_w4(weight, group=128, gate_up=False, scale_dtype=torch.bfloat16):
    """``weight`` [N, K] rounded to 4 bits, round-to-nearest: per group s = amax / 7 (rounded to ``scale_dtype``),
    q = clamp(round(w / s) + 8, 0, 15), no zero points."""
    n, k = weight.shape
    if n < 1 or k < 1 or group < 1:
        raise ValueError(f"a weight of {n} x {k} in groups of {group}")
    groups = -(-k // group)
    wide = F.pad(weight.float(), (0, groups * group - k)).unflatten(1, (groups, group))
    scales = (wide.abs().amax(dim=2) / 7).to(scale_dtype)
    s = scales.float()[:, :, None]
    codes = torch.where(s > 0, wide / s, 0.0).round().add(8).clamp(0, 15).to(torch.uint8)
    return pack_w4(codes.flatten(1)[:, :k], scales, None, group, gate_up)


def dequantize_w4(weight):
    """The weight itself, BF16 [rows, columns]: each s (q - z) rounded once."""
    _native.require_gpu(weight.codes)
    out = torch.empty((weight.rows, weight._handle.K), dtype=torch.bfloat16, device=weight.device)
    _native.call_on(out, "ftk_w4_dequantize_bf16", weight._ref, out.data_ptr())
    return out if weight.columns == weight._handle.K else out[:, : weight.columns].contiguous()


def _rows(x, weight):
    """x as [M, K] rows the kernel can read (unit stride, rows apart or one behind the other)."""
    if x.dtype != torch.bfloat16:
        raise ValueError(f"x must be BF16, got {x.dtype}")
    if x.shape[-1] != weight.columns:
        raise ValueError(f"x has {x.shape[-1]} columns, the weight {weight.columns}")
    if x.device != weight.device:
        raise ValueError(f"x is on {x.device}, the weight on {weight.device}")
    if not x.is_cuda:
        _native.require_gpu(x)
    flat = x if x.dim() == 2 else x.reshape(-1, weight.columns)
    stride = flat.stride()
    if stride[1] != 1 or (stride[0] < weight.columns and flat.shape[0] > 1):
        flat = flat.contiguous()
    return flat


def _like(name, t, shape, device):
    if t.dtype != torch.bfloat16 or t.shape != shape or t.device != device:
        raise ValueError(f"{name} must be BF16 {tuple(shape)} on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _project(x, weight, norm_weight, eps, residual):
    """The general call: refusals, copies, rows beyond the kernels', another device than the current one."""
    if x.is_cuda and x.get_device() != torch.cuda.current_device():
        with torch.cuda.device(x.device):
            return _project(x, weight, norm_weight, eps, residual)
    flat = _rows(x, weight)
    rows = flat.shape[0]
    shape = (*x.shape[:-1], weight.outputs)
    if residual is not None:
        _like("residual", residual, shape, x.device)
        residual = residual.reshape(rows, weight.outputs).contiguous()
    if norm_weight is not None:
        _like("norm_weight", norm_weight, (weight.columns,), x.device)
        norm_weight = norm_weight.contiguous()
    if rows > _native.MAX_ROWS:
        y = F.linear(flat if norm_weight is None else rms_norm(flat, norm_weight, eps), dequantize_w4(weight))
        y = swiglu(y) if weight.gate_up else y if residual is None else y + residual
        return y.view(shape)
    out = torch.empty((rows, weight.outputs), dtype=torch.bfloat16, device=x.device)
    if rows:
        if norm_weight is not None and weight.columns < 8:
            flat, norm_weight = rms_norm(flat, norm_weight, eps), None
        if weight.columns < 8:
            flat = F.pad(flat, (0, 8 - weight.columns))
        _native.call_on(out, "ftk_w4_project_bf16", flat.data_ptr(), flat.stride(0), _native.ptr(norm_weight),
                        float(eps), weight._ref, _native.ptr(residual), out.data_ptr(), rows)
    return out if x.dim() == 2 else out.view(shape)


def _plain_rows(weight):
    if weight.gate_up:
        raise ValueError("a gate_up weight is for gate_up_swiglu_w4")


def linear_w4(x, weight):
    """x [..., K] @ W.T, BF16 [..., N]."""
    out = _calls.w4(x, weight._rows, weight._index, weight.outputs, None, 0.0, None)
    if out is None:
        _plain_rows(weight)
        out = _project(x, weight, None, 0.0, None)
    return out


def linear_residual_w4(x, weight, residual):
    """x @ W.T + residual: the add in FP32, before the one rounding."""
    out = _calls.w4(x, weight._rows, weight._index, weight.outputs, None, 0.0, residual)
    if out is None:
        _plain_rows(weight)
        out = _project(x, weight, None, 0.0, residual)
    return out


def rms_norm_linear_w4(x, norm_weight, eps, weight, residual=None):
    """rms_norm(x, norm_weight, eps) @ W.T (+ residual), the norm without intermediate roundings."""
    out = _calls.w4(x, weight._rows, weight._index, weight.outputs, norm_weight, eps, residual)
    if out is None:
        _plain_rows(weight)
        out = _project(x, weight, norm_weight, eps, residual)
    return out


def gate_up_swiglu_w4(x, weight, norm_weight=None, eps=1e-6):
    """silu(xn @ Wg.T) * (xn @ Wu.T), xn = x or rms_norm(x), for a weight packed with ``gate_up``; BF16 [..., I]."""
    out = _calls.w4(x, weight._gate_up, weight._index, weight.outputs, norm_weight, eps, None)
    if out is None:
        if not weight.gate_up:
            raise ValueError("the weight must be packed with gate_up=True")
        out = _project(x, weight, norm_weight, eps, None)
    return out
