"""Microscaled 4-bit operands of the expert FFN: quantisation, grouped products, and the FFN itself for serving and
for training (``csrc/device/mx_quant.cu``, ``mx_gemm.cuh``).

An operand is quantised along the reduction in blocks of 32: with ``a = max |x|`` of a block and
``e = floor(log2 a) - 2`` (within [-127, 127]) every element becomes ``x / 2^e`` rounded to the nearest of
0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code, larger ones to 6) times ``2^e``.  A block with a NaN or an infinity
is all NaN.  17 bytes stand for 64 of bf16 (20 in one matrix, whose scales lie there four times), and the tensor cores
multiply such operands as they are.

========================  ==============================  =======================================
op                        math                            operands
========================  ==============================  =======================================
``quantize``              x -> ``MxTensor``               bf16, fp16, fp32; any sizes
``pack_gate_up``          Wg, Wu -> one ``MxTensor``      [G, H, H'] each, blocks along H
``matmul``                y = a W[g]^T                    a [rows,K] . W [G,N,K]
``gateup_swiglu``         act = silu(x Wg)*(x Wu)*w       x [rows,H] . packed Wg, Wu
``gateup_swiglu_bwd``     d gate, d up, d w               fp32 d act [rows,H'] and the forward's
``expert_ffn``            y = act Wd^T, with gradients    bf16 x [rows,H], Wg/Wu/Wd [G,H,H']
========================  ==============================  =======================================

Groups are those of ``cu_seqlens`` (int32, the end of every group), as in :mod:`.gemm`; rows may start and end anywhere.
Every call runs on the current device's current stream, allocates only its results and raises if the native library is
missing; there is no eager fallback.  Bounded waits that run out are reported by ``gemm.check_status``.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .. import _native as nat
from .._native import I, L, P
from . import elementwise as ew
from . import gemm

BLOCK = 32
PHASES = 4


# Descriptors, as the C side lays them out, packed in one call: filling a ctypes structure field by field, or converting as
# many arguments, took as long as the launch.
# product: four operand pointers; rows, K, groups, weight rows, N, gated, zero_tail, check_groups; cu_seqlens, pads,
#   row_scale, out, gate, up, codes, scales, d_act, d_scale; ldc, status, timeout
# quantise: x, x2, codes, scales, rows_ptr; batch, stride; type, mats, rows, cols, along_cols, out_rows, phases, unused
# dequantise: codes, scales, out, rows_ptr; mats, rows, cols, pair, in_rows, fp32
_DESC = struct.Struct("@4P8i10PqPq")
# dgrad: a[2], codes, scales, out, cu_seqlens, pads; lda, ldc; rows, K, N, nseg, groups, weight rows, fp32, unused; status, timeout
_DGRAD = struct.Struct("@7P2q8iPq")
_QUANT = struct.Struct("@5P2q8i")
_DEQUANT = struct.Struct("@4P6i")

nat.declare("mep_mx_quant_desc_bytes", I, [])
nat.declare("mep_mx_quantize", I, [ctypes.c_char_p, P])
nat.declare("mep_mx_dequantize", I, [ctypes.c_char_p, P])
nat.declare("mep_mx_desc_bytes", I, [])
nat.declare("mep_mx_dgrad_desc_bytes", I, [])
nat.declare("mep_mx_dgrad_launch", I, [ctypes.c_char_p, P])
nat.declare("mep_mx_sum_parts", I, [P, I, I, P, P, P])
nat.declare("mep_mx_gemm_launch", I, [ctypes.c_char_p, P])

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_MAX = 2 ** 31 - 1
_checked_layout = False


def _check_layouts() -> None:
    global _checked_layout
    assert nat.call("mep_mx_desc_bytes") == _DESC.size, "MxDesc layout mismatch"
    assert nat.call("mep_mx_dgrad_desc_bytes") == _DGRAD.size, "MxDgradDesc layout mismatch"
    assert nat.call("mep_mx_quant_desc_bytes") == (_QUANT.size << 16 | _DEQUANT.size), "MxQuantDesc layout mismatch"
    _checked_layout = True


def _launch_native(name: str, desc: bytes, what: str) -> None:
    if not _checked_layout:
        _check_layouts()
    rc = nat.call(name, desc, nat.stream())
    if rc != 0:
        ew._rc(rc, what)


_device = torch._C._cuda_getDevice       # (torch.cuda.current_device() without its check that CUDA is initialised)


def _here(t: torch.Tensor, name: str) -> int:
    """Index of the current device, which ``t`` has to be on."""
    at = t.get_device()
    assert at >= 0, f"{name} must be a CUDA tensor"
    assert at == _device(), f"{name} is on {t.device}, not on the current device"
    return at


def _rows_ptr(rows_ptr, index: int) -> int:
    if rows_ptr is None:
        return 0
    assert rows_ptr.dtype == torch.int32 and rows_ptr.numel() == 1 and rows_ptr.get_device() == index, \
        "rows_ptr must be one int32 on the operand's device"
    return rows_ptr.data_ptr()


class MxTensor:
    """A quantised operand of ``shape`` ``[rows, K]`` or ``[G, rows, K]``, blocks along K; ``[2, G, rows, K]`` for a
    gate and an up projection packed together.

    ``codes`` uint8 ``[..., rows, bytes]``: two elements a byte, the earlier one in the low half, rows padded with
    zeros to whole blocks.  ``scales`` uint8 ``[G, row atoms, K atoms, 512]``: E8M0 bytes in atoms of 128 rows x 4 blocks,
    row ``r`` and block ``j`` at ``16 (r % 32) + 4 (r // 32 % 4) + j % 4``; those of blocks behind the last are anything but
    NaN (255).  One matrix has them at four phases, ``[4, row atoms, K atoms, 512]``: the atoms of phase ``s`` begin at row
    ``32 s`` (row ``r`` is its row ``r - 32 s``), for the products' tiles of token rows, which start at any multiple of 32."""

    __slots__ = ("shape", "_codes", "_scales", "_data", "_index", "_mats", "_rows", "_at")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape):
        shape = tuple(int(n) for n in shape)
        assert len(shape) in (2, 3, 4) and (len(shape) < 4 or shape[0] == 2), "[rows, K], [G, rows, K] or [2, G, rows, K]"
        assert codes.dtype == torch.uint8 and scales.dtype == torch.uint8 and codes.device == scales.device
        sizes = _sizes(shape)
        assert codes.is_contiguous() and scales.is_contiguous() and (tuple(codes.shape), tuple(scales.shape)) == sizes, \
            f"a tensor of shape {shape} has codes and scales of {sizes}"
        assert codes.data_ptr() % 16 == 0 and scales.data_ptr() % 16 == 0, "codes and scales must be 16-byte aligned"
        self._codes, self._scales, self._data = codes, scales, codes
        self.shape, self._index = shape, codes.get_device()
        self._at = codes.data_ptr(), scales.data_ptr()
        self._mats, self._rows = (1 if len(shape) == 2 else shape[-3]), sizes[0][-2]

    @classmethod
    def _empty(cls, shape, device, index: int) -> "MxTensor":
        """A new one; codes and scales share an allocation, whose two views are made when somebody asks for them."""
        rows, K = shape[-2], shape[-1]
        if len(shape) == 2:
            mats, copies = 1, PHASES
        else:
            mats = copies = shape[-3]
            if len(shape) == 4:
                rows = (rows + 15) // 16 * 32
        n = (mats * rows * ((K + 31) // 32) + 31) // 32 * 512
        self = cls.__new__(cls)
        self._data = data = torch.empty(n + copies * ((rows + 127) // 128) * ((K + 127) // 128) * 512, dtype=torch.uint8, device=device)
        self._codes = self._scales = None
        at = data.data_ptr()
        self.shape, self._index, self._mats, self._rows, self._at = shape, index, mats, rows, (at, at + n)
        return self

    def _saved(self):
        """``(tensors, rest)`` to save and to make it again from, for autograd's saved tensors: they are then freed, or moved
        by hooks, as others are."""
        own = self._data.dim() == 1
        tensors = (self._data,) if own else (self._codes, self._scales)
        return tensors, (self.shape, self._mats, self._rows, self._at[1] - self._at[0] if own else None)

    @classmethod
    def _again(cls, tensors, rest) -> "MxTensor":
        self = cls.__new__(cls)
        self.shape, self._mats, self._rows, scales_at = rest
        self._data = data = tensors[0]
        self._index, at = data.get_device(), data.data_ptr()
        if scales_at is None:
            self._codes, self._scales = tensors
            self._at = at, tensors[1].data_ptr()
        else:
            self._codes = self._scales = None
            self._at = at, at + scales_at
        return self

    def _views(self):
        if self._codes is None:
            codes, scales = _sizes(self.shape)
            n, m = math.prod(codes), math.prod(scales)
            self._codes, self._scales = self._data[:n].view(codes), self._data[self._data.numel() - m:].view(scales)
        return self._codes, self._scales

    @property
    def codes(self) -> torch.Tensor:
        return self._views()[0]

    @property
    def scales(self) -> torch.Tensor:
        return self._views()[1]

    @property
    def device(self):
        return self._data.device

    @property
    def nbytes(self) -> int:
        return self.codes.nbytes + self.scales.nbytes

    def __repr__(self):
        return f"MxTensor(shape={self.shape}, device={self.device})"

    def dequantize(self, dtype: torch.dtype = torch.bfloat16, *, rows_ptr: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The values, exactly, in bf16 or fp32, of this tensor's shape;
        gate first, then up, for a packed pair.  ``rows_ptr`` as in :func:`quantize`."""
        assert dtype is torch.bfloat16 or dtype is torch.float32, "values are bf16 or fp32"
        data, shape = self._data, self.shape
        index = _here(data, "the operand")
        count = 0
        if rows_ptr is not None:
            assert len(shape) == 2, "rows_ptr goes with one matrix"
            count = _rows_ptr(rows_ptr, index)
        out = torch.empty(shape, dtype=dtype, device=data.device)
        _launch_native("mep_mx_dequantize",
                       _DEQUANT.pack(*self._at, out.data_ptr(), count, self._mats, shape[-2], shape[-1], len(shape) == 4, self._rows,
                                     dtype is torch.float32), "mx dequantise")
        return out


def _sizes(shape):
    """Sizes of a tensor's codes and scales.  (The rows of a packed pair are the gate's and the up projection's in turns
    of 16.)"""
    rows, K = shape[-2:]
    if len(shape) == 4:
        rows = (rows + 15) // 16 * 32
    code_bytes, atoms, k_atoms = (K + 31) // 32 * 16, (rows + 127) // 128, (K + 127) // 128
    if len(shape) == 2:
        return (rows, code_bytes), (PHASES, atoms, k_atoms, 512)
    G = shape[-3]
    return (G, rows, code_bytes), (G, atoms, k_atoms, 512)


def _operand(x: torch.Tensor, name: str):
    """Device, sizes, strides and type of what is to be quantised."""
    index = _here(x, name)
    size, stride, kind = x.shape, x.stride(), _TYPES.get(x.dtype)
    assert kind is not None, f"{name} must be bf16, fp16 or fp32"
    assert len(size) == 2 or len(size) == 3, f"{name} must be [rows, K] or [G, rows, K]"
    cols = size[-1]
    assert 1 <= cols <= _MAX and size[-2] <= _MAX, f"{name} has no columns, or too many rows"
    assert cols == 1 or stride[-1] == 1, f"{name} must be dense along its last axis"
    return index, size, stride, kind


def quantize(x: torch.Tensor, axis: int = -1, *, rows_ptr: Optional[torch.Tensor] = None) -> MxTensor:
    """``x`` ``[rows, K]`` or ``[G, rows, K]`` (bf16, fp16, fp32; any strides with a dense last axis) with the
    reduction along ``axis``: -1, or -2 for ``x`` ``[K, rows]`` / ``[G, K, rows]``, whose transpose is stored.

    ``rows_ptr`` (device int32, one matrix, ``axis=-1``) bounds the rows that are read without a host sync; the others'
    codes and scales are left undefined.  No gradient passes (see :func:`expert_ffn`)."""
    index, size, stride, kind = _operand(x, "x")
    assert axis == -1 or axis == -2, "axis must be -1 or -2"
    rows, cols = size[-2], size[-1]
    mats, batch = (size[0], stride[0]) if len(size) == 3 else (1, 0)
    count, one = 0, len(size) == 2
    if rows_ptr is not None:
        assert one and axis == -1, "rows_ptr goes with one matrix and axis=-1"
        count = _rows_ptr(rows_ptr, index)
    if axis == -1:
        n, k = rows, cols
    else:
        n, k = cols, rows
        assert k >= 1, "the reduction is empty"
    q = MxTensor._empty((n, k) if one else (mats, n, k), x.device, index)
    _launch_native("mep_mx_quantize",
                   _QUANT.pack(x.data_ptr(), 0, *q._at, count, batch, stride[-2], kind, mats, rows, cols, axis == -2, n,
                               PHASES if one else 1, 0), "mx quantise")
    return q


def pack_gate_up(wg: torch.Tensor, wu: torch.Tensor) -> MxTensor:
    """Gate and up projections ``[G, H, H']`` (or one expert's ``[H, H']``), quantised along H, as the one operand of
    :func:`gateup_swiglu`; its ``shape`` is ``[2, G, H', H]``."""
    index, size, stride, kind = _operand(wg, "wg")
    _operand(wu, "wu")
    assert size == wu.shape and wg.dtype == wu.dtype, "wg and wu must be alike"
    assert size[-2] >= 1, "the reduction is empty"
    if stride != wu.stride():
        wg, wu = wg.contiguous(), wu.contiguous()
        stride = wg.stride()
    G, batch = (size[0], stride[0]) if len(size) == 3 else (1, 0)
    H, Hp = size[-2], size[-1]
    q = MxTensor._empty((2, G, Hp, H), wg.device, index)
    _launch_native("mep_mx_quantize",
                   _QUANT.pack(wg.data_ptr(), wu.data_ptr(), *q._at, 0, batch, stride[-2], kind, G, H, Hp, 1, q._rows, 1, 0),
                   "mx quantise")
    return q


def _launch(a: MxTensor, w: MxTensor, N: int, gated: int, cu_seqlens, pads, row_scale, out: int, gate: int, up: int, codes: int,
            scales: int, ldc: int, d_act: int = 0, d_scale: int = 0, zero_tail: int = 0, check_groups: int = 0) -> None:
    index, groups, (rows, K) = a._index, w._mats, a.shape
    assert index >= 0 and index == _device(), "the operands are not on the current device"
    assert w._index == index and w.shape[-1] == K, "operands do not go together"
    assert 1 <= groups <= 1024, "1 to 1024 groups"
    cu = pad = scale = 0
    if cu_seqlens is None:
        assert groups == 1, "several groups need cu_seqlens"
        assert pads is None, "padding ranges go with cu_seqlens"
    else:
        assert cu_seqlens.dtype is torch.int32 and cu_seqlens.get_device() == index and cu_seqlens.is_contiguous() \
            and cu_seqlens.numel() == groups, "cu_seqlens must be int32, one entry a group"
        cu = cu_seqlens.data_ptr()
        if pads is not None:
            size = pads.shape
            assert pads.dtype is torch.int32 and pads.get_device() == index and pads.is_contiguous() and len(size) == 2 \
                and size[1] == 2 and size[0] >= groups, "pads must be int32 [groups, 2]"
            pad = pads.data_ptr()
    if row_scale is not None:
        assert row_scale.dtype is torch.float32 and row_scale.get_device() == index and row_scale.is_contiguous() \
            and row_scale.dim() == 1 and row_scale.numel() >= rows, "row_scale must be fp32, one a row"
        scale = row_scale.data_ptr()
    status = gemm._status.get(index)
    if status is None:
        status = gemm.status_word(a.device)
    _launch_native("mep_mx_gemm_launch",
                   _DESC.pack(*a._at, *w._at, rows, K, groups, w._rows, N, gated, zero_tail, check_groups, cu, pad, scale, out, gate,
                              up, codes, scales, d_act, d_scale, ldc, status.data_ptr(), 0), "mx product")


def matmul(a: MxTensor, w: MxTensor, cu_seqlens: Optional[torch.Tensor] = None, *, out: Optional[torch.Tensor] = None,
           pads: Optional[torch.Tensor] = None, zero_tail: bool = False) -> torch.Tensor:
    """``y[rows of g] = a w[g]^T`` in bf16, summed in fp32: ``a`` ``[rows, K]``, ``w`` ``[G, N, K]`` with ``cu_seqlens``
    ``[G]``, or ``[N, K]`` for all rows.

    ``out`` ``[rows or more, N]`` (bf16, dense rows) takes the result; rows that belong to no group are left as they
    are, or with ``zero_tail`` become zeros where they are behind the last group.  ``pads`` (a plan's
    ``zero_fill_ranges``): which rows of the groups are padding; they become zeros without being computed."""
    assert isinstance(a, MxTensor) and isinstance(w, MxTensor) and len(w.shape) < 4, "operands must be quantised"
    assert len(a.shape) == 2, "the rows' operand is one matrix"
    rows, N = a.shape[0], w.shape[-2]
    if out is None:
        out = torch.empty((rows, N), dtype=torch.bfloat16, device=a._data.device)
        ld = N
    else:
        assert out.get_device() == a._index and out.dtype == torch.bfloat16 and out.dim() == 2
        assert out.shape[0] >= rows and out.shape[1] == N and (N <= 1 or out.stride(1) == 1)
        ld = out.stride(0)
        assert out.shape[0] < 2 or ld >= N, "rows of out overlap"
    if N > 0:
        _launch(a, w, N, 0, cu_seqlens, pads, None, out.data_ptr(), 0, 0, 0, 0, ld, zero_tail=int(zero_tail))
    return out


def gateup_swiglu(a: MxTensor, wgu: MxTensor, cu_seqlens: Optional[torch.Tensor] = None, *,
                  row_scale: Optional[torch.Tensor] = None, save_gate_up: bool = False, quantize: bool = False,
                  pads: Optional[torch.Tensor] = None):
    """``act[rows,H'] = silu(x Wg[g]) * (x Wu[g]) * row_scale`` in one product; ``(act, gate, up)``.

    ``wgu`` comes from :func:`pack_gate_up`.  ``act`` is bf16, or with ``quantize`` that bf16 value quantised along H'
    (an operand of :func:`matmul`; the bf16 tensor is not written then).  ``gate`` and ``up`` are bf16 with
    ``save_gate_up``, else ``None``; the activation is computed from their fp32 sums.  Rows that belong to no group are
    undefined.  ``pads`` as in :func:`matmul`."""
    assert isinstance(a, MxTensor) and isinstance(wgu, MxTensor) and len(wgu.shape) == 4, "wgu must come from pack_gate_up"
    assert len(a.shape) == 2, "the rows' operand is one matrix"
    rows, Hp, device = a.shape[0], wgu.shape[2], a._data.device
    gate = up = None
    if save_gate_up:
        gate, up = (torch.empty((rows, Hp), dtype=torch.bfloat16, device=device) for _ in range(2))
    if quantize:
        act = MxTensor._empty((rows, Hp), device, a._index)
        outs = 0, nat.ptr(gate), nat.ptr(up), *act._at
    else:
        act = torch.empty((rows, Hp), dtype=torch.bfloat16, device=device)
        outs = act.data_ptr(), nat.ptr(gate), nat.ptr(up), 0, 0
    if Hp > 0:
        _launch(a, wgu, Hp, 1, cu_seqlens, pads, row_scale, *outs, Hp)
    return act, gate, up


def gateup_swiglu_bwd(d_act: torch.Tensor, a: MxTensor, wgu: MxTensor, cu_seqlens: Optional[torch.Tensor] = None, *,
                      row_scale: Optional[torch.Tensor] = None, want_dscale: bool = False, pads: Optional[torch.Tensor] = None):
    """Backward of :func:`gateup_swiglu` up to the products: ``(d_gate, d_up, d_scale)`` from the gradient ``d_act``
    ``[rows, H']`` (fp32) of the activation and the operands of the forward pass, whose product is computed again: gate
    and up need not be kept.  ``d_gate`` and ``d_up`` are bf16; ``d_scale`` (fp32 ``[rows]``, with ``want_dscale``) is
    summed in a fixed order and zero for the rows behind the last group."""
    assert isinstance(a, MxTensor) and isinstance(wgu, MxTensor) and len(wgu.shape) == 4, "wgu must come from pack_gate_up"
    assert len(a.shape) == 2, "the rows' operand is one matrix"
    rows, Hp, device = a.shape[0], wgu.shape[2], a._data.device
    assert d_act.dtype == torch.float32 and d_act.get_device() == a._index and d_act.is_contiguous() \
        and tuple(d_act.shape) == (rows, Hp), "d_act must be fp32 [rows, H']"
    d_gate, d_up = (torch.empty((rows, Hp), dtype=torch.bfloat16, device=device) for _ in range(2))
    d_scale, n = None, (wgu._rows + 255) // 256 * 2
    parts = torch.empty((n, rows), dtype=torch.float32, device=device) if want_dscale else None
    if Hp > 0:
        _launch(a, wgu, Hp, 1, cu_seqlens, pads, row_scale, 0, d_gate.data_ptr(), d_up.data_ptr(), 0, 0, Hp, d_act.data_ptr(),
                nat.ptr(parts))
    if want_dscale:
        d_scale = torch.empty(rows, dtype=torch.float32, device=device)
        end = 0 if cu_seqlens is None else cu_seqlens.data_ptr() + 4 * (cu_seqlens.numel() - 1)
        ew._rc(nat.call("mep_mx_sum_parts", parts.data_ptr(), n, rows, end, d_scale.data_ptr(), nat.stream()), "mx sum")
    return d_gate, d_up, d_scale


def _dgrad(segs, w: MxTensor, cu_seqlens, pads, out: torch.Tensor) -> torch.Tensor:
    a = segs[0]
    index, K, N, groups = w._index, w.shape[-2], w.shape[-1], w._mats
    assert index >= 0 and index == _device(), "the weights are not on the current device"
    for t in segs:
        gemm._bf16(t, "rows")
        assert t.get_device() == index and t.dim() == 2 and t.shape == a.shape and t.stride(0) == a.stride(0)
    assert a.shape[1] == K and K % 8 == 0, "rows must be [rows, K], K a multiple of 8"
    assert 1 <= groups <= 1024, "1 to 1024 groups"
    cu = pad = 0
    if cu_seqlens is None:
        assert groups == 1, "several groups need cu_seqlens"
        assert pads is None, "padding ranges go with cu_seqlens"
    else:
        assert cu_seqlens.dtype is torch.int32 and cu_seqlens.get_device() == index and cu_seqlens.is_contiguous() \
            and cu_seqlens.numel() == groups, "cu_seqlens must be int32, one entry a group"
        cu, pad = cu_seqlens.data_ptr(), gemm._pads(pads, cu_seqlens) or 0
        assert pads is None or pads.get_device() == index
    assert out.get_device() == index and out.dim() == 2 and out.shape[0] >= a.shape[0] and out.shape[1] == N and out.stride(1) == 1
    assert out.shape[0] < 2 or out.stride(0) >= N, "rows of out overlap"
    _launch_native("mep_mx_dgrad_launch",
                   _DGRAD.pack(a.data_ptr(), segs[-1].data_ptr(), *w._at, out.data_ptr(), cu, pad, a.stride(0), out.stride(0),
                               a.shape[0], K, N, len(segs), groups, w._rows, out.dtype is torch.float32, 0,
                               gemm.status_word(w.device).data_ptr(), 0), "mx dgrad")
    return out


def down_dgrad(dy: torch.Tensor, wd: MxTensor, cu_seqlens: Optional[torch.Tensor] = None, *, pads: Optional[torch.Tensor] = None,
               fp32: bool = False) -> torch.Tensor:
    """``d_act[rows,H'] = dy Wd[g]`` for bf16 ``dy`` ``[rows, H]`` and 4-bit ``wd`` ``[G, H, H']`` (or ``[H, H']``): the
    gradient of :func:`matmul` with respect to the values of its rows.  bf16, or the ``fp32`` sums (padding rows and rows
    of no group are undefined then; else zeros, padding and behind the last group, whatever ``dy`` holds there)."""
    assert isinstance(wd, MxTensor) and len(wd.shape) < 4, "wd must come from quantize"
    out = torch.empty(dy.shape[0], wd.shape[-1], dtype=torch.float32 if fp32 else torch.bfloat16, device=wd.device)
    return _dgrad((dy,), wd, cu_seqlens, pads, out)


def gateup_dgrad(dg: torch.Tensor, du: torch.Tensor, wgu: MxTensor, cu_seqlens: Optional[torch.Tensor] = None, *,
                 pads: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``dx[rows,H] = dg Wg[g]^T + du Wu[g]^T`` for bf16 ``dg``/``du`` ``[rows, H']`` and the packed weights of
    :func:`gateup_swiglu`; zeros in padding rows and behind the last group, whatever ``dg`` and ``du`` hold there.
    ``out`` ``[rows or more, H]`` bf16 takes it."""
    assert isinstance(wgu, MxTensor) and len(wgu.shape) == 4, "wgu must come from pack_gate_up"
    if out is None:
        out = torch.empty(dg.shape[0], wgu.shape[-1], dtype=torch.bfloat16, device=wgu.device)
    assert out.dtype is torch.bfloat16, "dx is bf16"
    return _dgrad((dg, du), wgu, cu_seqlens, pads, out)


def save_operands(ctx, operands, *tensors) -> None:
    """``ctx.save_for_backward`` of operands and tensors (or ``None``)."""
    saved = [q._saved() for q in operands]
    ctx.mx_rest = [(len(t), rest) for t, rest in saved]
    ctx.save_for_backward(*(x for t, _ in saved for x in t), *tensors)


def saved_operands(ctx):
    """``(operands, tensors)`` saved by :func:`save_operands`."""
    tensors, at, operands = ctx.saved_tensors, 0, []
    for n, rest in ctx.mx_rest:
        operands.append(MxTensor._again(tensors[at:at + n], rest))
        at += n
    return operands, tensors[at:]


def _pack(wg, wu, wd):
    """``(wgu, wd)`` quantised: as they are if they are so already."""
    if isinstance(wg, MxTensor):
        assert wu is None and isinstance(wd, MxTensor), "packed weights: wg from pack_gate_up, wu None, wd from quantize"
        return wg, wd
    return pack_gate_up(wg, wu), quantize(wd)


class _ExpertFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, wd, row_scale, cu_seqlens, pads, recorded):
        # (needs_input_grad says which inputs require grad, also where nothing is recorded)
        wgu, wdq = _pack(wg, wu, wd)
        keep = recorded and any(ctx.needs_input_grad)
        xq = quantize(x, rows_ptr=None if cu_seqlens is None else cu_seqlens[-1:])
        act, _, _ = gateup_swiglu(xq, wgu, cu_seqlens, row_scale=row_scale, quantize=True, pads=pads)
        y = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
        H = x.shape[1]
        _launch(act, wdq, H, 0, cu_seqlens, pads, None, y.data_ptr(), 0, 0, 0, 0, H, zero_tail=1,
                check_groups=int(recorded and any(ctx.needs_input_grad[1:4])))
        if keep:
            ctx.shapes = None if isinstance(wg, MxTensor) else (wg.shape, wd.shape)
            save_operands(ctx, (xq, act, wgu, wdq), row_scale, cu_seqlens, pads)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (xq, act, wgu, wdq), (row_scale, cu, pads) = saved_operands(ctx)
        need_x, need_g, need_u, need_d, need_s = ctx.needs_input_grad[:5]
        dy = dy.contiguous()
        if dy.data_ptr() % 16 != 0:
            dy = dy.clone()
        (G, Hp, H), rows_ptr = wgu.shape[1:], None if cu is None else cu[-1:]
        bf16 = dict(dtype=torch.bfloat16, device=dy.device)
        grads = [None] * 3
        if dy.shape[0] == 0:
            zeros = lambda need, i: torch.zeros(ctx.shapes[i], **bf16) if need else None
            return (torch.empty_like(dy) if need_x else None, zeros(need_g, 0), zeros(need_u, 0), zeros(need_d, 1),
                    torch.empty_like(row_scale) if need_s else None, None, None, None)
        if need_d:
            grads[2] = torch.empty(G, H, Hp, **bf16)
            gemm.wgrad(dy, act.dequantize(rows_ptr=rows_ptr), cu, grads[2], pads=pads)
            grads[2] = grads[2].view(ctx.shapes[1])
        dx = d_scale = None
        if need_x or need_g or need_u or need_s:
            d_act = down_dgrad(dy, wdq, cu, pads=pads, fp32=True)
            d_gate, d_up, d_scale = gateup_swiglu_bwd(d_act, xq, wgu, cu, row_scale=row_scale, want_dscale=need_s, pads=pads)
            if need_x:
                dx = gateup_dgrad(d_gate, d_up, wgu, cu, pads=pads)
            if need_g or need_u:
                out = torch.empty(2, G, H, Hp, **bf16)
                gemm.wgrad2(xq.dequantize(rows_ptr=rows_ptr), (d_gate, d_up), cu, (out[0], out[1]), pads=pads)
                grads[:2] = (out[i].view(ctx.shapes[0]) for i in range(2))
        return dx, grads[0], grads[1], grads[2], d_scale, None, None, None


def expert_ffn(x: torch.Tensor, wg, wu, wd, cu_seqlens: Optional[torch.Tensor] = None, *,
               row_scale: Optional[torch.Tensor] = None, pads: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[rows,H] = (silu(x Wg[g]) * (x Wu[g]) * row_scale) Wd[g]^T`` over quantised operands, differentiable.

    bf16 ``x`` ``[rows, H]`` and ``wg``/``wu``/``wd`` ``[G, H, H']`` (one expert: ``[H, H']``), which are quantised in the
    call; or weights packed before, ``expert_ffn(x, pack_gate_up(wg, wu), None, quantize(wd), ...)``, which get no
    gradient.  ``x`` is quantised along H, the activation (rounded to bf16) along H'.

    The gradients are those of the formula with the quantised operands in it; the quantisation itself is passed
    straight through: ``d Wg = x^T d_gate`` has the quantised ``x``, ``d x`` the quantised weights.  What forward keeps
    are the operands in 4 bits; backward computes gate and up again.  Sums run in fp32; ``d gate`` and ``d up`` are
    rounded to bf16, as operands of the bf16 products of :mod:`.gemm`, and the results once more.

    Rows behind the last group get zeros, in ``y`` and in ``x``'s gradient.  For gradients H must be a multiple of 128
    and H' of 8, and for the weights' every group's rows a multiple of 64, padding rows of ``x`` being zero and of ``y``'s
    gradient finite (what ``Buffer.dispatch`` gives), but for a group that ends with ``x`` itself; the weight grads of
    other groups are NaN, and ``gemm.check_status`` reports them, from the forward pass on, where autograd records it.
    Every call can be captured into a CUDA graph, forward and backward (``utils.graph.GraphedStep``); as with any captured
    ``backward()``, no eager graph of the same leaves may be alive meanwhile."""
    assert isinstance(x, torch.Tensor) and x.dim() == 2 and x.dtype == torch.bfloat16, "x must be bf16 [rows, H]"
    _operand(x, "x")
    H = x.shape[1]
    if isinstance(wg, MxTensor):
        assert wu is None and isinstance(wd, MxTensor), "packed weights: wg from pack_gate_up, wu None, wd from quantize"
        assert len(wg.shape) == 4 and len(wd.shape) < 4, "packed weights: wg from pack_gate_up, wd from quantize"
        G, Hp = wg.shape[1], wg.shape[2]
        assert wg.shape[3] == H and wd.shape[-2:] == (H, Hp), "operands do not go together"
        assert (wd.shape[0] if len(wd.shape) == 3 else 1) == G, "operands do not go together"
        trained = ()
    else:
        trained = (wg, wu, wd)
        for name, w in zip(("wg", "wu", "wd"), trained):
            assert _operand(w, name)[3] == 0, f"{name} must be bf16"
        assert wg.shape == wu.shape == wd.shape and wg.shape[-2] == H, "weights must be [G, H, H'] alike"
        Hp = wg.shape[-1]
    if row_scale is not None:
        assert row_scale.dtype == torch.float32 and row_scale.dim() == 1 and row_scale.shape[0] == x.shape[0], "one fp32 scale a row"
        row_scale = row_scale.contiguous()
    assert pads is None or cu_seqlens is not None, "padding ranges go with cu_seqlens"
    recorded = torch.is_grad_enabled()
    if recorded and any(t.requires_grad for t in (x, *trained) + (() if row_scale is None else (row_scale,))):
        assert H % 128 == 0 and Hp % 8 == 0, "gradients need H % 128 == 0 and H' % 8 == 0"
    return _ExpertFFN.apply(x, wg, wu, wd, row_scale, cu_seqlens, pads, recorded)
