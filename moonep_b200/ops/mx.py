"""Microscaled 4-bit operands of the expert FFN: quantisation, grouped products, and the FFN itself for serving and
for training (``csrc/device/mx_quant.cu``, ``mx_gemm.cuh``).

An operand is quantised along the reduction in blocks of 32: with ``a = max |x|`` of a block and
``e = floor(log2 a) - 2`` (within [-127, 127]) every element becomes ``x / 2^e`` rounded to the nearest of
0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code, larger ones to 6) times ``2^e``.  A block with a NaN or an infinity
is all NaN.  17 bits stand for 32 of bf16, and the tensor cores multiply such operands as they are.

========================  ==============================  =======================================
op                        math                            operands
========================  ==============================  =======================================
``quantize``              x -> ``MxTensor``               bf16, fp16, fp32; any sizes
``pack_gate_up``          Wg, Wu -> one ``MxTensor``      [G, H, H'] each, blocks along H
``matmul``                y = a W[g]^T                    a [rows,K] . W [G,N,K]
``gateup_swiglu``         act = silu(x Wg)*(x Wu)*w       x [rows,H] . packed Wg, Wu
``expert_ffn``            y = act Wd^T, with gradients    bf16 x [rows,H], Wg/Wu/Wd [G,H,H']
========================  ==============================  =======================================

Groups are those of ``cu_seqlens`` (int32, the end of every group), as in :mod:`.gemm`; rows may start and end anywhere.
Every call runs on the current device's current stream, allocates only its results and raises if the native library is
missing; there is no eager fallback.  Bounded waits that run out are reported by ``gemm.check_status``.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .. import _native as nat
from .._native import I, L, P
from . import elementwise as ew
from . import gemm

BLOCK = 32
PHASES = 4


class _MxDesc(ctypes.Structure):
    _fields_ = [
        ("a_codes", P), ("a_scales", P), ("w_codes", P), ("w_scales", P),
        ("rows", ctypes.c_int32), ("K", ctypes.c_int32), ("ngroups", ctypes.c_int32),
        ("w_rows", ctypes.c_int32), ("N", ctypes.c_int32), ("gated", ctypes.c_int32),
        ("cu_seqlens", P), ("pads", P), ("row_scale", P),
        ("out", P), ("gate", P), ("up", P), ("codes", P), ("scales", P),
        ("ldc", ctypes.c_int64), ("status", P), ("timeout_ns", ctypes.c_int64),
    ]


nat.declare("mep_mx_quantize", I, [P, I, L, L, I, I, I, I, I, I, I, P, P, P, P])
nat.declare("mep_mx_dequantize", I, [P, P, I, I, I, I, I, P, I, P, P])
nat.declare("mep_mx_desc_bytes", I, [])
nat.declare("mep_mx_gemm_launch", I, [ctypes.POINTER(_MxDesc), P])

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_MAX = 2 ** 31 - 1
_checked_layout = False


def _atoms(n: int) -> int:
    return (n + 127) // 128


def _here(t: torch.Tensor, name: str) -> torch.Tensor:
    assert t.is_cuda, f"{name} must be a CUDA tensor"
    assert t.device.index == torch.cuda.current_device(), f"{name} is on {t.device}, not on the current device"
    return t


def _rows_ptr(rows_ptr, device):
    if rows_ptr is None:
        return None
    assert rows_ptr.dtype == torch.int32 and rows_ptr.numel() == 1 and rows_ptr.device == device, \
        "rows_ptr must be one int32 on the operand's device"
    return rows_ptr.data_ptr()


class MxTensor:
    """A quantised operand of ``shape`` ``[rows, K]`` or ``[G, rows, K]``, blocks along K; ``[2, G, rows, K]`` for a
    gate and an up projection packed together.

    ``codes`` uint8 ``[..., rows, bytes]``: two elements a byte, the earlier one in the low half, rows padded to whole
    blocks.  ``scales`` uint8 ``[G, row atoms, K atoms, 512]``: E8M0 bytes in atoms of 128 rows x 4 blocks, row ``r``
    and block ``j`` at ``16 (r % 32) + 4 (r // 32 % 4) + j % 4``.  One matrix has them at four phases, ``[4, row atoms,
    K atoms, 512]``: the atoms of phase ``s`` begin at row ``32 s`` (row ``r`` is its row ``r - 32 s``), for the products'
    tiles of token rows, which start at any multiple of 32."""

    __slots__ = ("codes", "scales", "shape")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape):
        shape = tuple(int(n) for n in shape)
        assert len(shape) in (2, 3, 4) and (len(shape) < 4 or shape[0] == 2), "[rows, K], [G, rows, K] or [2, G, rows, K]"
        rows, K = _stored_rows(shape), shape[-1]
        lead = shape[-3:-2]
        assert codes.dtype == torch.uint8 and scales.dtype == torch.uint8 and codes.device == scales.device
        assert codes.is_contiguous() and tuple(codes.shape) == (*lead, rows, (K + BLOCK - 1) // BLOCK * (BLOCK // 2))
        assert scales.is_contiguous() and tuple(scales.shape) == (*(lead or (PHASES,)), _atoms(rows), _atoms(K), 512)
        self.codes, self.scales, self.shape = codes, scales, shape

    @property
    def device(self):
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.nbytes + self.scales.nbytes

    def __repr__(self):
        return f"MxTensor(shape={self.shape}, device={self.device})"

    def dequantize(self, dtype: torch.dtype = torch.bfloat16, *, rows_ptr: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The values, bf16 (exact down to 2^-133, the last bit of its subnormals) or fp32, of this tensor's shape;
        gate first, then up, for a packed pair.  ``rows_ptr`` as in :func:`quantize`."""
        assert dtype in (torch.bfloat16, torch.float32), "values are bf16 or fp32"
        _here(self.codes, "the operand")
        pair = len(self.shape) == 4
        assert rows_ptr is None or len(self.shape) == 2, "rows_ptr goes with one matrix"
        mats = self.codes.shape[0] if self.codes.dim() == 3 else 1
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        for i in range(2 if pair else 1):
            dst = out[i] if pair else out
            ew._rc(nat.call("mep_mx_dequantize", self.codes.data_ptr(), self.scales.data_ptr(), mats, self.shape[-2],
                            self.shape[-1], i + 1 if pair else 0, self.codes.shape[-2], _rows_ptr(rows_ptr, self.device),
                            int(dtype == torch.float32), dst.data_ptr(), nat.stream()), "mx dequantise")
        return out


def _stored_rows(shape) -> int:
    """Rows of a matrix of codes: for a pair the gate's and the up projection's in turns of 16."""
    return shape[-2] if len(shape) < 4 else (shape[-2] + 15) // 16 * 32


def _empty(shape, device, zero: bool = False) -> MxTensor:
    rows, K, lead = _stored_rows(shape), shape[-1], shape[-3:-2]
    make = torch.zeros if zero else torch.empty
    codes = make(*lead, rows, (K + BLOCK - 1) // BLOCK * (BLOCK // 2), dtype=torch.uint8, device=device)
    scales = make(*(lead or (PHASES,)), _atoms(rows), _atoms(K), 512, dtype=torch.uint8, device=device)
    return MxTensor(codes, scales, shape)


def _quantize_into(q: MxTensor, x: torch.Tensor, axis: int, interleave: int, rows_ptr) -> None:
    mats, (rows, cols) = (x.shape[0] if x.dim() == 3 else 1), x.shape[-2:]
    batch = x.stride(0) if x.dim() == 3 else 0
    ew._rc(nat.call("mep_mx_quantize", x.data_ptr(), _TYPES[x.dtype], batch, x.stride(-2), mats, rows, cols, int(axis == -2),
                    interleave, q.codes.shape[-2], PHASES if q.codes.dim() == 2 else 1, _rows_ptr(rows_ptr, x.device), q.codes.data_ptr(), q.scales.data_ptr(),
                    nat.stream()), "mx quantise")


def _operand(x: torch.Tensor, name: str) -> torch.Tensor:
    _here(x, name)
    assert x.dtype in _TYPES, f"{name} must be bf16, fp16 or fp32"
    assert x.dim() in (2, 3), f"{name} must be [rows, K] or [G, rows, K]"
    assert x.shape[-1] >= 1 and x.shape[-2] <= _MAX and x.shape[-1] <= _MAX
    assert x.shape[-1] == 1 or x.stride(-1) == 1, f"{name} must be dense along its last axis"
    return x


def quantize(x: torch.Tensor, axis: int = -1, *, rows_ptr: Optional[torch.Tensor] = None) -> MxTensor:
    """``x`` ``[rows, K]`` or ``[G, rows, K]`` (bf16, fp16, fp32; any strides with a dense last axis) with the
    reduction along ``axis``: -1, or -2 for ``x`` ``[K, rows]`` / ``[G, K, rows]``, whose transpose is stored.

    ``rows_ptr`` (device int32, one matrix, ``axis=-1``) bounds the rows that are read without a host sync; the others'
    codes and scales are left undefined.  No gradient passes (see :func:`expert_ffn`)."""
    _operand(x, "x")
    assert axis in (-1, -2), "axis must be -1 or -2"
    assert rows_ptr is None or (x.dim() == 2 and axis == -1), "rows_ptr goes with one matrix and axis=-1"
    x = x.detach()
    shape = x.shape if axis == -1 else (*x.shape[:-2], x.shape[-1], x.shape[-2])
    assert shape[-1] >= 1, "the reduction is empty"
    q = _empty(shape, x.device)
    _quantize_into(q, x, axis, 0, rows_ptr)
    return q


def pack_gate_up(wg: torch.Tensor, wu: torch.Tensor) -> MxTensor:
    """Gate and up projections ``[G, H, H']`` (or one expert's ``[H, H']``), quantised along H, as the one operand of
    :func:`gateup_swiglu`; its ``shape`` is ``[2, G, H', H]``."""
    _operand(wg, "wg"), _operand(wu, "wu")
    assert wg.shape == wu.shape and wg.dtype == wu.dtype and wg.device == wu.device, "wg and wu must be alike"
    assert wg.shape[-2] >= 1, "the reduction is empty"
    wg, wu = (w.detach() if w.dim() == 3 else w.detach()[None] for w in (wg, wu))
    G, H, Hp = wg.shape
    q = _empty((2, G, Hp, H), wg.device, zero=Hp % 16 != 0)      # (the last turn of 16 is not full: zeros)
    _quantize_into(q, wg, -2, 1, None)
    _quantize_into(q, wu, -2, 2, None)
    return q


def _launch(a: MxTensor, w: MxTensor, N: int, gated: bool, cu_seqlens, pads, row_scale, outs, ldc: int) -> None:
    global _checked_layout
    assert len(a.shape) == 2, "the rows' operand is one matrix"
    _here(a.codes, "a")
    assert w.device == a.device and w.shape[-1] == a.shape[-1], "operands do not go together"
    ngroups = w.codes.shape[0] if w.codes.dim() == 3 else 1
    assert 1 <= ngroups <= 1024, "1 to 1024 groups"
    d = _MxDesc()
    d.a_codes, d.a_scales, d.rows = a.codes.data_ptr(), a.scales.data_ptr(), a.shape[0]
    d.w_codes, d.w_scales, d.w_rows = w.codes.data_ptr(), w.scales.data_ptr(), w.codes.shape[-2]
    d.K, d.N, d.ngroups, d.gated = a.shape[1], N, ngroups, int(gated)
    if cu_seqlens is None:
        assert ngroups == 1, "several groups need cu_seqlens"
    else:
        assert cu_seqlens.device == a.device and cu_seqlens.numel() == ngroups, "one entry of cu_seqlens a group"
        d.cu_seqlens = gemm._groups(cu_seqlens, None)[0]
        if pads is not None:
            assert pads.device == a.device
            d.pads = gemm._pads(pads, cu_seqlens)
    if row_scale is not None:
        assert row_scale.dtype == torch.float32 and row_scale.device == a.device and row_scale.is_contiguous()
        assert row_scale.dim() == 1 and row_scale.numel() >= a.shape[0], "one scale a row"
        d.row_scale = row_scale.data_ptr()
    for name, t in outs.items():
        setattr(d, name, nat.ptr(t))
    d.ldc = ldc
    d.status = gemm.status_word(a.device).data_ptr()
    if not _checked_layout:
        assert nat.call("mep_mx_desc_bytes") == ctypes.sizeof(_MxDesc), "MxDesc layout mismatch"
        _checked_layout = True
    ew._rc(nat.call("mep_mx_gemm_launch", ctypes.byref(d), nat.stream()), "mx product")


def matmul(a: MxTensor, w: MxTensor, cu_seqlens: Optional[torch.Tensor] = None, *, out: Optional[torch.Tensor] = None,
           pads: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[rows of g] = a w[g]^T`` in bf16, summed in fp32: ``a`` ``[rows, K]``, ``w`` ``[G, N, K]`` with ``cu_seqlens``
    ``[G]``, or ``[N, K]`` for all rows.

    ``out`` ``[rows or more, N]`` (bf16, dense rows) takes the result; rows that belong to no group are left as they
    are.  ``pads`` (a plan's ``zero_fill_ranges``): which rows of the groups are padding; they become zeros without
    being computed."""
    assert isinstance(a, MxTensor) and isinstance(w, MxTensor) and len(w.shape) < 4, "operands must be quantised"
    N = w.shape[-2]
    if out is None:
        out = torch.empty(a.shape[0], N, dtype=torch.bfloat16, device=a.device)
    else:
        assert out.device == a.device and out.dtype == torch.bfloat16 and out.dim() == 2
        assert out.shape[0] >= a.shape[0] and out.shape[1] == N and (N == 1 or out.stride(1) == 1)
        assert out.shape[0] < 2 or out.stride(0) >= N, "rows of out overlap"
    if N > 0:
        _launch(a, w, N, False, cu_seqlens, pads, None, dict(out=out), out.stride(0) if out.shape[0] > 1 else max(N, out.stride(0)))
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
    rows, Hp = a.shape[0], wgu.shape[2]
    new = lambda: torch.empty(rows, Hp, dtype=torch.bfloat16, device=a.device)
    gate, up = (new(), new()) if save_gate_up else (None, None)
    act = _empty((rows, Hp), a.device) if quantize else new()
    outs = dict(gate=gate, up=up, **(dict(codes=act.codes, scales=act.scales) if quantize else dict(out=act)))
    _launch(a, wgu, Hp, True, cu_seqlens, pads, row_scale, outs, Hp)
    return act, gate, up


def _pack(wg, wu, wd):
    """``(wgu, wd)`` quantised: as they are if they are so already."""
    if isinstance(wg, MxTensor):
        assert wu is None and isinstance(wd, MxTensor), "packed weights: wg from pack_gate_up, wu None, wd from quantize"
        return wg, wd
    return pack_gate_up(wg, wu), quantize(wd)


class _ExpertFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, wd, row_scale, cu_seqlens, pads):
        wgu, wdq = _pack(wg, wu, wd)
        keep = any(ctx.needs_input_grad)
        xq = quantize(x, rows_ptr=None if cu_seqlens is None else cu_seqlens[-1:])
        act, gate, up = gateup_swiglu(xq, wgu, cu_seqlens, row_scale=row_scale, save_gate_up=keep, quantize=True, pads=pads)
        # (a pass over all rows leaves none; rows that belong to no group are zeros)
        new = torch.empty if cu_seqlens is None else torch.zeros
        y = matmul(act, wdq, cu_seqlens, pads=pads, out=new(x.shape, dtype=torch.bfloat16, device=x.device))
        if keep:
            ctx.packed, ctx.frozen = (xq, act, wgu, wdq), isinstance(wg, MxTensor)
            ctx.shapes = None if ctx.frozen else (wg.shape, wd.shape)
            ctx.save_for_backward(gate, up, row_scale, cu_seqlens, pads)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        xq, act, wgu, wdq = ctx.packed
        gate, up, row_scale, cu, pads = ctx.saved_tensors
        need_x, need_g, need_u, need_d, need_s = ctx.needs_input_grad[:5]
        dy = dy.contiguous()
        G = wgu.shape[1]
        rows_ptr = None if cu is None else cu[-1:]
        H, Hp = xq.shape[1], wgu.shape[2]
        grads = [None] * 3
        f32 = dict(dtype=torch.float32, device=dy.device)
        if need_d:
            g = torch.empty(G, H, Hp, **f32)
            gemm.wgrad(dy, act.dequantize(rows_ptr=rows_ptr), cu, g, pads=pads)
            grads[2] = g.to(torch.bfloat16).view(ctx.shapes[1])
        dx = d_scale = None
        if need_x or need_g or need_u or need_s:
            d_act = gemm.down_dgrad(dy, wdq.dequantize().view(G, H, Hp), cu, pads=pads)
            d_gate, d_up, d_scale = ew.swiglu_bwd(d_act, gate, up, row_scale, rows_ptr=rows_ptr, want_dscale=need_s)
            if need_x:
                new = torch.empty if cu is None else torch.zeros
                dx = new(dy.shape, dtype=torch.bfloat16, device=dy.device)
                w = wgu.dequantize()
                gemm.gateup_dgrad(d_gate, d_up, w[0], w[1], cu, out=dx, pads=pads, transposed=True)
            if need_g or need_u:
                xv = xq.dequantize(rows_ptr=rows_ptr)
                out = torch.empty(2, G, H, Hp, **f32)
                gemm.wgrad2(xv, (d_gate, d_up), cu, (out[0], out[1]), pads=pads)
                out = out.to(torch.bfloat16)
                grads[:2] = (out[i].view(ctx.shapes[0]) for i in range(2))
        return dx, grads[0], grads[1], grads[2], d_scale, None, None


def expert_ffn(x: torch.Tensor, wg, wu, wd, cu_seqlens: Optional[torch.Tensor] = None, *,
               row_scale: Optional[torch.Tensor] = None, pads: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[rows,H] = (silu(x Wg[g]) * (x Wu[g]) * row_scale) Wd[g]^T`` over quantised operands, differentiable.

    bf16 ``x`` ``[rows, H]`` and ``wg``/``wu``/``wd`` ``[G, H, H']`` (one expert: ``[H, H']``), which are quantised in the
    call; or weights packed before, ``expert_ffn(x, pack_gate_up(wg, wu), None, quantize(wd), ...)``, which get no
    gradient.  ``x`` is quantised along H, the activation (rounded to bf16) along H'.

    The gradients are those of the formula with the quantised operands in it; the quantisation itself is passed
    straight through: ``d Wg = x^T d_gate`` has the quantised ``x``, ``d x`` the quantised weights.  What forward keeps
    are the operands in 4 bits, gate and up in bf16.  Sums run in fp32; ``d act``, ``d gate`` and ``d up`` are
    rounded to bf16, as operands of the bf16 products of :mod:`.gemm`, and the results once more.

    Rows that belong to no group get zeros, in ``y`` and in ``x``'s gradient.  For gradients H must be a multiple of 128
    and H' of 8, and with ``cu_seqlens`` every group's rows a multiple of 64, of which padding rows of ``x`` are zero
    (what ``Buffer.dispatch`` gives)."""
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
            assert _operand(w, name).dtype == torch.bfloat16, f"{name} must be bf16"
        assert wg.shape == wu.shape == wd.shape and wg.shape[-2] == H, "weights must be [G, H, H'] alike"
        Hp = wg.shape[-1]
    if row_scale is not None:
        assert row_scale.dim() == 1 and row_scale.shape[0] == x.shape[0], "one scale a row"
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, *trained) + (() if row_scale is None else (row_scale,))):
        assert H % 128 == 0 and Hp % 8 == 0, "gradients need H % 128 == 0 and H' % 8 == 0"
    return _ExpertFFN.apply(x, wg, wu, wd, row_scale, cu_seqlens, pads)
