"""Microscaled 4-bit operators against the definition in 64 bits.

Quantised values have to be equal.  A product's result is within half a bf16 step, 2^-8 of its value, and what K sums in
fp32 can lose, K 2^-24 of the sum of magnitudes."""
import threading

import pytest
import torch

from tests import mx_oracle as ox

gpu = pytest.mark.gpu
HALF = 2.0 ** -8


def _gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.fixture(autouse=True)
def _status():
    yield
    if torch.cuda.is_available():
        from moonep_b200.ops import gemm
        torch.cuda.synchronize()
        gemm.check_status()


def _equal(got, want):
    got = got.cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def _spread(gen, *shape):
    """Values of many magnitudes, among them zeros and exact borders between codes."""
    x = torch.randn(*shape, generator=gen) * torch.exp2(torch.randint(-20, 20, shape[:-1] + (1,), generator=gen).float())
    border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 0.0])[torch.randint(0, 10, shape, generator=gen)]
    return torch.where(torch.rand(*shape, generator=gen) < 0.3, border, x)


def test_oracle_values():
    x = torch.tensor([[7.9, 0.25, -0.75, 1.25, 1.75, -2.5, 3.5, 5.0, 0.2, -6.0] + [0.0] * 22])
    want = torch.tensor([[6.0, 0.0, -1.0, 1.0, 2.0, -2.0, 4.0, 4.0, 0.0, -6.0] + [0.0] * 22]).double()
    assert torch.equal(ox.quantise(x), want)
    assert torch.equal(ox.quantise(x * 2.0 ** -30), want * 2.0 ** -30)
    assert ox.quantise(torch.tensor([[1.0, float("inf")]])).isnan().all()


# ---- quantisation ------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (3, 32), (16, 7168), (129, 1003), (2, 65, 40), (5, 130, 264)])
def test_quantise_rows(shape, dtype):
    from moonep_b200.ops import mx
    x = _spread(_gen(1), *shape).clamp(-60000, 60000).to(dtype)
    q = mx.quantize(x.cuda())
    assert q.shape == tuple(shape)
    want = ox.quantise(x)
    _equal(q.dequantize(torch.float32), want)
    _equal(q.dequantize(), want)                      # (no magnitude here is below bf16's subnormals)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (32, 3), (2048, 96), (1003, 129), (2, 40, 65), (3, 264, 130)])
def test_quantise_columns(shape, dtype):
    from moonep_b200.ops import mx
    x = _spread(_gen(2), *shape).clamp(-60000, 60000).to(dtype)
    q = mx.quantize(x.cuda(), axis=-2)
    assert q.shape == (*shape[:-2], shape[-1], shape[-2])
    _equal(q.dequantize(torch.float32), ox.quantise(x.transpose(-1, -2).contiguous()))


@gpu
@pytest.mark.parametrize("axis", [-1, -2])
def test_quantise_strides(axis):
    from moonep_b200.ops import mx
    base = _spread(_gen(3), 4, 70, 200).cuda()
    for x in (base[1:3, 5:69, 8:136], base[:, ::2, 3:166], base[::2, 1:2], base[0, :, 1:]):
        want = ox.quantise(x.cpu() if axis == -1 else x.cpu().transpose(-1, -2).contiguous())
        _equal(mx.quantize(x, axis).dequantize(torch.float32), want)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantise_rows_that_start_anywhere(dtype):
    """Every offset in 16 bytes, lengths around a lane's eight elements and a warp's 256; a neighbour's NaN stays out."""
    from moonep_b200.ops import mx
    base = _spread(_gen(26), 5, 311).clamp(-60000, 60000).to(dtype)
    for length in (1, 7, 8, 9, 23, 33, 257, 300):
        for at in range(1, 10):
            x = base.clone()
            x[:, :at], x[:, at + length:] = float("nan"), float("nan")
            q = mx.quantize(x.cuda()[:, at:at + length])
            want = ox.quantise(base[:, at:at + length].contiguous())
            _equal(q.dequantize(torch.float32), want)
            _equal(q.dequantize(), want)


@gpu
def test_quantise_extremes():
    """Largest, smallest, subnormal and non-finite values; zero blocks; a block that is not full."""
    from moonep_b200.ops import mx
    x = torch.randn(8, 70, generator=_gen(4))
    x[0, :32] = 0.0
    x[1, 3], x[2, 40], x[3, 69] = float("nan"), float("inf"), -float("inf")
    x[4, :32] *= 2.0 ** -126
    x[4, 32:64] = 2.0 ** -149
    x[5] *= 3.0e38 / x[5].abs().max()
    x[6, 0], x[6, 1] = 3.4e38, 2.0 ** -149
    x[7, :] = -0.0
    q = mx.quantize(x.cuda())
    _equal(q.dequantize(torch.float32), ox.quantise(x))
    _equal(mx.quantize(x.t().contiguous().cuda(), axis=-2).dequantize(torch.float32), ox.quantise(x))


@gpu
@pytest.mark.parametrize("dtype,exp", [(torch.bfloat16, -126), (torch.float16, -14)])
def test_quantise_subnormals(dtype, exp):
    """Blocks of numbers below their type's smallest normal one, which is 2^exp."""
    from moonep_b200.ops import mx
    x = (torch.randn(4, 96, generator=_gen(22)) * 2.0 ** (exp + 2)).to(dtype)
    x[1] *= 0.125
    x[2] *= 2.0 ** -4
    want = ox.quantise(x)
    assert float(want[2].abs().max()) > 0
    for q in (mx.quantize(x.cuda()), mx.quantize(x.t().contiguous().cuda(), axis=-2)):
        _equal(q.dequantize(torch.float32), want)
        _equal(q.dequantize(), want.float().bfloat16().double())


@gpu
def test_quantise_row_count_on_the_device():
    from moonep_b200.ops import mx
    x = torch.randn(300, 96, generator=_gen(5)).bfloat16()
    n = torch.tensor([131], dtype=torch.int32).cuda()
    q = mx.quantize(x.cuda(), rows_ptr=n)
    _equal(q.dequantize()[:131], ox.quantise(x[:131]))
    out = mx.quantize(x.cuda()).dequantize(rows_ptr=n)
    _equal(out[:131], ox.quantise(x[:131]))
    for bad in (-5, 0, 1000):
        mx.quantize(x.cuda(), rows_ptr=torch.tensor([bad], dtype=torch.int32).cuda())


@gpu
@pytest.mark.parametrize("shape", [(2, 96, 40), (1, 130, 16), (3, 64, 515), (70, 33)])
def test_pack_gate_up(shape):
    from moonep_b200.ops import mx
    gen = _gen(6)
    wg, wu = (_spread(gen, *shape).bfloat16() for _ in range(2))
    q = mx.pack_gate_up(wg.cuda(), wu.cuda())
    v = q.dequantize(torch.float32)
    three = [w if w.dim() == 3 else w[None] for w in (wg, wu)]
    assert q.shape == (2, three[0].shape[0], shape[-1], shape[-2])
    for i in range(2):
        _equal(v[i], ox.quantise(three[i].transpose(1, 2).contiguous()))


@gpu
def test_pack_gate_up_strides():
    from moonep_b200.ops import mx
    gen = _gen(20)
    both = torch.randn(3, 96, 2 * 50, generator=gen).bfloat16().cuda()
    wg, wu = both[:, :, :50], both[:, :, 50:]
    want = mx.pack_gate_up(wg.contiguous(), wu.contiguous()).dequantize()
    assert torch.equal(mx.pack_gate_up(wg, wu).dequantize(), want)
    assert torch.equal(mx.pack_gate_up(wg, wu.contiguous()).dequantize(), want)


@gpu
def test_empty_operands():
    from moonep_b200.ops import mx
    q = mx.quantize(torch.empty(0, 64, device="cuda", dtype=torch.bfloat16))
    w = mx.quantize(torch.randn(1, 48, 64, device="cuda"))
    assert q.dequantize().shape == (0, 64)
    assert mx.matmul(q, w, torch.zeros(1, dtype=torch.int32, device="cuda")).shape == (0, 48)
    some = mx.quantize(torch.randn(5, 64, device="cuda"))
    out = torch.full((5, 48), 7.0, device="cuda", dtype=torch.bfloat16)
    mx.matmul(some, w, torch.zeros(1, dtype=torch.int32, device="cuda"), out=out)
    assert (out == 7).all()


# ---- products ----------------------------------------------------------------------------------
GROUPS = [[5], [1, 0, 2], [128, 256, 0, 128], [100, 0, 300, 1, 129, 64], [225, 31, 33, 7], [448, 449, 1000]]


def _ends(sizes):
    return torch.tensor(sizes).cumsum(0).to(torch.int32)


def _product_case(sizes, N, K, seed):
    gen = _gen(seed)
    rows = sum(sizes)
    a, w = torch.randn(rows, K, generator=gen).bfloat16(), (torch.randn(len(sizes), N, K, generator=gen) * K ** -0.5).bfloat16()
    return a, w, ox.quantise(a), ox.quantise(w)


@gpu
@pytest.mark.parametrize("N,K", [(256, 256), (8, 32), (515, 1000), (640, 2048), (1, 1)])
@pytest.mark.parametrize("sizes", GROUPS)
def test_product(sizes, N, K):
    from moonep_b200.ops import mx
    a, w, av, wv = _product_case(sizes, N, K, 7)
    ends = _ends(sizes)
    y = mx.matmul(mx.quantize(a.cuda()), mx.quantize(w.cuda()), ends.cuda()).cpu().double()
    ref, mag = ox.product(av, wv, ends.tolist())
    err = (y - ref).abs() - HALF * ref.abs() - (K + 2) * 2.0 ** -24 * mag
    assert float(err.max()) <= 0, f"{float((y - ref).abs().max())} off, {int((err > 0).sum())} of {err.numel()}"


@gpu
def test_product_far_from_one():
    """Scales at both ends of what E8M0 holds, and a NaN block: its rows and columns are NaN, the others are not."""
    from moonep_b200.ops import mx
    gen = _gen(8)
    a, w = torch.randn(70, 96, generator=gen), torch.randn(1, 40, 96, generator=gen)
    a[3] *= 2.0 ** 60
    a[4] *= 2.0 ** -110
    w[0, 5] *= 2.0 ** -60
    a[7, 95], w[0, 9, 0] = float("nan"), float("inf")
    y = mx.matmul(mx.quantize(a.cuda()), mx.quantize(w.cuda()), _ends([70]).cuda()).cpu().double()
    ref, mag = ox.product(ox.quantise(a), ox.quantise(w), [70])
    assert torch.equal(y.isnan(), ref.isnan())
    # (row 4 times column 5 is of the size of 2^-170: bf16's smallest step is 2^-133, half of it rounding's at any size)
    err = (y - ref).abs() - HALF * ref.abs() - 98 * 2.0 ** -24 * mag - 2.0 ** -134
    assert float(err.nan_to_num(-1).max()) <= 0


@gpu
def test_product_leaves_other_rows():
    """Rows in front of, between and behind the groups' tiles: only the groups' rows are written, padding becomes zero."""
    from moonep_b200.ops import mx
    sizes, K, N = [37, 128, 0, 90], 320, 200
    a, w, av, wv = _product_case(sizes, N, K, 9)
    ends = _ends(sizes)
    pads = torch.tensor([[20, 17], [165, 0], [165, 0], [200, 55]], dtype=torch.int32)
    out = torch.full((sum(sizes) + 50, N + 24), 7.0).bfloat16().cuda()
    more = torch.cat([a, torch.full((30, K), float("nan"))]).cuda()
    y = mx.matmul(mx.quantize(more), mx.quantize(w.cuda()), ends.cuda(), out=out[:-20, 8:8 + N], pads=pads.cuda())
    assert y.data_ptr() == out[0, 8:].data_ptr()
    ref, _ = ox.product(av, wv, ends.tolist())
    ref[20:37], ref[200:255] = 0, 0
    got = out.cpu().double()
    assert float((got[:255, 8:8 + N] - ref).abs().max()) < 0.05
    assert (got[20:37, 8:8 + N] == 0).all() and (got[200:255, 8:8 + N] == 0).all()
    got[:255, 8:8 + N] = 7.0
    assert (got == 7.0).all()
    mx.matmul(mx.quantize(more), mx.quantize(w.cuda()), ends.cuda(), out=out[:-20, 8:8 + N], zero_tail=True)
    assert (out[255:-20, 8:8 + N] == 0).all() and (out[-20:] == 7).all() and (out[:, :8] == 7).all() and (out[:, 8 + N:] == 7).all()
    mx.matmul(mx.quantize(more), mx.quantize(w.cuda()), torch.zeros_like(ends).cuda(), out=out[:-20, 8:8 + N], zero_tail=True)
    assert (out[:-20, 8:8 + N] == 0).all() and (out[-20:] == 7).all()


@gpu
def test_product_of_one_matrix():
    """Without groups; the same numbers as one group, and on another stream."""
    from moonep_b200.ops import mx
    a, w, av, wv = _product_case([777], 384, 512, 10)
    ref, mag = ox.product(av, wv, [777])
    qa, qw = mx.quantize(a.cuda()), mx.quantize(w[0].cuda())
    y = mx.matmul(qa, qw)
    assert float(((y.cpu().double() - ref).abs() - HALF * ref.abs() - 514 * 2.0 ** -24 * mag).max()) <= 0
    assert torch.equal(y, mx.matmul(qa, mx.quantize(w.cuda()), _ends([777]).cuda()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = mx.matmul(mx.quantize(a.cuda()), qw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, z)


# ---- gate and up -------------------------------------------------------------------------------
def _gated_ref(xv, gv, uv, ends, scale):
    """act, gate, up and how far act may be off: fp32 sums, exp to 2^-16 (|x| steps), half a bf16 step."""
    K = xv.shape[1]
    gate, gm = ox.product(xv, gv, ends)
    up, um = ox.product(xv, uv, ends)
    sig = torch.sigmoid(gate)
    act = gate * sig * up * scale[:, None]
    dg, du = (K + 2) * 2.0 ** -24 * gm, (K + 2) * 2.0 ** -24 * um
    off = ((1.1 * dg * up.abs()) + (gate * sig).abs() * du + 1.1 * dg * du) * scale[:, None].abs()
    return act, gate, up, dg, du, off + act.abs() * (HALF + 1e-5 * (1 + gate.abs()))


@gpu
@pytest.mark.parametrize("H,Hp", [(256, 256), (64, 8), (1000, 515), (2048, 640), (32, 1)])
@pytest.mark.parametrize("sizes", GROUPS)
def test_gateup_swiglu(sizes, H, Hp):
    from moonep_b200.ops import mx
    gen = _gen(11)
    rows, G = sum(sizes), len(sizes)
    x = torch.randn(rows, H, generator=gen).bfloat16()
    wg, wu = ((torch.randn(G, H, Hp, generator=gen) * 2 * H ** -0.5).bfloat16() for _ in range(2))
    scale = torch.rand(rows, generator=gen) + 0.1
    ends = _ends(sizes)
    gv, uv = (ox.quantise(w.transpose(1, 2).contiguous()) for w in (wg, wu))
    act_ref, gate_ref, up_ref, dg, du, off = _gated_ref(ox.quantise(x), gv, uv, ends.tolist(), scale.double())
    xq, w = mx.quantize(x.cuda()), mx.pack_gate_up(wg.cuda(), wu.cuda())
    act, gate, up = mx.gateup_swiglu(xq, w, ends.cuda(), row_scale=scale.cuda(), save_gate_up=True)
    for got, ref, tol in ((act, act_ref, off), (gate, gate_ref, HALF * gate_ref.abs() + dg), (up, up_ref, HALF * up_ref.abs() + du)):
        assert float(((got.cpu().double() - ref).abs() - tol).max()) <= 1e-30
    alone, none, _ = mx.gateup_swiglu(xq, w, ends.cuda(), row_scale=scale.cuda())
    assert none is None and torch.equal(alone, act)
    want = mx.quantize(act).dequantize()
    for save in (False, True):
        q, g2, _ = mx.gateup_swiglu(xq, w, ends.cuda(), row_scale=scale.cuda(), quantize=True, save_gate_up=save)
        assert torch.equal(q.dequantize(), want) and (not save or torch.equal(g2, gate))
        # as an operand it is what quantising the activation gives
        wd = mx.quantize(torch.randn(G, 72, Hp, generator=gen).cuda())
        assert torch.equal(mx.matmul(q, wd, ends.cuda()), mx.matmul(mx.quantize(act), wd, ends.cuda()))


@gpu
def test_gateup_padding_rows():
    from moonep_b200.ops import mx
    gen = _gen(12)
    H, Hp, ends = 256, 160, _ends([128, 64, 192])
    pads = torch.tensor([[100, 28], [128, 64], [192, 0]], dtype=torch.int32)
    x = torch.randn(384, H, generator=gen).bfloat16()
    x[100:128], x[129:192] = 0, 0
    pads[1] = torch.tensor([129, 63])
    wg, wu = ((torch.randn(3, H, Hp, generator=gen) * H ** -0.5).bfloat16().cuda() for _ in range(2))
    xq, w = mx.quantize(x.cuda()), mx.pack_gate_up(wg, wu)
    plain = mx.gateup_swiglu(xq, w, ends.cuda(), save_gate_up=True)
    padded = mx.gateup_swiglu(xq, w, ends.cuda(), save_gate_up=True, pads=pads.cuda())
    for a, b in zip(plain, padded):
        assert torch.equal(a, b)
    q = mx.gateup_swiglu(xq, w, ends.cuda(), quantize=True, pads=pads.cuda())[0]
    assert torch.equal(q.dequantize(), mx.quantize(plain[0]).dequantize())


@gpu
@pytest.mark.parametrize("H,Hp", [(256, 256), (64, 8), (1000, 515), (2048, 640)])
@pytest.mark.parametrize("sizes", GROUPS)
def test_gateup_swiglu_backward(sizes, H, Hp):
    """d gate, d up and d scale against the formulas on the quantised operands in 64 bits.  Gate and up are fp32 sums, off
    by dg and du; the formulas' slopes in them are at most 1.1 and 0.5 (silu and its derivative)."""
    from moonep_b200.ops import mx
    gen = _gen(17)
    rows, G = sum(sizes), len(sizes)
    x = torch.randn(rows, H, generator=gen).bfloat16()
    wg, wu = ((torch.randn(G, H, Hp, generator=gen) * 2 * H ** -0.5).bfloat16() for _ in range(2))
    scale, d_act = torch.rand(rows, generator=gen) + 0.1, torch.randn(rows, Hp, generator=gen)
    ends = _ends(sizes)
    gv, uv = (ox.quantise(w.transpose(1, 2).contiguous()) for w in (wg, wu))
    _, gate, up, dg, du, _ = _gated_ref(ox.quantise(x), gv, uv, ends.tolist(), scale.double())
    sig = torch.sigmoid(gate)
    d = d_act.double()
    want_s = d * gate * sig * up
    ds = d * scale.double()[:, None]
    want_g, want_u = ds * up * sig * (1 + gate * (1 - sig)), ds * gate * sig
    slack = 1e-5 * (1 + gate.abs())              # exp, and a few fp32 steps
    off_g = ds.abs() * (1.1 * du + 0.5 * up.abs() * dg + 0.5 * du * dg + up.abs() * 1.1 * slack)
    off_u = ds.abs() * (1.1 * dg + slack * gate.abs())
    off_s = (d.abs() * (1.1 * dg * up.abs() + (gate * sig).abs() * du + 1.1 * dg * du)).sum(1) \
        + (want_s.abs() * (slack + Hp * 2.0 ** -24)).sum(1)
    xq, w = mx.quantize(x.cuda()), mx.pack_gate_up(wg.cuda(), wu.cuda())
    got = mx.gateup_swiglu_bwd(d_act.cuda(), xq, w, ends.cuda(), row_scale=scale.cuda(), want_dscale=True)
    for y, ref, tol in zip(got, (want_g, want_u, want_s.sum(1)), (HALF * want_g.abs() + off_g, HALF * want_u.abs() + off_u, off_s)):
        assert float(((y.cpu().double() - ref).abs() - tol).max()) <= 1e-30
    again = mx.gateup_swiglu_bwd(d_act.cuda(), xq, w, ends.cuda(), row_scale=scale.cuda())
    assert again[2] is None and torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])


@gpu
def test_gateup_backward_padding_rows():
    from moonep_b200.ops import mx
    gen = _gen(18)
    H, Hp, ends = 256, 160, _ends([128, 64, 192]).cuda()
    pads = torch.tensor([[100, 28], [129, 63], [192, 0]], dtype=torch.int32).cuda()
    x = torch.randn(384 + 30, H, generator=gen).bfloat16()
    x[100:128], x[129:192] = 0, 0
    d_act = torch.randn(384 + 30, Hp, generator=gen).cuda()
    bad = d_act.clone()
    bad[100:128], bad[129:192], bad[384:] = float("nan"), float("nan"), float("nan")
    wg, wu = ((torch.randn(3, H, Hp, generator=gen) * H ** -0.5).bfloat16().cuda() for _ in range(2))
    xq, w = mx.quantize(x.cuda()), mx.pack_gate_up(wg, wu)
    plain = mx.gateup_swiglu_bwd(d_act, xq, w, ends, want_dscale=True)
    padded = mx.gateup_swiglu_bwd(bad, xq, w, ends, want_dscale=True, pads=pads)
    for a, b in zip(plain, padded):
        assert torch.equal(a[:384], b[:384])
    assert (padded[2][384:] == 0).all()


@gpu
@pytest.mark.parametrize("H,Hp", [(256, 256), (64, 8), (1000, 515), (2048, 640), (8, 1)])
@pytest.mark.parametrize("sizes", GROUPS)
def test_dgrads(sizes, H, Hp):
    """bf16 rows times the values of quantised weights, along their scales: K sums in fp32, in bf16 half a step more."""
    from moonep_b200.ops import mx
    gen = _gen(23)
    rows, G = sum(sizes), len(sizes)
    ends = _ends(sizes)
    dy = torch.randn(rows, H, generator=gen).bfloat16()
    wd = _spread(gen, G, H, Hp).bfloat16() if H < 1000 else torch.randn(G, H, Hp, generator=gen).bfloat16()
    q = mx.quantize(wd.cuda())
    ref, mag = ox.product(dy.double(), ox.quantise(wd).transpose(1, 2), ends.tolist())
    slack = (H + 2) * 2.0 ** -24 * mag
    got = mx.down_dgrad(dy.cuda(), q, ends.cuda(), fp32=True)
    assert got.dtype == torch.float32 and float(((got.cpu().double() - ref).abs() - slack).max()) <= 0
    got = mx.down_dgrad(dy.cuda(), q, ends.cuda())
    assert float(((got.cpu().double() - ref).abs() - slack - HALF * ref.abs()).max()) <= 0
    if Hp % 8:
        return
    wg, wu = (torch.randn(G, H, Hp, generator=gen).bfloat16() for _ in range(2))
    dg, du = (torch.randn(rows, Hp, generator=gen).bfloat16() for _ in range(2))
    gv, uv = (ox.quantise(w.transpose(1, 2).contiguous()) for w in (wg, wu))        # [G, H', H]
    got = mx.gateup_dgrad(dg.cuda(), du.cuda(), mx.pack_gate_up(wg.cuda(), wu.cuda()), ends.cuda())
    (a, am), (b, bm) = (ox.product(d.double(), v.transpose(1, 2), ends.tolist()) for d, v in ((dg, gv), (du, uv)))
    assert float(((got.cpu().double() - a - b).abs() - (2 * Hp + 2) * 2.0 ** -24 * (am + bm) - HALF * (a + b).abs()).max()) <= 0


@gpu
def test_dgrad_over_all_scales():
    """One weight row a token, one scale a weight row, from E8M0's smallest to fp32's largest: the sums are the stored values."""
    from moonep_b200.ops import mx
    gen = _gen(25)
    scale = 2.0 ** torch.arange(-130, 126, dtype=torch.float64)
    w = ((torch.randn(256, 72, generator=gen, dtype=torch.float64).clamp(-1.9, 1.9) * scale[:, None]).float())[None]
    q = mx.quantize(w.cuda())
    y = mx.down_dgrad(torch.eye(256).bfloat16().cuda(), q, fp32=True)
    want = ox.quantise(w)[0]
    assert torch.equal(q.dequantize(torch.float32)[0].cpu().double(), want) and torch.equal(y.cpu().double(), want)


@gpu
def test_dgrad_padding_and_other_rows():
    from moonep_b200.ops import mx
    gen = _gen(24)
    H, Hp, ends = 256, 160, _ends([128, 64, 0, 192]).cuda()
    pads = torch.tensor([[100, 28], [129, 63], [192, 0], [192, 0]], dtype=torch.int32).cuda()
    dg, du = (torch.randn(384 + 40, Hp, generator=gen).bfloat16().cuda() for _ in range(2))
    w = mx.pack_gate_up(*((torch.randn(4, H, Hp, generator=gen) * H ** -0.5).bfloat16().cuda() for _ in range(2)))
    plain = mx.gateup_dgrad(dg, du, w, ends)
    assert (plain[384:] == 0).all() and float(plain[:384].float().abs().min(1).values.max()) > 0
    for d in (dg, du):
        d[100:128], d[129:192] = 0, 0
    want = mx.gateup_dgrad(dg, du, w, ends)
    for d in (dg, du):
        d[100:128], d[160:192], d[384:] = 0, float("nan"), float("nan")     # (a tile's own 32 rows are read)
    out = torch.full((430, H), 7.0, device="cuda", dtype=torch.bfloat16)
    got = mx.gateup_dgrad(dg, du, w, ends, pads=pads, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(out[:424], want) and (out[424:] == 7).all()
    # a NaN block of the weights reaches its columns' rows only
    wd = torch.randn(2, 64, 96, generator=gen)
    wd[1, 5, 40] = float("nan")
    y = mx.down_dgrad(dg[:100, :64].contiguous(), mx.quantize(wd.cuda()), _ends([50, 50]).cuda())
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[50:, 32:64] = True
    assert torch.equal(y.isnan(), bad)


@gpu
@pytest.mark.parametrize("G,H,Hp", [(3, 256, 72), (2, 384, 256), (1, 128, 8)])
def test_weight_grads_in_bf16(G, H, Hp):
    """The fp32 grads rounded; those of empty groups zero."""
    from moonep_b200.ops import gemm
    gen = _gen(19)
    sizes = [64, 0, 192][:G] if G > 1 else [100]
    rows = sum(sizes)
    a = torch.randn(rows, H, generator=gen).bfloat16().cuda()
    cu = None if G == 1 else _ends(sizes).cuda()
    d1, d2 = (torch.randn(rows, Hp, generator=gen).bfloat16().cuda() for _ in range(2))
    f32 = [torch.empty(G, H, Hp, device="cuda") for _ in range(3)]
    b16 = [torch.full((G, H, Hp), 7.0, device="cuda", dtype=torch.bfloat16) for _ in range(3)]
    for out in (f32, b16):
        gemm.wgrad(a, d1, cu, out[0])
        gemm.wgrad2(a, (d1, d2), cu, (out[1], out[2]))
    for x, y in zip(f32, b16):
        assert torch.equal(x.bfloat16(), y)


# ---- the FFN -----------------------------------------------------------------------------------
def _ffn_ref(x, wg, wu, wd, ends, scale, dy=None):
    """y, and with dy the gradients of x, wg, wu, wd, scale, by the formulas.  (The activation is rounded to bf16, then
    quantised: act is given as the kernel's where a rounding may fall to either side.)"""
    xv = ox.quantise(x)
    gv, uv, dv = ox.quantise(wg.transpose(1, 2).contiguous()), ox.quantise(wu.transpose(1, 2).contiguous()), ox.quantise(wd)
    gate, up = ox.product(xv, gv, ends)[0], ox.product(xv, uv, ends)[0]
    sig = torch.sigmoid(gate)
    act = ox.quantise((gate * sig * up * scale[:, None]).bfloat16())
    y = ox.product(act, dv, ends)[0]
    if dy is None:
        return y
    dy = dy.double()
    d_act = ox.product(dy, dv.transpose(1, 2), ends)[0]
    d_scale = (d_act * gate * sig * up).sum(1)
    d_act = d_act * scale[:, None]
    dg, du = d_act * up * sig * (1 + gate * (1 - sig)), d_act * gate * sig
    dx = ox.product(dg, gv.transpose(1, 2), ends)[0] + ox.product(du, uv.transpose(1, 2), ends)[0]
    dw = [torch.zeros(wg.shape, dtype=torch.float64) for _ in range(3)]
    for g, s, e in ox.groups(ends):
        dw[0][g], dw[1][g], dw[2][g] = xv[s:e].T @ dg[s:e], xv[s:e].T @ du[s:e], dy[s:e].T @ act[s:e]
    return y, dx, dw[0], dw[1], dw[2], d_scale


def _near(got, ref, tol):
    """2-norm of the difference over that of the result."""
    d = float((got.cpu().double() - ref).norm() / ref.norm().clamp_min(1e-30))
    assert d <= tol, d


# Independent roundings to bf16 are off by 2^-9 / sqrt(3) of a value in the mean square, at most 2^-8.  y has one; an
# activation near a border may be quantised to either side (relative difference of the sums 2^-20, borders some 0.3
# apart: one in 10^5, by a third of its value: 2^-10 in the norm).  A gradient of x passes the roundings of
# d act, gate / up, d gate / d up, the bf16 weights exactly, and its own: four.  (Now d act, gate and up are not rounded.)
Y_TOL, GRAD_TOL = 2 * HALF, 4 * HALF


@gpu
@pytest.mark.parametrize("sizes,H,Hp,scaled", [([777], 256, 72, False), ([64, 0, 192, 320], 384, 200, True), ([1], 128, 8, True),
                                               ([128], 1024, 512, False)])
def test_expert_ffn_gradients(sizes, H, Hp, scaled):
    from moonep_b200.ops import mx
    gen = _gen(13)
    rows, G = sum(sizes), len(sizes)
    x = torch.randn(rows, H, generator=gen).bfloat16()
    wg, wu, wd = ((torch.randn(G, H, Hp, generator=gen) * s).bfloat16() for s in (H ** -0.5, H ** -0.5, Hp ** -0.5))
    scale = torch.rand(rows, generator=gen) + 0.1 if scaled else torch.ones(rows)
    dy = (torch.randn(rows, H, generator=gen) * 0.01).bfloat16()
    ends = _ends(sizes)
    ref = _ffn_ref(x, wg, wu, wd, ends.tolist(), scale.double(), dy)
    one = G == 1
    leaves = [t.cuda().requires_grad_(True) for t in (x, *((w[0] if one else w) for w in (wg, wu, wd)))]
    s = scale.cuda().requires_grad_(True) if scaled else None
    y = mx.expert_ffn(*leaves, None if one else ends.cuda(), row_scale=s)
    _near(y, ref[0], Y_TOL)
    grads = torch.autograd.grad(y, leaves + ([s] if scaled else []), dy.cuda())
    for got, want in zip(grads, ref[1:]):
        assert got.shape == (want[0] if one and want.dim() == 3 else want).shape
        _near(got, want[0] if one and want.dim() == 3 else want, GRAD_TOL)


@gpu
def test_expert_ffn_gradient_against_differences():
    """Along a direction of the (already quantised) weights of the down projection, in which y is linear, and of the
    scale, in which it is too while no activation's code changes (powers of two)."""
    from moonep_b200.ops import mx
    gen = _gen(14)
    rows, H, Hp = 192, 256, 128
    x = torch.randn(rows, H, generator=gen).bfloat16().cuda()
    wg, wu = ((torch.randn(H, Hp, generator=gen) * H ** -0.5).bfloat16().cuda() for _ in range(2))
    dy = torch.randn(rows, H, generator=gen).bfloat16().cuda()
    wd = mx.quantize(torch.randn(H, Hp, generator=gen).cuda()).dequantize().requires_grad_(True)
    y = mx.expert_ffn(x, wg, wu, wd)
    g, = torch.autograd.grad(y, wd, dy)
    # twice the weights of every second output column: still values of the format
    v = torch.zeros_like(wd)
    v[::2] = wd.detach()[::2]
    diff = ((mx.expert_ffn(x, wg, wu, wd.detach() + v).double() - y.double()) * dy.double()).sum()
    along = (g.double() * v.double()).sum()
    # both sums have terms of either sign: compared with their sizes' sum over sqrt of their number
    size = ((y.double() * dy.double()) ** 2).sum().sqrt() + ((g.double() * v.double()) ** 2).sum().sqrt()
    assert float((diff - along).abs()) <= 8 * HALF * float(size), (float(diff), float(along))
    scale = torch.ones(rows, device="cuda", requires_grad=True)
    y = mx.expert_ffn(x, wg, wu, wd.detach(), row_scale=scale)
    g, = torch.autograd.grad(y, scale, dy)
    two = mx.expert_ffn(x, wg, wu, wd.detach(), row_scale=torch.full_like(scale, 2.0).detach())
    assert torch.equal(two, y.detach() * 2)          # y's slope along its scale is y itself ...
    d = ((two.double() - y.double()) * dy.double()).sum(1)
    # ... of the quantised activation; the straight-through gradient has the activation before, off by an eighth at most
    # of each value (half a step of 1 in [4, 6), of 0.5 in [2, 4); less in the mean), over sqrt(H') independent terms
    assert float((d - g.double()).norm() / d.norm()) < 0.25


@gpu
def test_expert_ffn_packed_weights():
    from moonep_b200.ops import mx
    gen = _gen(15)
    sizes, H, Hp = [64, 128, 0], 256, 96
    ends = _ends(sizes).cuda()
    x = torch.randn(192 + 40, H, generator=gen).bfloat16().cuda()
    wg, wu, wd = ((torch.randn(3, H, Hp, generator=gen) * 0.1).bfloat16().cuda() for _ in range(3))
    dy = torch.randn(232, H, generator=gen).bfloat16().cuda()
    xs = [x.clone().requires_grad_(True) for _ in range(2)]
    ys = [mx.expert_ffn(xs[0], wg, wu, wd, ends), mx.expert_ffn(xs[1], mx.pack_gate_up(wg, wu), None, mx.quantize(wd), ends)]
    gs = [torch.autograd.grad(y, v, dy)[0] for y, v in zip(ys, xs)]
    assert torch.equal(ys[0], ys[1]) and torch.equal(gs[0], gs[1])
    assert (ys[0][192:] == 0).all() and (gs[0][192:] == 0).all()      # rows of no group
    assert float(gs[0][:192].float().abs().sum()) > 0


@gpu
def test_expert_ffn_group_that_weight_grads_cannot_take():
    from moonep_b200.ops import gemm, mx
    bf = dict(device="cuda", dtype=torch.bfloat16)
    x, w = torch.randn(256, 128, **bf), [torch.randn(2, 128, 64, **bf).requires_grad_(True) for _ in range(3)]
    ends = lambda *e: torch.tensor(e, dtype=torch.int32, device="cuda")
    mx.expert_ffn(x, *w, ends(64, 256))
    mx.expert_ffn(x, *w, ends(128, 256))
    gemm.check_status()
    mx.expert_ffn(x, *(t.detach() for t in w), ends(100, 200))      # no weight grads: rows may end anywhere
    gemm.check_status()
    for bad, rows in ((ends(100, 256), 100), (ends(64, 200), 136)):
        mx.expert_ffn(x, *w, bad)
        with pytest.raises(RuntimeError, match=f"{rows} rows"):
            gemm.check_status()
        gemm.reset_status()


@gpu
def test_expert_ffn_some_gradients_only():
    """Each gradient alone is the one of them all; a leaf used twice gets both; rows broadcast from one."""
    from moonep_b200.ops import mx
    gen = _gen(21)
    H, Hp, rows = 128, 64, 96
    x = torch.randn(rows, H, generator=gen).bfloat16().cuda()
    ws = [(torch.randn(H, Hp, generator=gen) * 0.2).bfloat16().cuda() for _ in range(3)]
    scale, dy = torch.rand(rows, generator=gen).cuda() + 0.5, torch.randn(rows, H, generator=gen).bfloat16().cuda()
    leaves = [t.clone().requires_grad_(True) for t in (x, *ws, scale)]
    every = torch.autograd.grad(mx.expert_ffn(*leaves[:4], row_scale=leaves[4]), leaves, dy)
    for i in range(5):
        some = [t.clone().requires_grad_(i == j) for j, t in enumerate((x, *ws, scale))]
        one, = torch.autograd.grad(mx.expert_ffn(*some[:4], row_scale=some[4]), some[i], dy)
        assert torch.equal(one, every[i])
    tied = ws[0].clone().requires_grad_(True)
    g, = torch.autograd.grad(mx.expert_ffn(x, tied, tied, ws[2]), tied, dy)
    a, b = ws[0].clone().requires_grad_(True), ws[0].clone().requires_grad_(True)
    ga, gb = torch.autograd.grad(mx.expert_ffn(x, a, b, ws[2]), (a, b), dy)
    assert torch.equal(g, ga + gb)
    one = x[:1].clone().requires_grad_(True)
    g, = torch.autograd.grad(mx.expert_ffn(one.expand(rows, H), *ws).sum(), one)
    full = x[:1].repeat(rows, 1).requires_grad_(True)
    gf, = torch.autograd.grad(mx.expert_ffn(full, *ws), full, torch.ones(rows, H, device="cuda", dtype=torch.bfloat16))
    _near(g, gf.double().cpu().sum(0, keepdim=True), 2 * HALF)


@gpu
def test_expert_ffn_of_no_rows():
    from moonep_b200.ops import mx
    bf = dict(device="cuda", dtype=torch.bfloat16)
    x, w = torch.empty(0, 128, **bf).requires_grad_(True), [torch.randn(2, 128, 64, **bf).requires_grad_(True) for _ in range(3)]
    s = torch.empty(0, device="cuda").requires_grad_(True)
    y = mx.expert_ffn(x, *w, torch.zeros(2, dtype=torch.int32, device="cuda"), row_scale=s)
    grads = torch.autograd.grad(y, (x, *w, s), torch.empty(0, 128, **bf))
    assert y.shape == (0, 128) and [g.shape for g in grads] == [t.shape for t in (x, *w, s)]
    assert all((g == 0).all() for g in grads)
    # rows, but no group has any
    x = torch.randn(64, 128, **bf).requires_grad_(True)
    y = mx.expert_ffn(x, *w, torch.zeros(2, dtype=torch.int32, device="cuda"))
    grads = torch.autograd.grad(y, (x, *w), torch.ones(64, 128, **bf))
    assert (y == 0).all() and all((g == 0).all() for g in grads)


@gpu
def test_expert_ffn_saved_operands():
    """They go through hooks, are kept for a second backward pass on request and freed without."""
    from moonep_b200.ops import mx
    gen = _gen(25)
    H, Hp, rows = 256, 128, 192
    x, dy = (torch.randn(rows, H, generator=gen).bfloat16().cuda() for _ in range(2))
    ws = [(torch.randn(H, Hp, generator=gen) * 0.1).bfloat16().cuda().requires_grad_(True) for _ in range(3)]
    want = torch.autograd.grad(mx.expert_ffn(x, *ws), ws, dy)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        y = mx.expert_ffn(x, *ws)
    for a, b in zip(torch.autograd.grad(y, ws, dy), want):
        assert torch.equal(a, b)
    y = mx.expert_ffn(x, *ws)
    for keep in (True, False):
        for a, b in zip(torch.autograd.grad(y, ws, dy, retain_graph=keep), want):
            assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, ws, dy)
    frozen = mx.pack_gate_up(*ws[:2])
    frozen = mx.MxTensor(frozen.codes.clone(), frozen.scales.clone(), frozen.shape), None, mx.quantize(ws[2])
    xs = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(mx.expert_ffn(xs, *frozen), xs, dy)
    assert torch.equal(g, torch.autograd.grad(mx.expert_ffn(xs, *ws), xs, dy)[0])


@gpu
def test_expert_ffn_captured():
    """One token, and a training step, captured and replayed on new inputs."""
    from moonep_b200.ops import mx
    from moonep_b200.utils.graph import GraphedStep
    gen = _gen(16)
    H, Hp = 256, 128
    wg, wu, wd = ((torch.randn(4, H, Hp, generator=gen) * 0.1).bfloat16().cuda() for _ in range(3))
    packed = mx.pack_gate_up(wg, wu), None, mx.quantize(wd)

    def serve(x, ends):
        with torch.no_grad():
            return mx.expert_ffn(x, *packed, ends)

    def train(x, ends, dy):
        leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu, wd)]
        y = mx.expert_ffn(*leaves, ends)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    new = lambda rows: torch.randn(rows, H, generator=gen).bfloat16().cuda()
    e1 = [torch.tensor(e, dtype=torch.int32, device="cuda") for e in ([0, 0, 1, 1], [1, 1, 1, 1])]
    step = GraphedStep(serve, [new(1), e1[0]])
    for e in e1:
        x = new(1)
        assert torch.equal(step(x, e), serve(x, e))
    e2 = [torch.tensor(e, dtype=torch.int32, device="cuda") for e in ([64, 64, 192, 256], [0, 128, 192, 256])]
    step = GraphedStep(train, [new(256), e2[0], new(256)])
    for e in e2:
        x, dy = new(256), new(256)
        for a, b in zip(step(x, e, dy), train(x, e, dy)):
            assert torch.equal(a, b)


# ---- refusals ----------------------------------------------------------------------------------
@gpu
def test_refusals():
    from moonep_b200.ops import mx
    bf = dict(device="cuda", dtype=torch.bfloat16)
    x, w = torch.randn(8, 64, **bf), torch.randn(2, 32, 64, **bf)
    q, qw, ends = mx.quantize(x), mx.quantize(w), torch.tensor([4, 8], dtype=torch.int32, device="cuda")
    gu = mx.pack_gate_up(torch.randn(2, 64, 32, **bf), torch.randn(2, 64, 32, **bf))
    n = torch.tensor([3], dtype=torch.int32, device="cuda")
    bad = [
        lambda: mx.quantize(x.cpu()),
        lambda: mx.quantize(x.double()),
        lambda: mx.quantize(x.t()),
        lambda: mx.quantize(x[0]),
        lambda: mx.quantize(x, axis=0),
        lambda: mx.quantize(x[:, :0]),
        lambda: mx.quantize(x[:0], axis=-2),
        lambda: mx.quantize(w, rows_ptr=n),
        lambda: mx.quantize(x, rows_ptr=n.long()),
        lambda: mx.pack_gate_up(w, w[:, :, :32]),
        lambda: mx.pack_gate_up(w, w.float()),
        lambda: qw.dequantize(torch.float16),
        lambda: mx.MxTensor(q.codes, q.scales[:1].contiguous(), q.shape),
        lambda: mx.MxTensor(q.codes, q.scales, (8, 96)),
        lambda: mx.matmul(x, qw, ends),
        lambda: mx.matmul(q, qw),
        lambda: mx.matmul(q, qw, ends.long()),
        lambda: mx.matmul(q, qw, ends[:1]),
        lambda: mx.matmul(q, qw, ends.cpu()),
        lambda: mx.matmul(q, gu, ends),
        lambda: mx.matmul(qw, qw, ends),
        lambda: mx.matmul(q, mx.quantize(torch.randn(2, 32, 96, **bf)), ends),
        lambda: mx.matmul(q, qw, ends, out=torch.empty(8, 31, **bf)),
        lambda: mx.matmul(q, qw, ends, out=torch.empty(7, 32, **bf)),
        lambda: mx.matmul(q, qw, ends, out=torch.empty(8, 32, device="cuda")),
        lambda: mx.matmul(q, qw, ends, out=torch.empty(1, 32, **bf).expand(8, 32)),
        lambda: mx.matmul(q, qw, ends, pads=torch.zeros(1, 2, dtype=torch.int32, device="cuda")),
        lambda: mx.gateup_swiglu(q, qw, ends),
        lambda: mx.gateup_swiglu(q, gu, ends, row_scale=torch.ones(7, device="cuda")),
        lambda: mx.gateup_swiglu(q, gu, ends, row_scale=torch.ones(8, **bf)),
        lambda: mx.down_dgrad(x, gu, ends),
        lambda: mx.down_dgrad(x.float(), mx.quantize(torch.randn(2, 64, 32, **bf)), ends),
        lambda: mx.down_dgrad(x[:, :32].contiguous(), mx.quantize(torch.randn(2, 64, 32, **bf)), ends),
        lambda: mx.down_dgrad(x, mx.quantize(torch.randn(2, 64, 32, **bf))),
        lambda: mx.gateup_dgrad(x[:, :32].contiguous(), x[:4, :32].contiguous(), gu, ends),
        lambda: mx.gateup_dgrad(x, x, gu, ends),
        lambda: mx.gateup_dgrad(x, x, qw, ends),
        lambda: mx.gateup_swiglu_bwd(torch.zeros(8, 32, **bf), q, gu, ends),
        lambda: mx.gateup_swiglu_bwd(torch.zeros(7, 32, device="cuda"), q, gu, ends),
        lambda: mx.gateup_swiglu_bwd(torch.zeros(8, 32, device="cuda"), q, qw, ends),
        lambda: mx.expert_ffn(x.float(), w, w, w, ends),
        lambda: mx.expert_ffn(x, w, w, w, ends),
        lambda: mx.expert_ffn(x, gu, w, qw, ends),
        lambda: mx.expert_ffn(x, gu, None, qw, ends),
        lambda: mx.expert_ffn(x.requires_grad_(True), *(torch.randn(2, 64, 32, **bf) for _ in range(3)), ends),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(AssertionError):
            call()
            pytest.fail(f"call {i} was not refused")


def test_refusals_without_a_gpu():
    from moonep_b200.ops import mx
    with pytest.raises(AssertionError, match="CUDA"):
        mx.quantize(torch.randn(4, 32))
    with pytest.raises(AssertionError, match="CUDA"):
        mx.pack_gate_up(torch.randn(1, 4, 32), torch.randn(1, 4, 32))
    with pytest.raises(AssertionError):
        mx.MxTensor(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(1, 1, 512, dtype=torch.uint8), (4, 32))


# ---- sizes and use beside one another ------------------------------------------------------------
@gpu
def test_offsets_beyond_32_bits():
    """More than 2^31 elements in what is quantised, read back, and written by each product; the far ends are compared."""
    from moonep_b200.ops import mx
    gen = torch.Generator(device="cuda").manual_seed(26)
    bf = dict(device="cuda", dtype=torch.bfloat16)
    w = torch.empty(1100, 2048, 1024, **bf)
    assert w.numel() > 2 ** 31
    w[:-1] = 1.0
    w[-1] = torch.randn(2048, 1024, device="cuda", generator=gen)
    for axis in (-1, -2):
        v = mx.quantize(w, axis).dequantize()[-1].clone()
        assert torch.equal(v, mx.quantize(w[-1], axis).dequantize())
    del w, v
    rows, K, N = 140_000, 64, 16_384
    assert rows * N > 2 ** 31
    x = torch.zeros(rows, K, **bf)
    x[-300:] = torch.randn(300, K, device="cuda", generator=gen)
    qw = mx.quantize(torch.randn(N, K, device="cuda", generator=gen))
    qx = mx.quantize(x)
    last = mx.quantize(x[-300:])                  # (the same tiles: their first row is a multiple of 32 before the end)
    y = mx.matmul(qx, qw)
    assert torch.equal(y[-300:], mx.matmul(last, qw)) and (y[0] == 0).all()
    del y
    gu = mx.pack_gate_up(*(torch.randn(K, N, generator=gen, **bf) for _ in range(2)))
    act = mx.gateup_swiglu(qx, gu, quantize=True)[0]
    assert torch.equal(act.dequantize()[-300:], mx.gateup_swiglu(last, gu, quantize=True)[0].dequantize())
    del act
    d = torch.randn(K, N, device="cuda", generator=gen)
    wd = mx.quantize(d)                           # [K, N]: rows [rows, K] times it
    y = mx.down_dgrad(x, wd)
    assert torch.equal(y[-300:], mx.down_dgrad(x[-300:].contiguous(), wd))


@gpu
def test_two_streams_at_once():
    """Calls on two streams that share weights, and a captured one beside an eager one."""
    from moonep_b200.ops import mx
    gen = _gen(27)
    H, Hp = 512, 256
    ends = _ends([100, 60, 0, 200]).cuda()
    packed = mx.pack_gate_up(*((torch.randn(4, H, Hp, generator=gen) * 0.05).bfloat16().cuda() for _ in range(2))), None, \
        mx.quantize((torch.randn(4, H, Hp, generator=gen) * 0.05).bfloat16().cuda())
    xs = [torch.randn(360, H, generator=gen).bfloat16().cuda() for _ in range(2)]
    with torch.no_grad():
        want = [mx.expert_ffn(x, *packed, ends) for x in xs]
        streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
        graph, static = torch.cuda.CUDAGraph(), xs[0].clone()
        with torch.cuda.graph(graph):
            out = mx.expert_ffn(static, *packed, ends)
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for _ in range(20):
            for s, x, g in zip(streams, xs, got):
                with torch.cuda.stream(s):
                    g.append(mx.expert_ffn(x, *packed, ends))
            graph.replay()
        torch.cuda.synchronize()
    assert torch.equal(out, want[0])
    for g, w in zip(got, want):
        assert all(torch.equal(y, w) for y in g)


@gpu
@pytest.mark.parametrize("call", ["product", "gate and up", "gradients of rows", "bf16 gradients of rows"])
def test_first_call_of_a_thread(call):
    """A thread that has used no device yet, as autograd's before its first backward pass."""
    from moonep_b200.ops import gemm, mx
    gen = _gen(50)
    x, w = torch.randn(64, 128, generator=gen).bfloat16().cuda(), torch.randn(1, 128, 128, generator=gen).bfloat16().cuda()
    q, wq, pair, ends = mx.quantize(x), mx.quantize(w), mx.pack_gate_up(w, w), _ends([64]).cuda()
    run = {"product": lambda: mx.matmul(q, wq, ends), "gate and up": lambda: mx.gateup_swiglu(q, pair, ends)[0],
           "gradients of rows": lambda: mx.down_dgrad(x, wq, ends),
           "bf16 gradients of rows": lambda: gemm.down_dgrad(x, w, ends)}[call]
    want = run().cpu()
    got = []
    thread = threading.Thread(target=lambda: got.append(run()))
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert len(got) == 1 and torch.equal(got[0].cpu(), want)


@gpu
def test_repeated_calls_give_the_same_bits():
    from moonep_b200.ops import mx
    gen = _gen(28)
    H, Hp, sizes = 1024, 512, [64, 448, 0, 128, 256]
    ends, rows = _ends(sizes).cuda(), sum(sizes)
    leaves = [torch.randn(rows, H, generator=gen).bfloat16().cuda()] + \
        [(torch.randn(5, H, Hp, generator=gen) * 0.05).bfloat16().cuda() for _ in range(3)] + [torch.rand(rows, generator=gen).cuda()]
    leaves = [t.requires_grad_(True) for t in leaves]
    dy = torch.randn(rows, H, generator=gen).bfloat16().cuda()
    runs = []
    for _ in range(5):
        y = mx.expert_ffn(*leaves[:4], ends, row_scale=leaves[4])
        runs.append((y.detach(), *torch.autograd.grad(y, leaves, dy)))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))
