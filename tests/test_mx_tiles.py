"""4-bit products whose CTA pairs go through many tiles each: several hundred tiles of few k-blocks, with scales that differ from
row to row, against the definition in 64 bits, and the same bits every time.  (Tolerances as in test_mx.py: half a bf16 step of
the value, K 2^-24 of the magnitudes' sum for an fp32 sum, 1e-5 (1 + |gate|) for the sigmoid.)"""
import pytest
import torch

from tests import mx_oracle as ox
from tests.test_mx import HALF, _ends, _gated_ref, _gen, _status  # noqa: F401

pytestmark = pytest.mark.gpu
REPEATS = 30


def _sizes(seed, groups=104):
    """Most groups shorter than an epilogue's step of 32 rows, some of several steps, some of two tiles."""
    gen = _gen(seed)
    sizes = torch.randint(1, 41, (groups,), generator=gen)
    sizes[::13] = torch.randint(100, 301, (len(sizes[::13]),), generator=gen)
    sizes[5] = 0
    return sizes.tolist()


def _same(run):
    """What `run` returns, after many runs that have to give the same bits."""
    first = run()
    for _ in range(REPEATS):
        for a, b in zip(first, run()):
            assert torch.equal(a, b)
    return first


def _within(got, ref, tol):
    d = (got.cpu().double() - ref).abs() - tol
    assert float(d.max()) <= 1e-30, f"{int((d > 1e-30).sum())} of {d.numel()}"


def _operands(H, Hp, seed):
    gen = _gen(seed)
    sizes = _sizes(seed)
    rows, G = sum(sizes), len(sizes)
    x = torch.randn(rows, H, generator=gen).bfloat16()
    wg, wu = ((torch.randn(G, H, Hp, generator=gen) * 2 * H ** -0.5).bfloat16() for _ in range(2))
    scale = torch.rand(rows, generator=gen) * 4 + 0.1
    return gen, rows, _ends(sizes), x, wg, wu, scale


@pytest.mark.parametrize("H,Hp", [(64, 640), (200, 512), (320, 768), (1000, 515)])
def test_gate_and_up(H, Hp):
    from moonep_b200.ops import mx
    _, _, ends, x, wg, wu, scale = _operands(H, Hp, 31)
    gv, uv = (ox.quantise(w.transpose(1, 2).contiguous()) for w in (wg, wu))
    act_ref, gate_ref, up_ref, dg, du, off = _gated_ref(ox.quantise(x), gv, uv, ends.tolist(), scale.double())
    xq, w, cu, s = mx.quantize(x.cuda()), mx.pack_gate_up(wg.cuda(), wu.cuda()), ends.cuda(), scale.cuda()
    act, = _same(lambda: mx.gateup_swiglu(xq, w, cu, row_scale=s)[:1])
    _within(act, act_ref, off)
    values, = _same(lambda: (mx.gateup_swiglu(xq, w, cu, row_scale=s, quantize=True)[0].dequantize(),))
    assert torch.equal(values, mx.quantize(act).dequantize())
    kept = _same(lambda: mx.gateup_swiglu(xq, w, cu, row_scale=s, save_gate_up=True))
    assert torch.equal(kept[0], act)
    _within(kept[1], gate_ref, HALF * gate_ref.abs() + dg)
    _within(kept[2], up_ref, HALF * up_ref.abs() + du)


@pytest.mark.parametrize("H,Hp", [(64, 640), (200, 512), (320, 768), (1000, 515)])
def test_gradients_of_gate_and_up(H, Hp):
    from moonep_b200.ops import mx
    gen, rows, ends, x, wg, wu, scale = _operands(H, Hp, 32)
    d_act = torch.randn(rows, Hp, generator=gen)
    gv, uv = (ox.quantise(w.transpose(1, 2).contiguous()) for w in (wg, wu))
    _, gate, up, dg, du, _ = _gated_ref(ox.quantise(x), gv, uv, ends.tolist(), scale.double())
    sig, d = torch.sigmoid(gate), d_act.double()
    ds = d * scale.double()[:, None]
    want_g, want_u, want_s = ds * up * sig * (1 + gate * (1 - sig)), ds * gate * sig, d * gate * sig * up
    slack = 1e-5 * (1 + gate.abs())
    off_g = ds.abs() * (1.1 * du + 0.5 * up.abs() * dg + 0.5 * du * dg + up.abs() * 1.1 * slack)
    off_u = ds.abs() * (1.1 * dg + slack * gate.abs())
    off_s = (d.abs() * (1.1 * dg * up.abs() + (gate * sig).abs() * du + 1.1 * dg * du)).sum(1) \
        + (want_s.abs() * (slack + Hp * 2.0 ** -24)).sum(1)
    xq, w, cu, s, da = mx.quantize(x.cuda()), mx.pack_gate_up(wg.cuda(), wu.cuda()), ends.cuda(), scale.cuda(), d_act.cuda()
    got = _same(lambda: mx.gateup_swiglu_bwd(da, xq, w, cu, row_scale=s, want_dscale=True))
    _within(got[0], want_g, HALF * want_g.abs() + off_g)
    _within(got[1], want_u, HALF * want_u.abs() + off_u)
    _within(got[2], want_s.sum(1), off_s)


@pytest.mark.parametrize("K", [40, 128, 136, 200, 320, 448])
def test_gradients_of_rows(K):
    """Reductions of 1 to 7 k-blocks, from one projection; of twice as many from gate and up."""
    from moonep_b200.ops import mx
    N, gen, sizes = 1280, _gen(33), _sizes(33)
    rows, G, ends = sum(sizes), len(sizes), _ends(sizes)
    dy = torch.randn(rows, K, generator=gen).bfloat16()
    wd = torch.randn(G, K, N, generator=gen).bfloat16()
    q, d, cu = mx.quantize(wd.cuda()), dy.cuda(), ends.cuda()
    ref, mag = ox.product(dy.double(), ox.quantise(wd).transpose(1, 2), ends.tolist())
    slack = (K + 2) * 2.0 ** -24 * mag
    _within(_same(lambda: (mx.down_dgrad(d, q, cu, fp32=True),))[0], ref, slack)
    _within(_same(lambda: (mx.down_dgrad(d, q, cu),))[0], ref, slack + HALF * ref.abs())
    wg, wu = (torch.randn(G, N, K, generator=gen).bfloat16() for _ in range(2))
    du = torch.randn(rows, K, generator=gen).bfloat16()
    pair, e = mx.pack_gate_up(wg.cuda(), wu.cuda()), du.cuda()
    (a, am), (b, bm) = (ox.product(t.double(), ox.quantise(w.transpose(1, 2).contiguous()).transpose(1, 2), ends.tolist())
                        for t, w in ((dy, wg), (du, wu)))
    got, = _same(lambda: (mx.gateup_dgrad(d, e, pair, cu),))
    _within(got, a + b, (2 * K + 2) * 2.0 ** -24 * (am + bm) + HALF * (a + b).abs())


@pytest.mark.parametrize("N,K", [(1280, 64), (1285, 300), (1536, 520)])
def test_product(N, K):
    from moonep_b200.ops import mx
    gen, sizes = _gen(34), _sizes(34)
    ends = _ends(sizes)
    a, w = torch.randn(sum(sizes), K, generator=gen).bfloat16(), torch.randn(len(sizes), N, K, generator=gen).bfloat16()
    qa, qw, cu = mx.quantize(a.cuda()), mx.quantize(w.cuda()), ends.cuda()
    ref, mag = ox.product(ox.quantise(a), ox.quantise(w), ends.tolist())
    _within(_same(lambda: (mx.matmul(qa, qw, cu),))[0], ref, HALF * ref.abs() + (K + 2) * 2.0 ** -24 * mag)


def test_expert_ffn():
    """A training step with scales of rows: every result the same bits every time."""
    from moonep_b200.ops import mx
    gen, H, Hp = _gen(35), 256, 512
    sizes = (64 * torch.randint(0, 4, (128,), generator=gen)).tolist()
    rows, cu = sum(sizes), _ends(sizes).cuda()
    leaves = [torch.randn(rows, H, generator=gen).bfloat16()] + \
        [(torch.randn(128, H, Hp, generator=gen) * 0.06).bfloat16() for _ in range(3)] + [torch.rand(rows, generator=gen)]
    leaves = [t.cuda().requires_grad_(True) for t in leaves]
    dy = torch.randn(rows, H, generator=gen).bfloat16().cuda()

    def run():
        y = mx.expert_ffn(*leaves[:4], cu, row_scale=leaves[4])
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))
    _same(run)
