"""Padding rows of 4-bit operators: what is said to become zero does so, whatever the inputs hold there."""
import pytest
import torch

from tests.test_mx import _ends, _gen, _status  # noqa: F401

gpu = pytest.mark.gpu

# padding that begins inside a tile's rows, at the second row of a group, nowhere, and behind a whole tile
SIZES, PADS = [128, 64, 0, 192, 320], [[100, 28], [129, 63], [192, 0], [384, 0], [644, 60]]


def _padding(rows, pads=PADS):
    at = torch.zeros(rows, dtype=torch.bool)
    for first, n in pads:
        at[first:first + n] = True
    return at.cuda()


@gpu
@pytest.mark.parametrize("junk", [1.0, float("nan")])
def test_gradients_of_rows(junk):
    from moonep_b200.ops import mx
    gen = _gen(60)
    H, Hp, rows, G = 256, 160, sum(SIZES), len(SIZES)
    cu, pads, padding = _ends(SIZES).cuda(), torch.tensor(PADS, dtype=torch.int32).cuda(), _padding(rows + 40)
    dg, du, dy = (torch.randn(rows + 40, n, generator=gen).bfloat16().cuda() for n in (Hp, Hp, H))
    wgu = mx.pack_gate_up(*((torch.randn(G, H, Hp, generator=gen) * H ** -0.5).bfloat16().cuda() for _ in range(2)))
    wd = mx.quantize((torch.randn(G, H, Hp, generator=gen) * H ** -0.5).bfloat16().cuda())
    calls = (lambda pads: mx.gateup_dgrad(dg, du, wgu, cu, pads=pads), lambda pads: mx.down_dgrad(dy, wd, cu, pads=pads))
    plain = [call(None) for call in calls]
    for d in (dg, du, dy):
        d[padding] *= junk
    for call, want in zip(calls, plain):
        got = call(pads)
        assert (got[padding] == 0).all() and (got[rows:] == 0).all()
        assert torch.equal(got[~padding], want[~padding]) and float(got[~padding][:400].float().abs().min(1).values.max()) > 0
    got = mx.down_dgrad(dy, wd, cu, pads=pads, fp32=True)[:rows][~padding[:rows]]
    assert torch.equal(got.bfloat16(), plain[1][:rows][~padding[:rows]])


@gpu
def test_groups_of_padding_alone():
    """A range that covers a group: none of its rows is computed, the first like the others."""
    from moonep_b200.ops import mx
    gen = _gen(61)
    sizes, ranges = [64, 64, 128, 1], [[0, 64], [100, 28], [128, 128], [256, 1]]
    H, Hp, rows, G = 128, 96, sum(sizes), len(sizes)
    cu, pads, padding = _ends(sizes).cuda(), torch.tensor(ranges, dtype=torch.int32).cuda(), _padding(rows, ranges)
    x, dy = (torch.randn(rows, H, generator=gen).bfloat16().cuda() for _ in range(2))
    wg, wu, wd = ((torch.randn(G, H, Hp, generator=gen) * 0.1).bfloat16().cuda() for _ in range(3))
    d_act, scale = torch.randn(rows, Hp, generator=gen).cuda(), torch.rand(rows, generator=gen).cuda()
    d_act[padding], scale[padding] = float("nan"), float("nan")
    xq, wgu, wdq = mx.quantize(x), mx.pack_gate_up(wg, wu), mx.quantize(wd)
    dg = torch.randn(rows, Hp, generator=gen).bfloat16().cuda()

    def run(pads):
        act, gate, up = mx.gateup_swiglu(xq, wgu, cu, row_scale=scale, save_gate_up=True, pads=pads)
        q = mx.gateup_swiglu(xq, wgu, cu, row_scale=scale, quantize=True, pads=pads)[0]
        backward = mx.gateup_swiglu_bwd(d_act, xq, wgu, cu, row_scale=scale, want_dscale=True, pads=pads)
        return (act, gate, up, q.dequantize(), *backward, mx.matmul(mx.quantize(dg), wdq, cu, pads=pads),
                mx.down_dgrad(dy, wdq, cu, pads=pads), mx.gateup_dgrad(dg, dg, wgu, cu, pads=pads),
                mx.expert_ffn(x, wg, wu, wd, cu, row_scale=scale, pads=pads))

    for got, want in zip(run(pads), run(None)):
        assert (got[padding] == 0).all() and torch.equal(got[~padding], want[~padding])
    # gradients: whatever rows and scales of padding are, as if the groups were not there
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd, scale)]
    got = torch.autograd.grad(mx.expert_ffn(*leaves[:4], cu, row_scale=leaves[4], pads=pads), leaves, dy)
    assert (got[0][padding] == 0).all() and (got[4][padding] == 0).all()
    for t in got[1:4]:
        assert (t[0] == 0).all() and (t[2] == 0).all() and torch.isfinite(t[1]).all()


@gpu
def test_ranges_without_groups_are_refused():
    """They were taken and not looked at."""
    from moonep_b200.ops import mx
    bf = dict(device="cuda", dtype=torch.bfloat16)
    x, d_act, pads = torch.randn(64, 128, **bf), torch.zeros(64, 96, device="cuda"), torch.tensor([[32, 32]], dtype=torch.int32).cuda()
    wg, wd = torch.randn(128, 96, **bf), mx.quantize(torch.randn(128, 96, **bf))
    xq, wgu, dg = mx.quantize(x), mx.pack_gate_up(wg, wg), torch.randn(64, 96, **bf)
    for call in (lambda: mx.matmul(mx.quantize(dg), wd, pads=pads), lambda: mx.gateup_swiglu(xq, wgu, pads=pads),
                 lambda: mx.gateup_swiglu_bwd(d_act, xq, wgu, pads=pads), lambda: mx.down_dgrad(x, wd, pads=pads),
                 lambda: mx.gateup_dgrad(dg, dg, wgu, pads=pads), lambda: mx.expert_ffn(x, wgu, None, wd, pads=pads)):
        with pytest.raises(AssertionError, match="go with cu_seqlens"):
            call()
