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
