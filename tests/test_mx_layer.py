"""The MoE layer with 4-bit experts (one rank): inference and training against the formulas in 64 bits on the quantised
operands, the same layer in its several forms bit for bit, a decoder that trains on it."""
import pytest
import torch

from tests import mx_oracle as ox

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -8


def _buffer(S, H, K, E, **kw):
    from moonep_b200 import Buffer
    return Buffer(S, H, K, E, 1, num_sms=4, token_padding=kw.pop("pad", 64), timeout_s=5.0)


def _layer(buf, Hp, **kw):
    from moonep_b200.models.moe_layer import MoELayer
    return MoELayer(buf, Hp, None, seed=3, init_std=0.06, expert_format="mxfp4", **kw)


def _routing(layer, x):
    from moonep_b200.ops import elementwise as ew
    from moonep_b200.ops import gemm
    topk, w, _ = ew.router_topk(gemm.dense(x, layer.w_router), layer.buf.K, layer.router_bias)
    return topk.cpu().long(), w.cpu().double()


def _reference(layer, x, dy=None):
    """y, and with dy the gradients of x but for the router's share, of the three projections, and of the route weights."""
    S, H, K, E = layer.buf.S, layer.buf.H, layer.buf.K, layer.buf.E
    topk, w = _routing(layer, x)
    xv = ox.quantise(x.cpu())
    gv, uv = (ox.quantise(t.cpu().transpose(1, 2).contiguous()) for t in (layer.w_gate, layer.w_up))
    dv = ox.quantise(layer.w_down.cpu())
    y, dx = torch.zeros(S, H, dtype=torch.float64), torch.zeros(S, H, dtype=torch.float64)
    grads = [torch.zeros(layer.w_gate.shape, dtype=torch.float64) for _ in range(3)]
    dw = torch.zeros(S, K, dtype=torch.float64)
    for e in range(E):
        s, k = (topk == e).nonzero(as_tuple=True)
        gate, up = xv[s] @ gv[e].T, xv[s] @ uv[e].T
        sig = torch.sigmoid(gate)
        act = ox.quantise((gate * sig * up * w[s, k, None]).bfloat16())
        y.index_add_(0, s, act @ dv[e].T)
        if dy is not None:
            d = dy.cpu().double()[s]
            da = d @ dv[e]
            dw[s, k] = (da * gate * sig * up).sum(1)
            da = da * w[s, k, None]
            dg, du = da * up * sig * (1 + gate * (1 - sig)), da * gate * sig
            dx.index_add_(0, s, dg @ gv[e] + du @ uv[e])
            for i, g in enumerate((xv[s].T @ dg, xv[s].T @ du, d.T @ act)):
                grads[i][e] = g
    return y, dx, grads, dw, topk, w


def _near(got, ref, tol):
    d = float((got.detach().cpu().double() - ref).norm() / ref.norm().clamp_min(1e-30))
    assert d <= tol, d


# Roundings to bf16 are at most HALF of a value: a row of y has one per expert and one of the sum; gradients of x have
# those of d gate / d up, of the rows, of their sum, and of the router's share that is added to it.
@pytest.mark.parametrize("S,H,Hp,K,E,pad", [(256, 256, 128, 4, 8, 64), (1, 128, 64, 2, 8, 64), (333, 384, 192, 3, 16, 128)])
def test_inference(S, H, Hp, K, E, pad):
    from moonep_b200.ops import gemm
    buf = _buffer(S, H, K, E, pad=pad)
    layer = _layer(buf, Hp, train=False)
    x = torch.randn(S, H, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    with torch.no_grad():
        y = layer(x)
        again = layer(x)
    buf.check()
    gemm.check_status()
    _near(y, _reference(layer, x)[0], 2 * HALF)
    assert torch.equal(y, again)
    # the same weights quantised in the pass
    train = _layer(buf, Hp)
    assert torch.equal(train.w_gate, layer.w_gate)
    with torch.no_grad():
        assert torch.equal(train(x), y)
    buf.destroy()


@pytest.mark.parametrize("fused_combine", [True, False])
def test_training_step(fused_combine):
    from moonep_b200.ops import gemm
    S, H, Hp, K, E = 320, 256, 192, 4, 8
    buf = _buffer(S, H, K, E)
    bias = torch.zeros(E, device="cuda")
    bias[5] = -100.0                                   # one expert without tokens
    layer = _layer(buf, Hp, router_bias=bias, fused_combine=fused_combine)
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(S, H, generator=gen).bfloat16().cuda().requires_grad_(True)
    dy = torch.randn(S, H, generator=gen).bfloat16().cuda()
    y = layer(x)
    y.backward(dy)
    buf.check()
    gemm.check_status()
    ref, dx, grads, dw, topk, w = _reference(layer, x.detach(), dy)
    _near(y, ref, 2 * HALF)
    dl = torch.zeros(S, E, dtype=torch.float64)        # router: softmax over the selected logits
    dl.scatter_(1, topk, w * (dw - (w * dw).sum(1, keepdim=True)))
    _near(x.grad, dx + dl @ layer.w_router.cpu().double().T, 4 * HALF)
    for got, want in zip((layer.g_gate, layer.g_up, layer.g_down), grads):
        _near(got, want, 2 * HALF)
    _near(layer.g_router[0], x.detach().cpu().double().T @ dl, 4 * HALF)
    assert float(layer.g_gate[5].abs().sum()) == 0.0
    buf.destroy()


def test_fused_sgd_and_accumulation():
    """SGD in the weight-grad epilogues == grads stored, then SGD; accumulated grads == their sum."""
    S, H, Hp, K, E = 192, 256, 128, 2, 8
    buf = _buffer(S, H, K, E)
    gen = torch.Generator().manual_seed(7)
    x, dy = (torch.randn(S, H, generator=gen).bfloat16().cuda() for _ in range(2))
    res, grads = [], []
    for fused in (False, True):
        layer = _layer(buf, Hp)
        if fused:
            layer.fuse_sgd(0.5)
        xo = x.clone().requires_grad_(True)
        y = layer(xo)
        y.backward(dy)
        if not fused:
            grads = [g.clone() for g in (layer.g_gate, layer.g_up, layer.g_down)]
        layer.sgd_step(0.5)
        res.append((y.detach().clone(), xo.grad.clone(), layer.w_gate.clone(), layer.w_up.clone(), layer.w_down.clone()))
    for a, b in zip(*res):
        assert torch.equal(a, b)
    layer = _layer(buf, Hp)
    for step in range(2):
        layer.accumulate_grads = step > 0
        layer(x.clone().requires_grad_(True)).backward(dy)
    for got, one in zip((layer.g_gate, layer.g_up, layer.g_down), grads):
        assert torch.equal(got, one + one)
    buf.destroy()


def test_packed_weights_follow_the_layer():
    S, H, Hp, K, E = 64, 256, 128, 2, 8
    buf = _buffer(S, H, K, E)
    layer, other = _layer(buf, Hp, train=False), _layer(buf, Hp, train=False)
    x = torch.randn(S, H, generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
    with torch.no_grad():
        y0 = layer(x).clone()
        layer.w_gate.mul_(-1.5)
        assert torch.equal(layer(x), y0)               # the packed weights serve until they are packed again
        layer.pack_experts()
        y1 = layer(x).clone()
        assert not torch.equal(y0, y1)
        other.load_state_dict(layer.state_dict())
        assert torch.equal(other(x), y1)
    buf.destroy()


def test_captured_inference():
    from moonep_b200.utils.graph import GraphedStep
    S, H, Hp, K, E = 1, 256, 128, 2, 8
    buf = _buffer(S, H, K, E)
    layer = _layer(buf, Hp, train=False)
    gen = torch.Generator().manual_seed(9)
    xs = [torch.randn(S, H, generator=gen).bfloat16().cuda() for _ in range(3)]
    with torch.no_grad():
        want = [layer(x).clone() for x in xs]
        step = GraphedStep(lambda x: layer(x), [xs[0]])
        for x, y in zip(xs, want):
            assert torch.equal(step(x), y)
    buf.check()
    del step
    buf.destroy()


def test_decoder_with_4_bit_experts():
    """A decoder's step runs, with grads on every parameter, and saves and restores."""
    from moonep_b200.models.decoder import MoEDecoder
    S, H, Hp, K, E = 128, 256, 128, 2, 8
    buf = _buffer(S, H, K, E)
    model = MoEDecoder(512, H, 2, 4, lambda i: _layer(buf, Hp)).cuda()
    tokens = torch.randint(0, 512, (S,), generator=torch.Generator().manual_seed(1)).cuda()
    loss = model(tokens, tokens.roll(-1))
    loss.backward()
    assert torch.isfinite(loss) and all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())
    assert all(float(m.g_down.abs().sum()) > 0 for m in model.moe_layers())
    model.zero_grad()
    model.train_step(tokens, tokens.roll(-1), 1e-3, fuse_expert_sgd=True)
    with torch.no_grad():
        want = model(tokens, tokens.roll(-1))
    served = MoEDecoder(512, H, 2, 4, lambda i: _layer(buf, Hp, train=False)).cuda()
    served.load_state_dict_all(model.state_dict_all())
    with torch.no_grad():
        assert torch.equal(served(tokens, tokens.roll(-1)), want)
    buf.destroy()


def test_refusals():
    from moonep_b200.models.moe_layer import MoELayer
    buf = _buffer(64, 256, 2, 8)
    for kw in (dict(expert_format="fp4"), dict(expert_format="mxfp4", hidden_in_place=True),
               dict(expert_format="mxfp4", fused_dispatch=True)):
        with pytest.raises(AssertionError):
            MoELayer(buf, 128, None, **kw)
    with pytest.raises(AssertionError):
        MoELayer(buf, 128, None).pack_experts()
    buf.destroy()
