"""What the expert FFN reports of groups that weight grads cannot take, and when."""
import pytest
import torch

from tests.test_mx import _gen, _status  # noqa: F401

gpu = pytest.mark.gpu


def _inputs(rows=256, H=128, Hp=64, G=2):
    gen = _gen(70)
    x = torch.randn(rows, H, generator=gen).bfloat16().cuda()
    return x, [(torch.randn(G, H, Hp, generator=gen) * 0.1).bfloat16().cuda().requires_grad_(True) for _ in range(3)]


def _cu(*ends):
    return torch.tensor(ends, dtype=torch.int32, device="cuda")


@gpu
@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_parameters_without_gradients(mode):
    """Inference over leaves that require grad: groups may be of any length, and nothing is reported."""
    from moonep_b200.ops import gemm, mx
    x, w = _inputs()
    with mode():
        y = mx.expert_ffn(x, *w, _cu(100, 200))
    gemm.check_status()
    assert not y.requires_grad
    assert torch.equal(y, mx.expert_ffn(x, *(t.detach() for t in w), _cu(100, 200)))


@gpu
@pytest.mark.parametrize("ends,bad", [((100, 256), [0]), ((64, 200), [1]), ((128, 256), []), ((64, 256), []), ((128, 250), [1]),
                                      ((96, 160), [0])])
def test_gradients_of_groups_that_weight_grads_cannot_take(ends, bad):
    """They are NaN; those of other groups, and the gradients of rows, are what they are."""
    from moonep_b200.ops import gemm, mx
    x, w = _inputs()
    x.requires_grad_(True)
    dy = torch.randn(256, 128, generator=_gen(71)).bfloat16().cuda()
    grads = torch.autograd.grad(mx.expert_ffn(x, *w, _cu(*ends)), (x, *w), dy)
    if bad:
        with pytest.raises(RuntimeError, match=f"group {bad[0]} has"):
            gemm.check_status()
        gemm.reset_status()
    gemm.check_status()
    start = 0
    for g, end in enumerate(ends):
        rows = x.detach()[start:end].clone().requires_grad_(True)
        one = [t.detach()[g].clone().requires_grad_(True) for t in w]
        want = torch.autograd.grad(mx.expert_ffn(rows, *one), (rows, *one), dy[start:end])
        assert torch.equal(grads[0][start:end], want[0])
        for got, ref in zip(grads[1:], want[1:]):
            assert got[g].isnan().all() if g in bad else torch.equal(got[g], ref)
        start = end


def test_every_launch_is_counted():
    from moonep_b200 import _native as nat
    from moonep_b200.ops import mx  # noqa: F401
    launching = {"mep_mx_quantize", "mep_mx_dequantize", "mep_mx_gemm_launch", "mep_mx_dgrad_launch", "mep_mx_sum_parts"}
    names = [n for n in nat._SIGNATURES if n.startswith("mep_mx_")]
    assert launching <= set(names) and all(nat._resolve(n)[1] == (n in launching) for n in names)


@gpu
def test_a_layer_that_stops_training():
    """`training` set to False on a layer that was built for training: its present weights serve, packed in the call until it is
    told to keep them."""
    from tests.test_mx_layer import _buffer, _layer
    buf = _buffer(64, 256, 2, 8)
    layer = _layer(buf, 128)
    x = torch.randn(64, 256, generator=_gen(72)).bfloat16().cuda()
    with torch.no_grad():
        want = layer(x).clone()
        layer.training = False
        assert torch.equal(layer(x), want)
        layer.w_gate.mul_(-1.5)
        turned = layer(x).clone()
        assert not torch.equal(turned, want)
        layer.pack_experts()
        assert torch.equal(layer(x), turned)
    buf.destroy()
