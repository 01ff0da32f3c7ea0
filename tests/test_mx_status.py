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
