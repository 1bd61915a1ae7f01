"""The calls of the operators around the expert layer under torch's transforms."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.fixture(scope="module")
def data():
    g = torch.Generator(device="cuda").manual_seed(0)
    return [torch.randn(s, generator=g, device="cuda").to(BF) for s in ((4, 64), (64, 64), (64,))]


def _calls(x, w, v):
    import dw_tpu_b200 as dw
    return [(x, lambda t: dw.dense_matmul(t, w)), (w, lambda t: dw.dense_matmul(x, t)),
            (x, lambda t: dw.pre_norm(t, v)), (v, lambda t: dw.pre_norm(x, t)),
            (x, lambda t: dw.post_norm(t, x)[0]), (x, lambda t: dw.post_norm(x, t)[0]),
            (x, lambda t: dw.route_grouped_topk(t, 4, 8, 4)[0])]


def test_tangents_and_gradients_are_refused(data):
    """Forward mode, and the transforms that wrap tensors: an error, not a result
    without its derivative."""
    import torch.autograd.forward_ad as fw
    for t, call in _calls(*data):
        with fw.dual_level(), pytest.raises(ValueError, match="inference only"):
            call(fw.make_dual(t, torch.ones_like(t)))
        for transform in (lambda: torch.func.jvp(call, (t,), (torch.ones_like(t),)),
                          lambda: torch.func.grad(lambda u: call(u).float().sum())(t),
                          lambda: torch.func.vmap(call)(t[None])):
            with pytest.raises((RuntimeError, ValueError)):
                transform()


def test_inference_mode_keeps_the_results(data):
    for t, call in _calls(*data):
        plain = call(t)
        with torch.inference_mode():
            assert torch.equal(call(t.clone()), plain)
        with torch.no_grad():
            assert torch.equal(call(t.clone().requires_grad_()), plain)
