"""Forward-mode derivatives: no operator of the package has them, so a tensor with a tangent is refused, not taken for one without."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from gridnet_b200.backend_cuda import _Op


class _Twice(_Op):
    @staticmethod
    def forward(ctx, x):
        return x * 2

    @staticmethod
    def backward(ctx, g):
        return g * 2


def test_ops_refuse_tangents_with_and_without_gradients():
    x = torch.randn(3)
    for enabled in (True, False):
        with torch.set_grad_enabled(enabled), fw.dual_level():
            with pytest.raises(NotImplementedError):
                _Twice.apply(fw.make_dual(x, torch.ones(3)))
            assert torch.equal(_Twice.apply(x), x * 2)
    # a parameter without a tangent still comes detached where gradients are off
    with torch.no_grad(), fw.dual_level():
        assert _Twice.apply(x.clone().requires_grad_(True)).grad_fn is None


@pytest.mark.gpu
@pytest.mark.parametrize("enabled", [True, False])
def test_scan_and_models_refuse_tangents(enabled):
    import gridnet_b200 as gb

    z, u, s = torch.randn(2, 5, 8, device="cuda"), torch.randn(2, 5, 8, device="cuda"), torch.randn(2, 8, device="cuda")
    want = gb.gated_scan(z, u, s)
    model = gb.GridnetModel((8, 8, 8), 1, 2, 8, "cuda").requires_grad_(False)
    gated = gb.GridnetModel((8, 8, 8), 1, 2, 8, "cuda", activation="tanh", gated=True).requires_grad_(False)
    mnist = gb.MnistModel(2, 2, 1.0, 1.0, False, 1.0, "silu", "cuda").requires_grad_(False)
    grid, images = torch.randn(2, 8, 8, 8, device="cuda"), torch.randn(2, 1, 28, 28, device="cuda")
    with torch.set_grad_enabled(enabled), fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        for args in ((dual(z), u, s), (z, dual(u), s), (z, u, dual(s))):
            with pytest.raises(NotImplementedError):
                gb.gated_scan(*args)
        for call in (lambda: model(dual(grid)), lambda: gated(dual(grid)), lambda: mnist(dual(images)),
                     lambda: torch.func.functional_call(model, {"norm.weight": dual(model.norm.weight)}, (grid,))):
            with pytest.raises(NotImplementedError):
                call()
        # inside such a level, tensors without a tangent are what they were
        assert all(torch.equal(a, b) for a, b in zip(gb.gated_scan(z, u, s), want))
        assert model(grid).isfinite().all()
