"""What the package writes in place through addresses is seen by torch's autograd like torch's own in-place operations."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("packed", [False, True])
def test_a_state_stepped_in_place_ahead_of_the_backward_pass(packed):
    """The backward pass of a scan needs the state that it started from: stepping that state in place is refused there, as z.add_(1) is."""
    import gridnet_b200 as gb

    z, u = (torch.randn(2, 9, 8, device="cuda").requires_grad_(True) for _ in range(2))
    state = torch.randn(2, 8, device="cuda")
    h, _ = gb.gated_scan(z, u, state, packed=packed)
    gb.gated_scan_step(z[:, 0].detach(), u[:, 0].detach(), state, out_state=state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()
    # a view of the state counts too; a step that leaves the state alone does not
    h, _ = gb.gated_scan(z, u, state, packed=packed)
    gb.gated_scan_step(z[:1, 0].detach(), u[:1, 0].detach(), state[1:].clone(), out_state=state[1:])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()
    h, _ = gb.gated_scan(z, u, state, packed=packed)
    gb.gated_scan_step(z[:, 0].detach(), u[:, 0].detach(), state)
    h.sum().backward()


def test_a_state_that_requires_a_gradient_is_not_overwritten():
    import gridnet_b200 as gb

    z, u, state = (torch.randn(2, 8, device="cuda") for _ in range(3))
    before = state.clone()
    leaf = state.requires_grad_(True)
    for out in (leaf, leaf * 1):
        with pytest.raises(RuntimeError, match="out_state requires a gradient"):
            gb.gated_scan_step(z, u, out.detach(), out_state=out)
    assert torch.equal(leaf, before)
    version = leaf._version
    with torch.no_grad():  # as torch's own operations
        gb.gated_scan_step(z, u, leaf, out_state=leaf)
    assert leaf._version > version and not torch.equal(leaf, before)


def test_the_loop_without_gradients_into_a_tensor_that_a_graph_keeps():
    import gridnet_b200 as gb

    model = gb.GridnetModel((8, 8, 8), 1, 1, 8, "cuda")
    net, norm = model.network, model.norm
    x, out = torch.randn(1, 8, 8, 8, device="cuda"), torch.randn(1, 8, 8, 8, device="cuda")
    w = torch.randn(1, 8, 8, 8, device="cuda", requires_grad=True)
    loop = lambda out: gb.outer_forward(net.weight, net.bias, net.residual_scale, norm.weight, norm.bias, x, 1, 1, 8, out=out)  # noqa: E731
    product = w * out
    loop(out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()
