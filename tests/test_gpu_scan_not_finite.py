"""An infinite state is infinite from then on, however small the factors of the steps in between become: what the recurrence gives step by step, and
not the 0 * inf of a run whose factors' product is below the smallest number. The same for gradients backward."""
import pytest
import torch

pytestmark = pytest.mark.gpu

INF = float("inf")


def _step_by_step(z, u, state, g, gl):
    """[steps, n] in float64, where the products of gates used here do not underflow."""
    z, u, g, c = z.double(), u.double(), g.double(), gl.double()
    a, n = torch.sigmoid(z), torch.sigmoid(-z)
    h, hs, before = state.double(), [], []
    for t in range(z.shape[0]):
        before.append(h)
        h = a[t] * h + n[t] * u[t]
        hs.append(h)
    cs = [None] * z.shape[0]
    for t in reversed(range(z.shape[0])):
        dh = g[t] + c
        cs[t] = dh
        c = a[t] * dh
    dh = torch.stack(cs)
    return torch.stack(hs), h, a * n * (torch.stack(before) - u) * dh, n * dh, c


# walks and chunks, tiles of a thread's, a warp's and several CTAs' steps; many sequences (a walk), ragged rows
@pytest.mark.parametrize("n,steps", [(1, 3), (1, 16), (1, 40), (2, 65), (3, 200), (1, 1500), (160, 300), (1, 9000)])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("ragged", [False, True])
def test_infinite_states_and_gradients(n, steps, packed, ragged):
    import gridnet_b200 as gb

    width = 8
    # whole gates, values of 1 and 2 in turn and infinities: the packed copies are the inputs, and no value is next to the state ahead of it
    gate = torch.full((n, steps, width), -24.0)  # s is 4e-11: four steps of it are below the smallest number
    gate[..., 4:] = -1.0
    value = (1.0 + torch.arange(steps) % 2)[None, :, None].repeat(n, 1, width)
    state = torch.zeros(n, width)
    state[:, 0], state[:, 4] = INF, -INF
    value[:, steps // 2, 1] = INF
    value[:, steps // 3, 5] = -INF
    grad = torch.ones(n, steps, width)
    grad_last = torch.ones(n, width)
    grad_last[:, 2] = INF
    grad[:, steps // 2, 3] = -INF
    grad[:, steps - 1, 6], grad_last[:, 7] = INF, -INF
    h, last, dz, du, ds = _step_by_step(*(t.transpose(0, 1) for t in (gate, value)), state, grad.transpose(0, 1), grad_last)
    shape = (n * steps, width) if ragged else (n, steps, width)
    leaves = [t.cuda().reshape(s).requires_grad_(True) for t, s in ((gate, shape), (value, shape), (state, (n, width)))]
    offsets = torch.arange(0, n * steps + 1, steps, device="cuda") if ragged else None
    got = gb.gated_scan(*leaves, offsets, packed=packed)
    grads = torch.autograd.grad(got, leaves, [grad.cuda().view(shape), grad_last.cuda()])
    for name, a, b in (("h", got[0], h.transpose(0, 1)), ("last", got[1], last), ("gate", grads[0], dz.transpose(0, 1)),
                       ("value", grads[1], du.transpose(0, 1)), ("state", grads[2], ds)):
        a, b = a.detach().cpu().double().reshape(b.shape), b
        kind = lambda t: torch.where(t.isnan(), 3.0, torch.where(t.isinf(), t.sign(), 0.0))  # noqa: E731
        wrong = (kind(a) != kind(b)).nonzero()
        assert not len(wrong), (name, len(wrong), wrong[0].tolist(), a[tuple(wrong[0])].item(), b[tuple(wrong[0])].item())
        # finite ones: terms of at most 3, rounded 16 times to a step of which a third is passed on
        fine = b.isfinite()
        assert (a[fine] - b[fine]).abs().max() <= 1e-5
