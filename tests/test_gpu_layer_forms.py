"""GatedRecurrence over ragged rows, in 16 bits, and with copies in 8 bits: the projection's halves through the scan, gradients included."""
import pytest
import torch

from plain_scan import assert_within, scan_all

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ragged", [False, True])
def test_layer(dtype, ragged):
    import gridnet_b200 as gb

    torch.manual_seed(1)
    layer = gb.GatedRecurrence(12, 40, "cuda", dtype=dtype)
    x = torch.randn(27, 12, device="cuda", dtype=dtype)
    state = torch.randn(3, 40, device="cuda")
    ends = [0, 4, 4, 27] if ragged else [0, 9, 18, 27]
    offsets = torch.tensor(ends, device="cuda") if ragged else None
    x, state = (x if ragged else x.view(3, 9, 12)).requires_grad_(True), state.requires_grad_(True)
    h, last = layer(x, state, offsets)
    z, u = layer.proj(x).reshape(27, 80).chunk(2, -1)
    want = scan_all(z.detach().cpu().double(), u.detach().cpu().double(), state.detach().cpu().double(), list(zip(ends, ends[1:])))
    assert h.dtype == dtype and last.dtype == torch.float32
    assert_within(h.reshape(27, 40), *want["h"], "h", dtype)
    assert_within(last, *want["last"], "last")
    # the layer's gradients are those of the scan taken through the projection
    up, upl = torch.randn_like(h), torch.randn_like(last)
    leaves = [x, state, *layer.parameters()]
    for packed in (False, True):
        previous = gb.keep_packed(packed)
        try:
            got = torch.autograd.grad(layer(x, state, offsets), leaves, [up, upl])
        finally:
            gb.keep_packed(previous)
        gate, value = layer.proj(x).chunk(2, -1)
        direct = torch.autograd.grad(gb.gated_scan(gate, value, state, offsets, packed=packed), leaves, [up, upl])
        assert all(torch.equal(a, b) for a, b in zip(got, direct))
        assert all(g.isfinite().all() and g.any() for g in got)
