"""Unpacking into a tensor of the caller's is an in-place write like torch's own; and what the copies stand for in a type with fewer exponents."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_tensor_unpacked_into_is_seen_as_changed():
    import gridnet_b200 as gb

    packed = gb.pack_activations(torch.randn(3, 40, device="cuda"))
    kept = torch.randn(3, 40, device="cuda")
    w = torch.randn(3, 40, device="cuda", requires_grad=True)
    product = w * kept
    gb.unpack_activations(packed, out=kept)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()
    for out in (w, w * 1):
        with pytest.raises(RuntimeError, match="out requires a gradient"):
            gb.unpack_activations(packed, out=out)
    with torch.no_grad():
        gb.unpack_activations(packed, out=w)
    assert torch.equal(w, kept)
