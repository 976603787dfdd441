"""What a copy of a wide type stands for in a half: 65536, which only rounding to the format makes of a half, is 65504; what is beyond that is
rounded as every conversion to half, to infinity."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [64, 33])  # whole groups, and the kernels for other widths
def test_large_values_unpacked_to_halves(dtype, cols):
    import gridnet_b200 as gb

    x = torch.zeros(4, cols, device="cuda", dtype=dtype)
    x[0, :6] = torch.tensor([65536.0, -65536.0, 65536.0 * 2, 1e6, -3e38, 60000.0])
    x[1, :3] = torch.tensor([float("inf"), float("-inf"), float("nan")])
    x[2, :3] = torch.tensor([65536.0, -65536.0, 1000.0])
    x[3, :2] = torch.tensor([1e6, -1e6])
    packed = gb.pack_activations(x)
    stands_for = gb.unpack_activations(packed, out=torch.empty(4, cols, device="cuda"))
    half = gb.unpack_activations(packed, out=torch.empty(4, cols, device="cuda", dtype=torch.float16))
    want = torch.where(stands_for.abs() == 65536, 65504 * stands_for.sign(), stands_for).half()
    assert want[3, 0] == float("inf") and want[2, 0] == 65504 and want[1, 2].isnan()
    assert torch.equal(half.nan_to_num(nan=7.0, posinf=1.0, neginf=-1.0), want.nan_to_num(nan=7.0, posinf=1.0, neginf=-1.0))
