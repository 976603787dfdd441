"""Outputs of a caller's that share memory with what a kernel reads are refused, whatever part of it they share."""
import numpy as np
import pytest
import torch

from gridnet_b200.packed import overlaps


def test_overlaps_are_found_byte_by_byte():
    r = np.random.default_rng(0)
    memory = torch.zeros(160, dtype=torch.uint8)
    base = memory.data_ptr()
    found = 0
    for _ in range(4000):
        out_type, in_type = (torch.float32, torch.float16, torch.int8)[r.integers(3)], (torch.float32, torch.bfloat16, torch.uint8)[r.integers(3)]
        lo, nbytes = 4 * int(r.integers(30)), 4 * int(r.integers(12))
        out = memory[lo:lo + nbytes].view(out_type)
        size = torch.empty(0, dtype=in_type).element_size()
        rows, width, distance, at = int(r.integers(0, 5)), int(r.integers(0, 6)), int(r.integers(0, 9)), int(r.integers(0, 8))
        whole = memory[:160].view(in_type)
        if rows and width and at + (rows - 1) * distance + width > whole.numel():
            continue
        t = whole.as_strided((rows, width), (distance, 1), at)
        of_out = set(range(lo, lo + nbytes))
        of_t = {t.data_ptr() - base + i * distance * size + j for i in range(rows) for j in range(width * size)}
        assert overlaps(out, t) == bool(of_out & of_t), (lo, nbytes, in_type, rows, width, distance, at)
        found += bool(of_out & of_t)
    assert 500 < found < 3500


@pytest.mark.gpu
def test_states_and_copies_that_share_memory():
    import gridnet_b200 as gb

    buffer = torch.randn(6, 8, device="cuda")
    both = torch.randn(4, 24, device="cuda")
    z, u, state = torch.randn(4, 8, device="cuda"), torch.randn(4, 8, device="cuda"), torch.randn(4, 8, device="cuda")
    flat = torch.randn(100, device="cuda")
    for args, out in (((z, u, buffer[:4]), buffer[1:5]), ((z, u, buffer[1:5]), buffer[:4]), ((z, u, state), z), ((z, u, state), u),
                      ((z, buffer[2:], state), buffer[:4]), ((both[:, :8], both[:, 16:], state), both.view(-1)[9:41].view(4, 8)),
                      ((z, u, flat[1:33].view(4, 8)), flat[32:64].view(4, 8))):
        with pytest.raises(RuntimeError, match="out_state shares memory with"):
            gb.gated_scan_step(*args, out_state=out)
    # next to each other, in a gap between rows, a state that had to be copied: none of it shared
    want = gb.gated_scan_step(z, u, state)[1]
    for args, out in (((z, u, buffer[:2].view(-1)[:4 * 3].view(4, 3)), buffer[2:].view(-1)[:12].view(4, 3)),):
        args = (args[0][:, :3].contiguous(), args[1][:, :3].contiguous(), args[2])
        assert torch.equal(gb.gated_scan_step(*args)[1], gb.gated_scan_step(*args, out_state=out)[1])
    wide = torch.zeros(2, 64, device="cuda")
    wide[:, :4], wide[:, 60:] = z[:2, :4], u[:2, :4]
    gap = wide[0, 20:28].view(2, 4)
    assert torch.equal(gb.gated_scan_step(wide[:, :4], wide[:, 60:], state[:2, :4].contiguous(), out_state=gap)[1], want[:2, :4])
    turned = state.t().contiguous().t()  # read from a copy, written where it lies
    assert torch.equal(gb.gated_scan_step(z, u, turned, out_state=torch.empty_like(state))[1], want)
    assert torch.equal(gb.gated_scan_step(z, u, state, out_state=state)[1], want)
    memory = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    made = gb.pack_activations(torch.randn(8, 32, device="cuda"))
    codes, scales = memory[:256].view(torch.int8).view(8, 32), memory[1280:1288].view(8, 1)
    codes.copy_(made.codes), scales.copy_(made.scales)
    packed = gb.PackedActivations(codes, scales, torch.float32)
    for lo in (0, 128, 264):
        with pytest.raises(RuntimeError, match="out shares memory with"):
            gb.unpack_activations(packed, out=memory[lo:lo + 1024].view(torch.float32).view(8, 32))
    assert torch.equal(gb.unpack_activations(packed, out=memory[256:1280].view(torch.float32).view(8, 32)), gb.unpack_activations(made))
