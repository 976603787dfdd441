"""What the gated scan, the packed copies and the packed norm refuse, none of it on a GPU; and the definitions that the GPU tests hold the kernels
to, held to torch's own differentiation."""
import numpy as np
import pytest
import torch

import plain_scan


def test_plain_gradients_are_the_derivatives():
    g = torch.Generator().manual_seed(0)
    make = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    z, u, h0, up, upl = make(9, 5) * 2, make(9, 5), make(5), make(9, 5), make(5)
    leaves = [t.clone().requires_grad_(True) for t in (z, u, h0)]
    h, hs = leaves[2], []
    for t in range(9):
        h = torch.sigmoid(leaves[0][t]) * h + torch.sigmoid(-leaves[0][t]) * leaves[1][t]
        hs.append(h)
    want = torch.autograd.grad([torch.stack(hs), h], leaves, [up, upl])
    got = plain_scan.scan(z, u, h0, up, upl)
    for name, w in zip(("gate", "value", "state"), want):
        assert torch.allclose(got[name][0], w, rtol=1e-12, atol=1e-14)


def test_plain_packing():
    x = np.array([[1.0, -125.0, 62.49, 0.5, 1.5, np.inf, np.nan] + [0.0] * 25 + [250.0, 251.0]])
    codes, scales, values = plain_scan.pack(x)
    assert scales.tolist() == [[127, 129]] and codes[0, :7].tolist() == [1, -125, 62, 0, 2, 127, -128]
    assert values[0, 32:].tolist() == [248.0, 252.0]


def test_argument_errors_of_the_library():
    from gridnet_b200._lib import lib

    one = 16  # an address that nothing follows: the checks come first
    assert lib.gn_pack8(one, one, one, -1, 4, 0, None) == -3
    assert lib.gn_pack8(one, one, one, 1 << 40, 1 << 40, 0, None) == -3
    assert lib.gn_pack8(one, one, one, 1, 4, 3, None) == -8
    assert lib.gn_pack8(None, one, one, 1, 4, 0, None) == -1 and lib.gn_unpack8(one, None, one, 1, 4, 0, None) == -1
    assert lib.gn_pack8(None, None, None, 0, 4, 0, None) == 0 and lib.gn_unpack8(None, None, None, 4, 0, 2, None) == 0
    fwd, bwd, step = lib.gn_gated_scan_forward, lib.gn_gated_scan_backward, lib.gn_gated_scan_step
    head, tail = [one, one, None, None, one, None], [32, 8, 32, 8]
    assert fwd(*head, *[None] * 5, 1, 4, 4, 0, *tail, 0, None, 0, None) == -3  # width
    assert fwd(*head, *[None] * 5, 1, 4, 5, 8, *tail, 0, None, 0, None) == -3  # total
    assert fwd(*head, *[None] * 5, 1, 4, 4, 8, *tail, 9, None, 0, None) == -8  # type
    assert fwd(*head, *[None] * 5, 1, 1 << 40, 1 << 40, 1 << 20, *tail, 0, None, 0, None) == -9
    assert fwd(*head, *[None] * 5, 1 << 30, 1 << 40, 1, 8, *tail, 0, None, 0, None) == -9
    assert fwd(None, *head[1:], *[None] * 5, 1, 4, 4, 8, *tail, 0, None, 0, None) == -1
    assert fwd(*head, one, *[None] * 4, 1, 4, 4, 8, *tail, 0, None, 0, None) == -1  # codes of the gate alone
    assert fwd(None, None, None, None, None, None, *[None] * 5, 0, 4, 0, 8, *tail, 0, None, 0, None) == 0
    assert bwd(one, one, one, None, None, None, None, one, None, one, one, None, 1, 4, 4, 8, *tail, 0, None, 0, None) == -1
    assert bwd(one, one, None, None, None, None, None, None, None, one, one, None, 1, 4, 4, 8, *tail, 0, None, 0, None) == -1
    # scratch that is needed and is not there, too small, or not on 16 bytes; what the forward pass leaves for the backward pass
    few, many = (1, 100000, 100000, 8), (1000, 100, 100000, 64)
    need = lib.gn_gated_scan_workspace_bytes(*few, 0, 0, 0, 0)
    assert need > 0 and lib.gn_gated_scan_bounds_bytes(*few, 0, 0) == 0
    for work in ((None, need), (one, need - 1), (one + 4, need)):
        assert fwd(*head, *[None] * 5, *few, *tail, 0, *work, None) == -6
    for packed in (0, 1):
        need = lib.gn_gated_scan_workspace_bytes(*few, 0, 0, 1, packed)
        scales = (one, one) if packed else (None, None)
        for work in ((None, need), (one, need - 1), (one + 4, need)):
            assert bwd(one, one, *scales, None, None, None, one, None, one, one, None, *few, *tail, 0, *work, None) == -6
    assert lib.gn_gated_scan_workspace_bytes(*many, 0, 0, 0, 0) == 0 and lib.gn_gated_scan_workspace_bytes(*many, 0, 0, 1, 1) > 0
    assert lib.gn_gated_scan_bounds_bytes(*many, 0, 0) > 0
    assert bwd(one, one, None, None, None, None, None, one, None, one, one, None, *many, 6400, 64, 6400, 64, 0, None, 0, None) == -6
    assert lib.gn_gated_scan_bounds_bytes(1, 1, 1, 8, 0, 0) == 0 and lib.gn_gated_scan_bounds_bytes(-1, 1, 1, 8, 0, 0) == 0
    assert step(one, one, one, one, one, -1, 8, 8, 8, 0, None) == -3 and step(one, one, one, one, one, 1, 0, 8, 8, 0, None) == -3
    assert step(one, one, one, one, one, 1, 8, 8, 8, -1, None) == -8 and step(one, one, None, one, one, 1, 8, 8, 8, 0, None) == -1
    nf, nb = lib.gn_norm_forward_packed_f32, lib.gn_norm_backward_packed_f32
    assert nf(*[one] * 7, -1, 8, 1e-5, one, 1 << 20, None) == -3 and nf(*[one] * 7, 1, 0, 1e-5, one, 1 << 20, None) == -3
    assert nf(*[one] * 7, 1, 8, 1e-5, one, 16, None) == -6 and nf(*[one] * 7, 1, 8, 1e-5, one + 4, 1 << 20, None) == -6
    assert nf(*[one] * 5, None, one, 1, 8, 1e-5, one, 1 << 20, None) == -1
    assert nf(*[one] * 4, one + 4, one, one, 1, 8, 1e-5, one, 1 << 20, None) == -8
    assert nb(*[one] * 5, None, one, one, 1, 8, one, 1 << 20, None) == -1 and nb(*[one] * 8, 1, 8, None, 0, None) == -6


def test_tiles_of_ragged_sequences_lie_apart():
    """Rows that hold states and maps of tiles (first / tile + sequence + k): rows of the scratch, no two the same, and found again by the
    search that the kernels do, whatever the lengths. The numbers of rows are found from the sizes that the library asks for."""
    from gridnet_b200._lib import lib

    r = np.random.default_rng(0)
    for n, total, width in ((1, 5000, 8), (7, 5000, 100), (40, 3000, 64), (600, 4000, 64)):
        size = (n, 0, total, width, 0, 1)
        padded = (width + 63) // 64 * 64
        found = [(64, lib.gn_gated_scan_workspace_bytes(*size, 0, 0), 8 * padded), (32, lib.gn_gated_scan_workspace_bytes(*size, 1, 1), 12 * padded),
                 (32, lib.gn_gated_scan_bounds_bytes(*size), 4 * width)]
        assert sum(nbytes > 0 for _, nbytes, _ in found) == 2
        for tile, nbytes, row_bytes in found:
            if not nbytes:
                continue
            rows, rest = divmod(nbytes, row_bytes)
            assert rest == 0
            for _ in range(20):
                ends = np.sort(np.concatenate([[0, total], r.integers(0, total + 1, n - 1)]))
                base = [int(first) // tile + i for i, first in enumerate(ends[:-1])]
                used = {base[i] + k: (i, k) for i, (first, end) in enumerate(zip(ends, ends[1:])) for k in range((end - first + tile - 1) // tile)}
                assert len(used) == sum((end - first + tile - 1) // tile for first, end in zip(ends, ends[1:]))
                assert all(0 <= u < rows for u in used)
                for row in range(rows):
                    lo, hi = 0, n
                    while hi - lo > 1:
                        mid = (lo + hi) // 2
                        lo, hi = (mid, hi) if base[mid] <= row else (lo, mid)
                    k = row - base[lo]
                    valid = k >= 0 and k * tile < ends[lo + 1] - ends[lo]
                    assert used.get(row) == ((lo, k) if valid else None)


def test_python_refusals():
    import gridnet_b200 as gb

    x = torch.zeros(2, 3, 4)
    for call in (lambda: gb.pack_activations(x), lambda: gb.unpack_activations(gb.PackedActivations(x.to(torch.int8), x.to(torch.uint8), x.dtype)),
                 lambda: gb.gated_scan(x, x), lambda: gb.gated_scan_step(x, x, x), lambda: gb.GatedRecurrence(4, 2, "cpu")(x),
                 lambda: gb.PackedGridNormOp.apply(torch.zeros(1, 2, 3, 4), torch.zeros(2, 3, 4), torch.zeros(2, 3, 4), 1e-5)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


@pytest.mark.gpu
def test_python_refusals_of_tensors_on_the_device():
    import gridnet_b200 as gb

    x = torch.zeros(2, 3, 4, device="cuda")
    s = torch.zeros(2, 4, device="cuda")
    bad = [
        lambda: gb.pack_activations(x, rows=4), lambda: gb.pack_activations(x, rows=-1),
        lambda: gb.unpack_activations(gb.PackedActivations(x.to(torch.int8), x.to(torch.uint8), x.dtype)),
        lambda: gb.unpack_activations(gb.pack_activations(x), out=torch.zeros(2, 3, 5, device="cuda")),
        lambda: gb.unpack_activations(gb.pack_activations(x), out=torch.zeros(2, 3, 4)),
        lambda: gb.gated_scan(x, x[:, :2]), lambda: gb.gated_scan(x, x.bfloat16()), lambda: gb.gated_scan(s, s), lambda: gb.gated_scan(x, x, s[:1]),
        lambda: gb.gated_scan(x, x, s.bfloat16()), lambda: gb.gated_scan(x, x, s.cpu()), lambda: gb.gated_scan(x[..., :0], x[..., :0]),
        lambda: gb.gated_scan(x, x, None, torch.zeros(0, dtype=torch.long)), lambda: gb.gated_scan(x, x, None, torch.zeros(2, device="cuda")),
        lambda: gb.gated_scan(x, x, None, torch.tensor([0, 3])), lambda: gb.gated_scan(x, x, None, [1, 2]), lambda: gb.gated_scan(x, x, None, [0, 2, 1, 2]),
        lambda: gb.gated_scan_step(s, s, s[:1]), lambda: gb.gated_scan_step(s, s, s.half()), lambda: gb.gated_scan_step(s, s, s, out_state=s[:1]),
        lambda: gb.gated_scan_step(s[0], s[0], s[0]), lambda: gb.PackedGridNormOp.apply(x[None], x, s, 1e-5),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(AssertionError):
            call()
            pytest.fail(f"call {i} was not refused")
    wrong = [lambda: gb.pack_activations(x.double()), lambda: gb.gated_scan(x.double(), x.double()), lambda: gb.gated_scan_step(s.double(), s.double(), s),
             lambda: gb.unpack_activations(gb.pack_activations(x), out=torch.zeros(4, 3, 2, device="cuda").transpose(0, 2)),
             lambda: gb.gated_scan_step(s, s, s, out_state=torch.zeros(4, 2, device="cuda").t()),
             lambda: gb.PackedGridNormOp.apply(x[None].double(), x.double(), x.double(), 1e-5),
             lambda: gb.PackedGridNormOp.apply(torch.zeros(2, 4, 3, 2, device="cuda").transpose(1, 3), x.transpose(0, 0), x, 1e-5)]
    for i, call in enumerate(wrong):
        with pytest.raises((RuntimeError, AssertionError)) as e:
            call()
        assert "not refused" not in str(e.value)


def test_packed_loop_errors():
    from gridnet_b200._lib import lib

    one = 256
    assert lib.gn_loop_packed_bytes(5, 8, 8, 8) == 2 * 512 * 4 + 2 * 16 * 4 + 128 and lib.gn_loop_packed_bytes(0, 8, 8, 8) == 0
    assert lib.gn_loop_packed_workspace_bytes(1, 8, 8, 12, 1, 1, 4, 0, 0, 0) == 0  # no multiple of 8
    assert lib.gn_loop_forward_packed_f32(*[one] * 3, 1, *[one] * 6, 5, 8, 8, 8, 2, 3, 3, 1e-5, 2, 0, one, 1 << 40, None) == -2
    assert lib.gn_loop_backward_packed_f32(*[one] * 3, 2, *[one] * 11, 5, 8, 8, 8, 2, 3, 8, 2, 0, one, 1 << 40, None) == -3  # sets of parameters
    assert lib.gn_gated_loop_forward_packed_f32(*[one] * 8, 5, 8, 8, 8, 0, 3, 1e-5, 3, one, 1 << 40, None) == -5
    assert lib.gn_gated_loop_backward_packed_f32(*[one] * 12, 5, 8, 8, 8, 2, 3, 9, one, 1 << 40, None) == -4


@pytest.mark.gpu
def test_packed_loop_workspaces():
    """The library asks the device whether its kernels apply, so these need one; nothing is launched."""
    from gridnet_b200._lib import lib

    one = 256
    need = lib.gn_loop_packed_workspace_bytes(5, 8, 8, 8, 2, 3, 8, 0, 0, 0)
    fwd = lambda *work, packed=one: lib.gn_loop_forward_packed_f32(  # noqa: E731
        one, one, one, 1, one, one, one, one, packed, one, 5, 8, 8, 8, 2, 3, 8, 1e-5, 2, 0, *work, None)
    assert need > 0 and fwd(one, need - 1) == -6 and fwd(one + 8, need) == -6 and fwd(None, need) == -1 and fwd(one, need, packed=None) == -1
    need = lib.gn_loop_packed_workspace_bytes(5, 8, 8, 8, 2, 3, 8, 0, 0, 1)
    assert lib.gn_loop_backward_packed_f32(*[one] * 3, 1, *[one] * 11, 5, 8, 8, 8, 2, 3, 8, 2, 0, one, need - 1, None) == -6
    need = lib.gn_loop_packed_workspace_bytes(5, 8, 8, 8, 2, 3, 8, 0, 1, 0)
    assert lib.gn_gated_loop_forward_packed_f32(*[one] * 8, 5, 8, 8, 8, 2, 3, 1e-5, 3, one, need - 1, None) == -6
    assert lib.gn_gated_loop_forward_packed_f32(*[one] * 6, None, one, 5, 8, 8, 8, 2, 3, 1e-5, 3, one, need, None) == -1
    need = lib.gn_loop_packed_workspace_bytes(5, 8, 8, 8, 2, 3, 8, 0, 1, 1)
    assert lib.gn_gated_loop_backward_packed_f32(*[one] * 12, 5, 8, 8, 8, 2, 3, 3, one, need - 1, None) == -6
