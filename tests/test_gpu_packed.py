"""Activations in 8 bits on the GPU: the format bit by bit, and the norm's gradients at packed inputs, against plain_scan.py and float64."""
import numpy as np
import pytest
import torch

from plain_scan import U, assert_within, pack

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _values(seed, rows, cols, kind):
    """Rows of every scale, groups of zeros, single large values, what is not finite, ties between two codes."""
    r = np.random.default_rng(seed)
    x = r.standard_normal((rows, cols)) * 2.0 ** r.integers(-20, 8, (rows, 1))
    x[r.random(x.shape) < 0.02] *= 50
    if cols > 40:
        x[0, 32:64] = 0
        x[-1, :32] = np.ldexp(1.0, -130)
    flat = x.reshape(-1)
    for v in (np.nan, np.inf, -np.inf, 125.0, 124.5, 123.5, -125.5, 62.5):
        flat[r.integers(0, flat.size, 2)] = v
    return torch.from_numpy(x.astype(np.float32)).to(kind)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (5, 31), (3, 33), (7, 64), (2, 100), (129, 36), (1, 4099), (300, 256)])
def test_codes_scales_and_back(rows, cols, dtype):
    import gridnet_b200 as gb

    x = _values(rows * 1000 + cols, rows, cols, TYPES[dtype])
    codes, scales, values = pack(x.float().numpy())
    p = gb.pack_activations(x.cuda())
    assert p.dtype == x.dtype and p.nbytes == rows * cols + rows * ((cols + 31) // 32)
    assert np.array_equal(p.scales.cpu().numpy(), scales)
    assert np.array_equal(p.codes.cpu().numpy(), codes)
    y = gb.unpack_activations(p)
    # seven bits and a sign fit every type; a half that would be 65536 is 65504
    want = torch.from_numpy(values)
    if dtype == "f16":
        want = torch.where(want.isfinite(), want.clamp(-65504, 65504), want)
    assert y.dtype == x.dtype and torch.equal(y.cpu().double().nan_to_num(nan=1e300), want.nan_to_num(nan=1e300))
    # packing what came back changes nothing
    again = gb.unpack_activations(gb.pack_activations(y))
    assert torch.equal(again.nan_to_num(nan=7.0), y.nan_to_num(nan=7.0))
    wide = gb.unpack_activations(p, out=torch.empty(rows, cols, device="cuda"))
    assert torch.equal(wide.cpu().double().nan_to_num(nan=1e300), torch.from_numpy(values).nan_to_num(nan=1e300))


def test_every_scale():
    """Powers of two from the smallest number to the largest, each just below and at the border where a group takes the next scale."""
    import gridnet_b200 as gb

    tops = [float(m) * 2.0 ** e for e in range(-149, 122) for m in (1, 125 / 64, np.nextafter(np.float32(125 / 64), np.float32(4)))]
    tops = np.array([t for t in tops if t < 3.4e38], np.float32)
    x = np.zeros((len(tops), 32), np.float32)
    x[:, 7], x[:, 30] = tops, -tops / 3
    x[-1, 7] = np.finfo(np.float32).max
    codes, scales, values = pack(x)
    p = gb.pack_activations(torch.from_numpy(x).cuda())
    assert np.array_equal(p.scales.cpu().numpy(), scales) and np.array_equal(p.codes.cpu().numpy(), codes)
    assert scales.min() == 1 and scales.max() == 249
    back = gb.unpack_activations(p).cpu().numpy().astype(np.float64)
    assert np.isfinite(back).all() and np.array_equal(back, values)


def test_large_halves():
    import gridnet_b200 as gb

    x = torch.full((1, 64), 65504.0, dtype=torch.float16, device="cuda")
    x[0, 1], x[0, 2] = float("inf"), float("-inf")
    y = gb.unpack_activations(gb.pack_activations(x))
    assert y[0, 0] == 65504 and y[0, 1] == float("inf") and y[0, 2] == float("-inf") and y[0, 3:].eq(65504).all()


def test_shapes_and_rows():
    import gridnet_b200 as gb

    x = torch.randn(3, 5, 4, 9, device="cuda")
    for rows in range(5):
        p = gb.pack_activations(x, rows=rows)
        codes, scales, values = pack(x.cpu().numpy(), rows)
        assert p.codes.shape == x.shape and tuple(p.scales.shape) == scales.shape
        assert np.array_equal(p.scales.cpu().numpy(), scales) and np.array_equal(gb.unpack_activations(p).cpu().numpy(), values.astype(np.float32))
    # not contiguous: as the values lie in the tensor's order
    t = x.transpose(1, 3)
    assert torch.equal(gb.unpack_activations(gb.pack_activations(t)), gb.unpack_activations(gb.pack_activations(t.contiguous())))
    # an odd address
    flat = torch.randn(1 + 6 * 40, device="cuda")[1:].view(6, 40)
    assert np.array_equal(gb.pack_activations(flat).codes.cpu().numpy(), pack(flat.cpu().numpy())[0])
    for kind in TYPES.values():
        flat = torch.randn(1 + 6 * 64, device="cuda").to(kind)[1:].view(6, 64)
        p = gb.pack_activations(flat)
        assert np.array_equal(p.codes.cpu().numpy(), pack(flat.float().cpu().numpy())[0])
        out = torch.zeros(1 + 6 * 64, device="cuda", dtype=kind)[1:].view(6, 64)
        assert torch.equal(gb.unpack_activations(p, out=out), gb.unpack_activations(p))
    for shape in ((0, 5), (5, 0)):
        e = torch.empty(shape, device="cuda")
        assert gb.unpack_activations(gb.pack_activations(e)).shape == shape


def test_places_past_32_bits():
    """2^31 + 2^12 values: codes of the last row are those of the row alone."""
    import gridnet_b200 as gb

    rows, cols = (1 << 19) + 1, 1 << 12
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[:-2] = 1
    x[-2:] = torch.randn(2, cols, device="cuda")
    p = gb.pack_activations(x)
    alone = gb.pack_activations(x[-2:].clone())
    assert torch.equal(p.codes[-2:], alone.codes) and torch.equal(p.scales[-2:], alone.scales)
    back = gb.unpack_activations(p)
    assert torch.equal(back[-2:], gb.unpack_activations(alone)) and torch.equal(back[:2], x[:2])
    del x, p, back


def _norm_want(x, gamma, beta, g, eps=1e-5):
    """Values and how far float32 may be off. Sums are double over sums of four products in float32, so a mean is off by 4 U of the mean
    magnitude; mean and deviation are rounded to float32, the deviation after a variance that is off by 4 U of the mean square."""
    B = x.shape[0]
    x, g = x.double().reshape(B, -1), g.double().reshape(B, -1)
    ga, be = gamma.double().reshape(-1), beta.double().reshape(-1)
    m, var = x.mean(1, keepdim=True), x.var(1, unbiased=False, keepdim=True)
    r = (var + eps).rsqrt()
    em = 5 * U * x.abs().mean(1, keepdim=True)
    er = r * (2 * U + 2 * U * (x.square().mean(1, keepdim=True)) * r * r)
    hat = lambda v: ((v - m) * r, U * 3 * ((v - m) * r).abs() + r * em + U * r * (v.abs() + m.abs()) + er * (v - m).abs())  # noqa: E731
    y, ey = hat(x)
    out = {"y": (y * ga + be, ey * ga.abs() + 2 * U * ((y * ga).abs() + be.abs()))}
    xt = torch.from_numpy(pack(x.float().numpy())[2])
    p, ep = hat(xt)
    q, eq = g * ga, U * (g * ga).abs()
    mq, mqp = q.mean(1, keepdim=True), (q * p).mean(1, keepdim=True)
    emq, emqp = 5 * U * q.abs().mean(1, keepdim=True), (6 * U * (q * p).abs() + q.abs() * ep).mean(1, keepdim=True)
    inner, einner = q - mq - p * mqp, eq + emq + ep * mqp.abs() + p.abs() * emqp + 4 * U * (q.abs() + mq.abs() + (p * mqp).abs())
    out["x"] = r * inner, r * einner + er * inner.abs() + U * (r * inner).abs()
    # over the batch: a rounding per sample
    out["gamma"] = (g * p).sum(0), (g.abs() * ep).sum(0) + (B + 1) * U * (g * p).abs().sum(0)
    out["beta"] = g.sum(0), (B + 1) * U * g.abs().sum(0)
    return out


@pytest.mark.parametrize("B,grid", [(1, (4, 4, 4)), (3, (8, 8, 8)), (2, (1, 1, 1)), (5, (3, 5, 7)), (4, (2, 9, 18)), (9, (16, 24, 16)), (2, (32, 32, 40)), (130, (8, 8, 4)), (1100, (4, 4, 4)), (9600, (2, 2, 2)), (2, (64, 72, 72))])
def test_norm(B, grid):
    import gridnet_b200 as gb

    gen = torch.Generator().manual_seed(B)
    x, g = 1.5 * torch.randn(B, *grid, generator=gen) + 0.3, torch.randn(B, *grid, generator=gen)
    gamma, beta = 1 + 0.2 * torch.randn(grid, generator=gen), 0.3 * torch.randn(grid, generator=gen)
    want = _norm_want(x, gamma, beta, g)
    leaves = [t.cuda().requires_grad_(True) for t in (x, gamma, beta)]
    y = gb.PackedGridNormOp.apply(*leaves, 1e-5)
    grads = torch.autograd.grad(y, leaves, g.cuda())
    for name, got in zip(("y", "x", "gamma", "beta"), (y, *grads)):
        assert_within(got.reshape(want[name][0].shape), *want[name], name)


def test_norm_module_and_setting():
    """keep_packed: the module's gradients are those of the packed op, a pass that started before is not touched, and nothing is kept
    where no gradient is wanted. Memory between the passes: 33/128 of the input."""
    import gridnet_b200 as gb

    grid, B = (32, 32, 32), 16
    norm = gb.GridNorm(grid, "cuda")
    x = torch.randn(B, *grid, device="cuda", requires_grad=True)
    g = torch.randn(B, *grid, device="cuda")
    plain = norm(x)
    assert gb.keep_packed(True) is False
    try:
        ours = norm(x)
        assert torch.equal(plain, ours)
        a, b = torch.autograd.grad(plain, x, g)[0], torch.autograd.grad(ours, x, g)[0]
        direct = torch.autograd.grad(gb.PackedGridNormOp.apply(x, norm.weight, norm.bias, norm.eps), x, g)[0]
        assert torch.equal(b, direct) and not torch.equal(a, b)
        # half a step of the largest of 32 each: what it does to the gradient's mean terms and p
        assert (a - b).abs().max() < 0.1
        with torch.no_grad():
            quiet = norm(x)
        assert torch.equal(quiet, plain)
        h = x.detach() * 1  # nobody else holds it
        h.requires_grad_(True)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = norm(h.clone())
        kept = torch.cuda.memory_allocated() - before - y.numel() * 4
        assert kept < 0.3 * h.numel() * 4, kept
    finally:
        assert gb.keep_packed(False) is True
    assert torch.equal(torch.autograd.grad(norm(x), x, g)[0], a)


def test_norm_odd_address_and_empty_batch():
    import gridnet_b200 as gb

    grid = (4, 4, 6)
    gen = torch.Generator().manual_seed(2)
    x, g = torch.randn(3, *grid, generator=gen), torch.randn(3, *grid, generator=gen)
    gamma, beta = torch.ones(grid), torch.zeros(grid)
    shifted = lambda t: torch.cat([torch.zeros(1), t.reshape(-1)]).cuda()[1:].view(t.shape)  # noqa: E731
    leaves = [shifted(t).requires_grad_(True) for t in (x, gamma, beta)]
    y = gb.PackedGridNormOp.apply(*leaves, 1e-5)
    want = _norm_want(x, gamma, beta, g)
    for name, got in zip(("y", "x", "gamma", "beta"), (y, *torch.autograd.grad(y, leaves, shifted(g)))):
        assert_within(got.reshape(want[name][0].shape), *want[name], name)
    e = torch.empty(0, *grid, device="cuda", requires_grad=True)
    w = torch.ones(grid, device="cuda", requires_grad=True)
    y = gb.PackedGridNormOp.apply(e, w, torch.zeros(grid, device="cuda"), 1e-5)
    ge, gw = torch.autograd.grad(y, (e, w), torch.empty_like(y))
    assert y.shape == ge.shape == (0, *grid) and not gw.any()


def test_norm_captured_and_bit_stable():
    import gridnet_b200 as gb

    grid, B = (16, 16, 24), 7
    x, g = torch.randn(B, *grid, device="cuda"), torch.randn(B, *grid, device="cuda")
    w, b = torch.rand(grid, device="cuda"), torch.rand(grid, device="cuda")

    def run():
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = gb.PackedGridNormOp.apply(*leaves, 1e-5)
        return [y.detach(), *torch.autograd.grad(y, leaves, g)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for _ in range(2):
        x.normal_(), g.normal_()
        graph.replay()
        want, again = run(), run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) and torch.equal(c, d) for a, c, d in zip(outs, want, again))
