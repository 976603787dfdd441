"""The gated scan on the GPU against its definition in float64 (plain_scan.py)."""
import pytest
import torch

from plain_scan import U, assert_within, pack, scan, scan_all

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _inputs(seed, total, n, width, dtype):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(total, width, generator=g) * 2 + 1.5 + torch.randn(width, generator=g)
    make = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return z.to(dtype), make(total, width).to(dtype), make(n, width), make(total, width).to(dtype), make(n, width)


def _want(z, u, h0, spans, g, gl, packed):
    """Outputs at the inputs, gradients at the packed copies if so."""
    out = scan_all(z.double(), u.double(), h0.double(), spans)
    zz, uu = (torch.from_numpy(pack(t.float().numpy())[2]) for t in (z, u)) if packed else (z.double(), u.double())
    back = scan_all(zz, uu, h0.double(), spans, g.double(), gl.double())
    return {**{k: back[k] for k in ("gate", "value", "state")}, "h": out["h"], "last": out["last"]}


def _check(want, h, last, grads, dtype, shape):
    for name, got in (("h", h), ("gate", grads[0]), ("value", grads[1])):
        assert got.dtype == dtype
        assert_within(got.reshape(shape), *want[name], name, dtype)
    assert_within(last, *want["last"], "last")
    assert_within(grads[2], *want["state"], "state")


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("n,steps,width", [(1, 1, 1), (1, 2, 4), (3, 7, 33), (2, 8, 32), (2, 9, 36), (1, 64, 64), (1, 65, 5), (2, 128, 40),
                                           (1, 129, 68), (1, 257, 12), (2, 513, 100), (1, 1025, 8), (1, 4099, 6)])
def test_dense(n, steps, width, packed, dtype):
    import gridnet_b200 as gb

    kind = TYPES[dtype]
    z, u, h0, g, gl = _inputs(steps * 131 + width, n * steps, n, width, kind)
    want = _want(z, u, h0, [(i * steps, (i + 1) * steps) for i in range(n)], g, gl, packed)
    leaves = [t.cuda().requires_grad_(True) for t in (z.view(n, steps, width), u.view(n, steps, width), h0)]
    h, last = gb.gated_scan(*leaves, packed=packed)
    grads = torch.autograd.grad([h, last], leaves, [g.view(n, steps, width).cuda(), gl.cuda()])
    _check(want, h, last, grads, kind, (n * steps, width))


def _far_values(seed, rows, cols):
    """Rows of every scale, zeros, the largest numbers; what is not finite in every third group only, so that both ways of packing are taken."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp2(torch.randint(-140, 122, (rows, 1), generator=g).float())
    x[::5] = 0
    x[1::7] = torch.randn(x[1::7].shape, generator=g) * 2.0**125
    for v in (float("inf"), float("-inf"), float("nan")):
        x[torch.randint(0, rows, (1 + rows // 40,), generator=g), torch.randint(0, cols, (1 + rows // 40,), generator=g)] = v
    return x


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("lengths,width", [([1], 1), ([16, 15, 17, 0, 1], 64), ([37, 70], 33), ([64, 129, 3], 63), ([300], 100), ([700, 5], 34), ([2000], 65),
                                           ([40] * 9, 128)])
def test_copies_are_those_of_packing(lengths, width, dtype):
    """What the forward pass keeps of gate and value has the codes and scales of the format, whole tiles, last rows and odd widths alike."""
    import gridnet_b200 as gb
    from gridnet_b200.scan import _packed_at

    total = sum(lengths)
    offsets = torch.tensor([0, *lengths]).cumsum(0).cuda()
    z, u = (_far_values(seed + width, total, width).to(TYPES[dtype]) for seed in (1, 1000))
    leaves = [t.cuda().requires_grad_(True) for t in (z, u)]
    for one, spans in ((leaves, offsets), ([t.detach()[None].requires_grad_(True) for t in leaves], None)):
        h, _ = gb.gated_scan(*one, None, spans, packed=True)
        kept, places = h.grad_fn.saved_tensors[0], _packed_at(total, width)
        for i, x in enumerate((z, u)):
            codes, scales, _ = pack(x.float().numpy())
            got = kept[places[i]:][:total * width].view(torch.int8).cpu()
            assert torch.equal(got, torch.from_numpy(codes).reshape(-1))
            assert torch.equal(kept[places[i + 2]:][:scales.size].cpu(), torch.from_numpy(scales).reshape(-1))


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("lengths,width", [([0, 1, 0, 5, 130, 0], 36), ([700, 3, 64, 65, 1], 7), ([0, 0], 4), ([1] * 40, 64), ([2100, 0, 9], 20)])
def test_ragged_with_held_and_reset_steps(lengths, width, packed, dtype):
    """Gates of +inf hold the state whatever the value is, gates of -inf take the value; offsets of both types, on host and device."""
    import gridnet_b200 as gb

    kind, n, total = TYPES[dtype], len(lengths), sum(lengths)
    z, u, h0, g, gl = _inputs(total + width, total, n, width, kind)
    if total > 4:
        held, reset = torch.arange(total) % 5 == 2, torch.arange(total) % 11 == 3
        z[held], u[held] = float("inf"), float("nan")
        z[reset] = float("-inf")
        z[:, 1] = torch.where(torch.arange(total) % 3 == 0, float("inf"), z[:, 1].float()).to(kind)  # in some channels only
    ends = torch.tensor([0] + lengths).cumsum(0)
    spans = list(zip(ends.tolist(), ends.tolist()[1:]))
    want = _want(z, u, h0, spans, g, gl, packed)
    for offsets in (ends.cuda(), ends.int().cuda(), ends, ends.tolist()):
        leaves = [t.cuda().requires_grad_(True) for t in (z, u, h0)]
        h, last = gb.gated_scan(*leaves, offsets, packed=packed)
        grads = torch.autograd.grad([h, last], leaves, [g.cuda(), gl.cuda()])
        _check(want, h, last, grads, kind, (total, width))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("lengths", [[9000, 0, 3, 40], [20000], [2500, 2500]])
def test_long_sequences_with_few_resets(lengths, packed):
    """Many tiles to a run of tiles: a reset in some of the channels of some of them, not finite values ahead of one."""
    import gridnet_b200 as gb

    n, total, width = len(lengths), sum(lengths), 34
    z, u, h0, g, gl = _inputs(total, total, n, width, torch.float32)
    for at, ch in ((1700, 3), (1701, 3), (2111, 20), (4444 % total, 33), (total - 70, 0)):
        z[at, ch] = float("-inf")
    ends = torch.tensor([0] + lengths).cumsum(0)
    want = _want(z, u, h0, list(zip(ends.tolist(), ends.tolist()[1:])), g, gl, packed)
    leaves = [t.cuda().requires_grad_(True) for t in (z, u, h0)]
    h, last = gb.gated_scan(*leaves, ends, packed=packed)
    grads = torch.autograd.grad([h, last], leaves, [g.cuda(), gl.cuda()])
    _check(want, h, last, grads, torch.float32, (total, width))
    # a state that is not finite ends at the next reset: from there on nothing has changed
    u[900:905, 3], u[2100, 20] = float("nan"), float("inf")
    spoilt, _ = gb.gated_scan(z.cuda(), u.cuda(), h0.cuda(), ends)
    assert not spoilt[905:1700, 3].isfinite().any() and not spoilt[2100:2111, 20].isfinite().any()
    assert torch.equal(spoilt[1700:, 3], h[1700:, 3]) and torch.equal(spoilt[2111:, 20], h[2111:, 20])


@pytest.mark.parametrize("packed", [False, True])
def test_rows_of_no_sequence_are_zero(packed):
    import gridnet_b200 as gb

    z, u, h0, g, gl = _inputs(3, 50, 2, 24, torch.float32)
    spans = [(4, 11), (11, 40)]
    want = _want(z, u, h0, spans, g, gl, packed)
    leaves = [t.cuda().requires_grad_(True) for t in (z, u, h0)]
    h, last = gb.gated_scan(*leaves, torch.tensor([4, 11, 40], device="cuda"), packed=packed)
    grads = torch.autograd.grad([h, last], leaves, [g.cuda(), gl.cuda()])
    _check(want, h, last, grads, torch.float32, (50, 24))
    for t in (h, grads[0], grads[1]):
        assert not t[:4].any() and not t[40:].any()
    # no sequence at all: every row is zero
    h, last = gb.gated_scan(leaves[0].detach(), leaves[1].detach(), None, torch.zeros(1, dtype=torch.long, device="cuda"))
    assert not h.any() and last.shape == (0, 24)


def test_offsets_out_of_place_touch_nothing_outside():
    """What no caller should pass: the kernels take the nearest possible offsets. Checked for staying inside the rows."""
    import gridnet_b200 as gb

    z, u, h0, g, gl = _inputs(4, 300, 3, 8, torch.float32)
    for bad in ([0, 400, 500, 1 << 40], [-5, 10, 20, 300], [0, 200, 100, 300]):
        around = [torch.full((340, 8), 7.0, device="cuda") for _ in range(2)]
        for t, v in zip(around, (z, u)):
            t[20:320] = v.cuda()
        leaves = [around[0][20:320].requires_grad_(True), around[1][20:320].requires_grad_(True), h0.cuda().requires_grad_(True)]
        h, last = gb.gated_scan(*leaves, torch.tensor(bad, device="cuda"))
        torch.autograd.grad([h, last], leaves, [g.cuda(), gl.cuda()])
        assert all((t[:20] == 7).all() and (t[320:] == 7).all() for t in around)
    # one sequence that is cut at the last row
    h, last = gb.gated_scan(z.cuda(), u.cuda(), h0[:1].cuda(), torch.tensor([0, 1 << 40], device="cuda"))
    assert_within(h, *scan_all(z.double(), u.double(), h0[:1].double(), [(0, 300)])["h"], "h")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides(dtype):
    """Halves of one projection, transposed batches, a broadcast gate, odd addresses."""
    import gridnet_b200 as gb

    kind, B, T, D = TYPES[dtype], 3, 37, 24
    gen = torch.Generator().manual_seed(1)
    both = (torch.randn(B, T, 2 * D, generator=gen) * 2).to(kind)
    late = (torch.randn(T, B, D, generator=gen) * 2).to(kind)
    odd = torch.randn(B * T * D + 1, generator=gen).to(kind)
    side = (torch.randn(B, T, D, 2, generator=gen)).to(kind)
    d = lambda t: t.cuda()  # noqa: E731
    pairs = [(d(both).chunk(2, -1)), (d(late).transpose(0, 1), d(both)[..., 1:D + 1]), (d(late)[:1].transpose(0, 1).expand(B, T, D), d(odd)[1:].view(B, T, D)),
             (d(side)[..., 0], d(side)[..., 1])]
    for z, u in pairs:
        got, last = gb.gated_scan(z, u)
        want = scan_all(z.cpu().double().reshape(B * T, D), u.cpu().double().reshape(B * T, D), torch.zeros(B, D, dtype=torch.float64),
                        [(i * T, i * T + T) for i in range(B)])
        assert_within(got.reshape(B * T, D), *want["h"], "h", kind)
        assert_within(last, *want["last"], "last")
    # gradients through a projection's halves and a broadcast gate (its gradients add up)
    for packed in (False, True):
        x = d(both).requires_grad_(True)
        h, _ = gb.gated_scan(*x.chunk(2, -1), packed=packed)
        c, w = d(both[..., :D]).contiguous().requires_grad_(True), d(both[..., D:]).contiguous().requires_grad_(True)
        h2, _ = gb.gated_scan(c, w, packed=packed)
        assert torch.equal(h, h2)
        up = torch.randn(B, T, D, generator=gen).to(kind).cuda()
        gx, (gc, gw) = torch.autograd.grad(h, x, up)[0], torch.autograd.grad(h2, (c, w), up)
        assert torch.equal(gx[..., :D], gc) and torch.equal(gx[..., D:], gw)
    one = d(both[:, :, :1]).requires_grad_(True)
    h, _ = gb.gated_scan(one.expand(B, T, D), w)
    full = one.detach().expand(B, T, D).contiguous().requires_grad_(True)
    h2, _ = gb.gated_scan(full, w)
    assert torch.equal(torch.autograd.grad(h, one, up)[0], torch.autograd.grad(h2, full, up)[0].sum(-1, keepdim=True))
    # a gradient that is a view
    wide = torch.randn(B, T, 2 * D, generator=gen).to(kind).cuda()
    h, _ = gb.gated_scan(c, w)
    a = torch.autograd.grad(h, c, wide[..., :D])[0]
    h, _ = gb.gated_scan(c, w)
    assert torch.equal(a, torch.autograd.grad(h, c, wide[..., :D].contiguous())[0])


def test_more_dimensions_and_missing_parts():
    """Grids as steps; no state, no gradient of h or of last; outputs that do not depend on whether gradients are kept."""
    import gridnet_b200 as gb

    B, T, grid = 2, 11, (4, 8, 12)
    z, u, h0, g, gl = (t.cuda() for t in _inputs(5, B * T, B, 384, torch.float32))
    z5, u5 = z.view(B, T, *grid).requires_grad_(True), u.view(B, T, *grid).requires_grad_(True)
    h, last = gb.gated_scan(z5, u5, h0.view(B, *grid))
    h2, last2 = gb.gated_scan(z.detach().view(B, T, 384), u.detach().view(B, T, 384), h0)
    assert h.shape == (B, T, *grid) and last.shape == (B, *grid)
    assert torch.equal(h.view(B, T, 384), h2) and torch.equal(last.view(B, 384), last2)
    only_last = torch.autograd.grad(last, (z5, u5), gl.view(B, *grid), retain_graph=True)
    with_zeros = torch.autograd.grad([h, last], (z5, u5), [torch.zeros_like(h), gl.view(B, *grid)], retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(only_last, with_zeros))
    only_h = torch.autograd.grad(h, z5, g.view(B, T, *grid), retain_graph=True)[0]
    zero_last = torch.autograd.grad([h, last], z5, [g.view(B, T, *grid), torch.zeros_like(last)])[0]
    assert torch.equal(only_h, zero_last)
    # without a state: zeros
    a, b = gb.gated_scan(z5.detach(), u5.detach()), gb.gated_scan(z5.detach(), u5.detach(), torch.zeros(B, *grid, device="cuda"))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    # no steps: the state comes back, and so does its gradient
    s = h0.clone().requires_grad_(True)
    h, last = gb.gated_scan(torch.empty(B, 0, 384, device="cuda"), torch.empty(B, 0, 384, device="cuda"), s)
    assert h.shape == (B, 0, 384) and torch.equal(last, h0) and torch.equal(torch.autograd.grad(last, s, gl)[0], gl)
    h, last = gb.gated_scan(torch.empty(0, 5, 8, device="cuda"), torch.empty(0, 5, 8, device="cuda"))
    assert h.shape == (0, 5, 8) and last.shape == (0, 8)


def test_what_is_not_finite_stays_until_a_reset():
    import gridnet_b200 as gb

    T = 700
    z = torch.zeros(1, T, 4)
    u = torch.ones(1, T, 4)
    u[0, 3, 0], u[0, 3, 1] = float("nan"), float("inf")
    z[0, 500, 0] = float("-inf")
    z[0, 2, 2] = float("nan")
    h, last = gb.gated_scan(z.cuda(), u.cuda())
    h = h.cpu()[0]
    assert h[:3, 0].isfinite().all() and not h[3:500, 0].isfinite().any() and h[500:, 0].isfinite().all()
    assert h[:3, 1].isfinite().all() and not h[3:, 1].isfinite().any()
    assert h[:2, 2].isfinite().all() and not h[2:, 2].isfinite().any()
    assert h[:, 3].isfinite().all() and not last[0, 1:3].cpu().isfinite().any()


def test_hold_is_exact():
    """10000 held steps leave the state's bits alone."""
    import gridnet_b200 as gb

    s = torch.randn(2, 12, generator=torch.Generator().manual_seed(0)).cuda()
    z = torch.full((2, 10000, 12), float("inf"), device="cuda")
    h, last = gb.gated_scan(z, torch.full_like(z, float("nan")), s)
    assert torch.equal(last, s) and torch.equal(h, s[:, None].expand_as(h))


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 1024), (7, 33), (513, 132)])
def test_step(rows, width, dtype):
    """One step, in place and not, from the halves of a projection; a sequence step by step is the sequence at once."""
    import gridnet_b200 as gb

    kind = TYPES[dtype]
    z, u, h0, _, _ = _inputs(rows + width, rows, rows, width, kind)
    z[:, 0], u[:, 0] = float("inf"), float("nan")
    want = scan_all(z.double(), u.double(), h0.double(), [(i, i + 1) for i in range(rows)])
    both = torch.cat([z, u], 1).cuda()
    for args in ((z.cuda(), u.cuda()), both.chunk(2, 1)):
        state = h0.cuda()
        h, new = gb.gated_scan_step(*args, state)
        assert torch.equal(state, h0.cuda()) and h.dtype == kind
        assert_within(h, *want["h"], "h", kind)
        assert_within(new, *want["last"], "state")
        h2, same = gb.gated_scan_step(*args, state, out_state=state)
        assert same is state and torch.equal(same, new) and torch.equal(h, h2)


def test_step_by_step_is_the_scan():
    import gridnet_b200 as gb

    z, u, h0, _, _ = (t.cuda() for t in _inputs(9, 3 * 20, 3, 40, torch.float32))
    z, u = z.view(3, 20, 40), u.view(3, 20, 40)
    h, last = gb.gated_scan(z, u, h0)
    state = h0.clone()
    rows = [gb.gated_scan_step(z[:, t], u[:, t], state, state)[0] for t in range(20)]
    want = scan_all(z.reshape(60, 40).cpu().double(), u.reshape(60, 40).cpu().double(), h0.cpu().double(), [(20 * i, 20 * i + 20) for i in range(3)])
    assert_within(torch.stack(rows, 1).reshape(60, 40), *want["h"], "steps")
    assert_within(h.reshape(60, 40), *want["h"], "scan")
    assert_within(state, *want["last"], "state")
    assert_within(last, *want["last"], "last")


@pytest.mark.parametrize("packed", [False, True])
def test_gradient_against_differences(packed):
    """The sum of w h + v last along a direction, from the kernel's outputs on both sides. 2^-5 is the step; what a difference of that step is
    off by is taken from the definition in float64, rounding by the bound on the outputs."""
    import gridnet_b200 as gb

    T, D, eps = 150, 12, 2.0 ** -5
    z, u, h0, w, v = _inputs(21, T, 1, D, torch.float32)
    if packed:  # at values that the packed copy holds as they are
        z, u = (torch.from_numpy(pack(t.numpy())[2]).float() for t in (z, u))
    dirs = [torch.randn(t.shape, generator=torch.Generator().manual_seed(i)).sign() for i, t in enumerate((z, u, h0))]
    leaves = [t.cuda().requires_grad_(True) for t in (z[None], u[None], h0)]
    grads = torch.autograd.grad(gb.gated_scan(*leaves, packed=packed), leaves, [w[None].cuda(), v.cuda()])
    slope = sum((g.cpu().double().reshape(d.shape) * d).sum() for g, d in zip(grads, dirs))

    def plain(sign):
        out = scan(*(t.double() + sign * eps * d for t, d in zip((z, u), dirs)), (h0.double() + sign * eps * dirs[2])[0])
        at = (out["h"][0] * w).sum() + (out["last"][0] * v[0]).sum()
        return at, (out["h"][1] * w.abs()).sum() + (out["last"][1] * v[0].abs()).sum()

    def kernel(sign):
        with torch.no_grad():
            h, last = gb.gated_scan(*((t + sign * eps * d.view(t.shape).cuda()) for t, d in zip(leaves, dirs)))
        return (h[0].cpu().double() * w).sum() + (last[0].cpu().double() * v[0]).sum()

    (up, eup), (down, edown) = plain(1), plain(-1)
    exact = scan(z.double(), u.double(), h0.double()[0], w.double(), v.double()[0])
    true = sum((exact[k][0].reshape(d.shape) * d).sum() for k, d in zip(("gate", "value", "state"), dirs))
    off = abs((up - down) / (2 * eps) - true) + (eup + edown) / (2 * eps)
    # moved inputs are rounded to float32: half a step of at most 16 each
    off = off + sum(16 * U * exact[k][0].abs().sum() for k in ("gate", "value", "state")) / eps
    own = sum(exact[k][1].sum() for k in ("gate", "value", "state"))
    assert off < 0.05 * abs(true), "the differences say something"
    assert abs((kernel(1) - kernel(-1)) / (2 * eps) - slope) <= off + own


def test_captured_replayed_and_on_another_stream():
    """Forward and backward in one graph, replayed on new inputs, and eagerly on a second stream: the same bits."""
    import gridnet_b200 as gb

    make = lambda seed: [t.cuda() for t in _inputs(seed, 4 * 300, 4, 64, torch.float32)]  # noqa: E731

    def run(z, u, h0, g, gl, packed):
        z, u, h0 = (t.detach().requires_grad_(True) for t in (z, u, h0))
        h, last = gb.gated_scan(z.view(4, 300, 64), u.view(4, 300, 64), h0, packed=packed)
        return [h, last, *torch.autograd.grad([h, last], (z, u, h0), [g.view(4, 300, 64), gl])]

    for packed in (False, True):
        static = make(1)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(*static, packed)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run(*static, packed)
        for seed in (2, 3):
            new = make(seed)
            for a, b in zip(static, new):
                a.copy_(b)
            graph.replay()
            want = run(*new, packed)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                beside = run(*new, packed)
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) and torch.equal(b, c) for a, b, c in zip(outs, want, beside))


@pytest.mark.parametrize("shape,ragged", [((2, 2100, 40), None), ((1, 3000, 72), [0, 5, 5, 1900, 3000]), ((160, 300, 64), None)])
def test_captured_by_chunks_and_as_a_walk(shape, ragged):
    """Long sequences in three kernels, many in one: replayed twice in a row, the second time on other inputs."""
    import gridnet_b200 as gb

    gen = torch.Generator().manual_seed(5)
    total = shape[0] * shape[1]
    offsets = None if ragged is None else torch.tensor(ragged, device="cuda")
    kind = shape if ragged is None else (total, shape[2])
    n = shape[0] if ragged is None else len(ragged) - 1
    make = lambda: [torch.randn(*s, generator=gen).cuda() for s in (kind, kind, (n, shape[2]), kind, (n, shape[2]))]  # noqa: E731

    def run(z, u, h0, g, gl, packed):
        z, u, h0 = (t.detach().requires_grad_(True) for t in (z, u, h0))
        h, last = gb.gated_scan(z, u, h0, offsets, packed=packed)
        return [h, last, *torch.autograd.grad([h, last], (z, u, h0), [g, gl])]

    for packed in (False, True):
        static, new = make(), make()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(*static, packed)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run(*static, packed)
        graph.replay()
        for a, b in zip(static, new):
            a.copy_(b)
        graph.replay()
        want = run(*new, packed)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("n,steps", [(1, 600000), (4, 150000)])
def test_places_past_32_bits(n, steps):
    """2.4e9 values, as chunks and as a walk: the last sequence's end, behind a reset, is what the end alone is."""
    import gridnet_b200 as gb

    width, tail = 4096, 200
    z = torch.zeros(n, steps, width, dtype=torch.bfloat16, device="cuda")
    u = torch.ones_like(z)
    g = torch.zeros_like(z)
    z[-1, -tail:], u[-1, -tail:], g[-1, -tail:] = (torch.randn(tail, width, device="cuda") for _ in range(3))
    z[-1, -tail] = float("-inf")
    for packed in (False, True):
        leaves, short = ([t.detach().requires_grad_(True) for t in pair] for pair in ((z, u), (z[-1:, -tail:].clone(), u[-1:, -tail:].clone())))
        h, last = gb.gated_scan(*leaves, packed=packed)
        grads = torch.autograd.grad(h, leaves, g)
        h2, last2 = gb.gated_scan(*short, packed=packed)
        grads2 = torch.autograd.grad(h2, short, g[-1:, -tail:])
        # runs of steps are put together in other places: a few units of float32 each, then at most one step of bfloat16 apart
        for a, b in ((h[-1, -tail:], h2[0]), *((x[-1, -tail:], y[0]) for x, y in zip(grads, grads2))):
            assert ((a.float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + 1e-6).all()
        assert torch.allclose(last[-1], last2[0], rtol=1e-5, atol=1e-5)
        assert (h[0, 1000].float() - 1).abs().max() < 1e-2 or n == 1
        del h, last, grads, leaves
    del z, u, g


def test_the_same_bits_every_time_and_two_graphs_alive():
    import gridnet_b200 as gb

    z, u, h0, g, gl = (t.cuda() for t in _inputs(8, 2000, 1, 96, torch.bfloat16))
    z, u = z[None].requires_grad_(True), u[None].requires_grad_(True)
    for packed in (False, True):
        first, second = gb.gated_scan(z, u, h0, packed=packed), gb.gated_scan(z, u, h0, packed=packed)
        b = torch.autograd.grad(second[0], (z, u), g[None])
        a = torch.autograd.grad(first[0], (z, u), g[None])
        assert torch.equal(first[0], second[0]) and all(torch.equal(x, y) for x, y in zip(a, b))
        # inputs changed in place between the passes: torch refuses, or the packed copy is what was
        h, _ = gb.gated_scan(z, u, h0, packed=packed)
        with torch.no_grad():
            z.add_(0)
        if packed:
            assert torch.equal(torch.autograd.grad(h, u, g[None])[0], a[1])
        else:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(h, u, g[None])


def test_second_derivatives_are_refused():
    import gridnet_b200 as gb

    z = torch.randn(1, 5, 4, device="cuda", requires_grad=True)
    h, _ = gb.gated_scan(z, z.detach())
    (gz,) = torch.autograd.grad(h.sum(), z, create_graph=True)
    with pytest.raises(RuntimeError):
        gz.sum().backward()


def test_layer():
    """GatedRecurrence: the projection's halves through the scan, and the same layer one step at a time."""
    import gridnet_b200 as gb

    torch.manual_seed(0)
    layer = gb.GatedRecurrence(20, 32, "cuda")
    assert layer.proj.bias[:32].eq(1).all()
    x = torch.randn(3, 9, 20, device="cuda")
    h, last = layer(x)
    z, u = layer.proj(x).double().cpu().detach().reshape(27, 64).chunk(2, -1)
    want = scan_all(z, u, torch.zeros(3, 32, dtype=torch.float64), [(9 * i, 9 * i + 9) for i in range(3)])
    assert_within(h.reshape(27, 32), *want["h"], "h")
    h.sum().backward()
    assert layer.proj.weight.grad.isfinite().all() and layer.proj.weight.grad.abs().sum() > 0
    state = torch.zeros(3, 32, device="cuda")
    for t in range(9):
        out, state = layer.step(x[:, t], state, state)
    # a matrix product of other sizes may add up in another order: a few units of 20 products each, through 9 steps
    assert torch.allclose(state, last, rtol=1e-4, atol=1e-4)
