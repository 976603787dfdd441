"""Steps, loops and models that keep 8-bit copies between their passes. Their gradients are those of the calls that keep float32, given inputs that
are what the copies stand for: the same kernels on the same numbers, so the same bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture()
def packed():
    import gridnet_b200 as gb

    gb.keep_packed(True)
    yield
    gb.keep_packed(False)
    gb.keep_forward_stash(None)


def _rounded(x, rows=1):
    import gridnet_b200 as gb

    return gb.unpack_activations(gb.pack_activations(x, rows))


def _params(shape, gated=False, n=1, seed=0):
    g = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    if gated:
        return [(0.2 * make(27, 2, *shape), 0.1 * make(2, *shape))]
    return [(0.2 * make(27, *shape), 0.1 * make(*shape), 1 + 0.1 * make(*shape)) for _ in range(n)]


@pytest.mark.parametrize("B,shape,block,normalize", [(3, (16, 8, 24), 8, False), (64, (16, 16, 16), 8, True), (5, (8, 8, 8), 4, False), (130, (16, 16, 8), 4, True),
                                                     (2, (12, 4, 20), 4, True)])
def test_step(packed, B, shape, block, normalize):
    import gridnet_b200 as gb

    (w, b, s), x, g = _params(shape)[0], torch.randn(B, *shape, device="cuda"), torch.randn(B, *shape, device="cuda")

    def run(x):
        leaves = [t.detach().requires_grad_(True) for t in (w, b, s, x)]
        y = gb.GridnetCudaOp.apply(*leaves, 2, block, 1e-5, normalize, "silu")
        return y.detach(), torch.autograd.grad(y, leaves, g)

    y, grads = run(x)
    gb.keep_packed(False)
    gb.keep_forward_stash(False)
    assert torch.equal(run(x)[0], y)
    want = run(_rounded(x))[1]
    # blocks of 4 with normalisation, small batches: the general kernel adds up by atomics, in another order every time
    ordered = not normalize or block == 8
    for a, c in zip(grads, want):
        assert torch.equal(a, c) if ordered else torch.allclose(a, c, rtol=1e-4, atol=1e-5 * c.abs().max().item())


@pytest.mark.parametrize("block", [8, 4])
def test_gated_step(packed, block):
    import gridnet_b200 as gb

    shape = (16, 8, 16)
    (w, b), x, g = _params(shape, gated=True)[0], torch.randn(5, *shape, device="cuda"), torch.randn(5, *shape, device="cuda")

    def run(x):
        leaves = [t.detach().requires_grad_(True) for t in (w, b, x)]
        y = gb.GatedGridnetCudaOp.apply(*leaves, 2, block, "tanh")
        return y.detach(), torch.autograd.grad(y, leaves, g)

    y, grads = run(x)
    gb.keep_packed(False)
    assert torch.equal(run(x)[0], y)
    want = run(_rounded(x))[1]
    # block 4 adds up with atomics of shared memory where a CTA has them: sums of at most 27 x 2 x 5 products
    assert all(torch.equal(a, c) if block == 8 else torch.allclose(a, c, rtol=1e-4, atol=1e-5) for a, c in zip(grads, want))


def _rounded_il4(t, Q, P):
    """An IL4 tensor ([Q][P][4]) as its packed copy gives it: groups of 32 positions of a sample."""
    v = t.view(torch.float32).view(Q, P, 4).permute(0, 2, 1).contiguous()
    t.view(torch.float32).view(Q, P, 4).copy_(_rounded(v, 2).permute(0, 2, 1))


@pytest.mark.parametrize("kind", ["shared", "separate", "residual", "residual separate", "gated"])
@pytest.mark.parametrize("B,shape,block,outer", [(1, (16, 16, 16), 8, 1), (3, (8, 16, 24), 8, 3), (7, (16, 8, 8), 4, 4), (20, (32, 32, 32), 8, 2)])
def test_loop(packed, kind, B, shape, block, outer):
    import gridnet_b200 as gb
    from gridnet_b200 import backend_cuda as bc

    gated, residual = kind == "gated", kind.startswith("residual")
    block = 8 if gated else block
    plist = _params(shape, gated, outer if "separate" in kind else 1)
    gen = torch.Generator().manual_seed(3)
    ga, be = (1 + 0.1 * torch.randn(shape, generator=gen)).cuda(), (0.1 * torch.randn(shape, generator=gen)).cuda()
    x, g = torch.randn(B, *shape, generator=gen).cuda(), torch.randn(B, *shape, generator=gen).cuda()
    act = "tanh" if gated else "silu"
    args = (plist, ga, be, x, 2, outer, block, act, 1e-5, residual)
    y, saved = bc._loop_forward(*args, True, gated)
    assert isinstance(saved, bc._PackedLoop)
    got = bc._loop_backward(plist, ga, be, saved, g, 2, outer, block, act, residual, gated)
    gb.keep_packed(False)
    gb.keep_forward_stash(False)
    y2, pool = bc._loop_forward(*args, True, gated)
    assert torch.equal(y, y2)
    x_il4, stats, outs, stashes = pool
    Q, P = (B + 3) // 4, shape[0] * shape[1] * shape[2]
    for t in (x_il4, *outs):
        _rounded_il4(t, Q, P)
    want = bc._loop_backward(plist, ga, be, pool.pieces(), g, 2, outer, block, act, residual, gated)
    for a, c in zip([*(t for p in got[0] for t in p), *got[1:]], [*(t for p in want[0] for t in p), *want[1:]]):
        assert a.isfinite().all() and torch.equal(a, c)


def test_loop_with_what_is_not_finite_in_one_sample(packed):
    """A sample's infinities and NaN stay that sample's: gradients of the others' inputs are what they are without it."""
    import gridnet_b200 as gb
    from gridnet_b200 import backend_cuda as bc

    shape, B = (8, 8, 16), 4
    plist = _params(shape)
    ga, be = torch.ones(shape, device="cuda"), torch.zeros(shape, device="cuda")
    x, g = torch.randn(B, *shape, device="cuda"), torch.randn(B, *shape, device="cuda")
    bad = x.clone()
    bad[2, 3, 3, 3], bad[2, 1, 1, 1] = float("nan"), float("inf")
    grads = []
    for v in (x, bad):
        y, saved = bc._loop_forward(plist, ga, be, v, 2, 2, 8, "silu", 1e-5, False, True)
        grads.append(bc._loop_backward(plist, ga, be, saved, g, 2, 2, 8, "silu", False)[3])
    keep = [0, 1, 3]
    assert torch.equal(grads[0][keep], grads[1][keep]) and not grads[1][2].isfinite().all()


def test_loop_on_patches(packed):
    """A batch of one on a grid beyond 128^3: the register-patch kernels. The copies are in the grid's own layout."""
    import gridnet_b200 as gb
    from gridnet_b200 import backend_cuda as bc

    shape, outer = (136, 128, 128), 2
    assert bc.on_patches(1, *shape)
    plist = _params(shape)
    ga, be = torch.ones(shape, device="cuda"), torch.zeros(shape, device="cuda")
    x, g = torch.randn(1, *shape, device="cuda"), torch.randn(1, *shape, device="cuda")
    for residual in (False, True):
        gb.keep_packed(True)
        args = (plist, ga, be, x, 2, outer, 8, "silu", 1e-5, residual)
        y, saved = bc._loop_forward(*args, True)
        assert isinstance(saved, bc._PackedPatches)
        got = bc._loop_backward(plist, ga, be, saved, g, 2, outer, 8, "silu", residual)
        gb.keep_packed(False)
        gb.keep_forward_stash(False)
        y2, (px, stats, outs, stashes) = bc._loop_forward(*args, True)
        assert torch.equal(y, y2) and not any(s is not None for s in stashes)
        want = bc._loop_backward(plist, ga, be, (_rounded(px), stats, [_rounded(o) for o in outs], stashes), g, 2, outer, 8, "silu", residual)
        for a, c in zip([*got[0][0], *got[1:]], [*want[0][0], *want[1:]]):
            assert a.isfinite().all() and torch.equal(a, c)


def test_models_train_and_hold_a_quarter(packed):
    """A model with a recurrence over its frames, as it would be used: grid, read-out, gated scan, loss. With 8-bit copies the loop holds a quarter of
    its activations, outputs are the same, and the gradients point the same way."""
    import gridnet_b200 as gb

    torch.manual_seed(0)
    B, T, shape = 4, 8, (16, 16, 16)
    model = gb.GridnetModel(shape, 2, 4, 8, "cuda")
    readout = gb.Readout(shape, 48, "cuda")
    layer = gb.GatedRecurrence(48, 32, "cuda")
    head = torch.nn.Linear(32, 10, device="cuda")
    frames = torch.zeros(B * T, *shape, device="cuda")
    frames[..., 0] = torch.randn(B * T, *shape[:2], device="cuda")
    labels = torch.randint(10, (B,), device="cuda")
    modules = torch.nn.ModuleList([model, readout, layer, head])

    def run():
        modules.zero_grad(set_to_none=True)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        grid = model(frames)
        held = torch.cuda.memory_allocated() - before - grid.numel() * 4
        h, last = layer(readout(grid).view(B, T, 48))
        out = head(last)
        torch.nn.functional.cross_entropy(out, labels).backward()
        return out.detach(), held, [p.grad.clone() for p in modules.parameters()]

    run()
    out, held, grads = run()
    gb.keep_packed(False)
    gb.keep_forward_stash(False)
    out2, held2, grads2 = run()
    assert torch.equal(out, out2)
    assert held < 0.3 * held2, (held, held2)
    for a, b in zip(grads, grads2):
        assert a.isfinite().all()
        # one in 250 of a group's largest value at every step, which is a few per cent of a typical one
        assert torch.nn.functional.cosine_similarity(a.flatten(), b.flatten(), 0) > 0.95


def test_loop_captured(packed):
    import gridnet_b200 as gb

    shape, B = (16, 16, 16), 6
    plist = _params(shape)
    ga, be = torch.ones(shape, device="cuda"), torch.zeros(shape, device="cuda")
    x, g = torch.randn(B, *shape, device="cuda"), torch.randn(B, *shape, device="cuda")

    def run():
        leaves = [t.detach().requires_grad_(True) for t in (*plist[0], ga, be, x)]
        y = gb.FusedLoopTrainOp.apply(*leaves, 2, 3, 8, "silu", 1e-5)
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
        want = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(outs, want))
