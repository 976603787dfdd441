"""Scans with so many tiles that a CTA has several of them one after the other, of one sequence and the next; and the other ways to go at sizes where
they are chosen by the number of CTAs. Against the definition in float64."""
import numpy as np
import pytest
import torch

from plain_scan import assert_within, pack, scan, scan_all

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _packed(t):
    """What the packed copy of [rows, width] stands for, in float64, a row's groups at a time."""
    x = t.double()
    rows, width = x.shape
    groups = (width + 31) // 32
    x = torch.nn.functional.pad(x, (0, 32 * groups - width)).view(rows, groups, 32)
    finite = x.isfinite()
    top = x.abs().masked_fill(~finite, 0).amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(top)  # top = mantissa * 2^exponent, mantissa in [1/2, 1)
    e = (exponent - 7 + (mantissa > 125 / 128)).clamp(min=-126)
    held = torch.where(finite, torch.ldexp(torch.round(torch.ldexp(x, -e)), e), x)
    return held.view(rows, -1)[:, :width]


def test_packing_by_groups_is_packing_by_values():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(40, 71, generator=g) * torch.exp2(torch.randint(-30, 30, (40, 1), generator=g).float())
    x[3, 4], x[3, 40], x[5] = float("inf"), float("nan"), 0
    x[7, :4] = torch.tensor([125.0, 124.5, -62.5, 3.5])
    assert np.array_equal(_packed(x).numpy(), pack(x.numpy())[2], equal_nan=True)


def _lengths(seed, n, total):
    """Lengths that add up to total: some sequences empty, some of whole tiles, most of neither."""
    r = np.random.default_rng(seed)
    lengths = r.multinomial(total - 64 * 3, r.dirichlet(np.full(n, 0.7)))
    lengths[1::9] = 0
    lengths[:3] += 64
    lengths[-1] += total - lengths.sum()
    return lengths.tolist()


def _compare(gb, z, u, h0, g, gl, offsets, n, packed, want):
    dtype, width = z.dtype, z.shape[-1]
    shape = z.shape if offsets is not None else (n, z.shape[0] // n, width)
    leaves = [t.cuda().requires_grad_(True) for t in (z.view(shape), u.view(shape), h0)]
    h, last = gb.gated_scan(*leaves, offsets, packed=packed)
    grads = torch.autograd.grad([h, last], leaves, [g.view(shape).cuda(), gl.cuda()])
    for name, got in (("h", h), ("gate", grads[0]), ("value", grads[1]), ("last", last), ("state", grads[2])):
        rows = got.reshape(-1, width)
        assert_within(rows, *want[name], name, dtype if name in ("h", "gate", "value") else torch.float32)


def _inputs(seed, total, n, width, dtype):
    gen = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    z = make(total, width) * 2 + 1.5 + make(width)
    z[torch.rand(total, generator=gen) < 0.02] = float("inf")
    z[torch.rand(total, generator=gen) < 0.01, :7] = float("-inf")
    return z.to(dtype), make(total, width).to(dtype), make(n, width), make(total, width).to(dtype), make(n, width)


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
# 16 slabs; rows of tiles are total / 32 + n + 1 backward and total / 64 + n + 1 forward. 60 sequences: 4 tiles to a CTA backward; 290: 8 backward
# and 2 forward, whatever ends inside a CTA
@pytest.mark.parametrize("n,total", [(60, 8000), (290, 10500)])
def test_ragged_tiles_of_several_sequences_in_a_cta(n, total, dtype, packed):
    import gridnet_b200 as gb

    width = 1000
    z, u, h0, g, gl = _inputs(n, total, n, width, TYPES[dtype])
    ends = np.concatenate([[0], np.cumsum(_lengths(n, n, total))]).tolist()
    assert ends[-1] == total and all(a <= b for a, b in zip(ends, ends[1:]))
    spans = list(zip(ends, ends[1:]))
    out = scan_all(z.double(), u.double(), h0.double(), spans)
    zz, uu = (_packed(z), _packed(u)) if packed else (z.double(), u.double())
    back = scan_all(zz, uu, h0.double(), spans, g.double(), gl.double())
    want = {**back, "h": out["h"], "last": out["last"]}
    _compare(gb, z, u, h0, g, gl, torch.tensor(ends, device="cuda"), n, packed, want)


def _dense_want(z, u, h0, g, gl, n, packed):
    """Channels are apart, so all sequences are channels of one."""
    total, width = z.shape
    steps = total // n
    side = lambda t: t.double().view(n, steps, width).transpose(0, 1).reshape(steps, n * width)  # noqa: E731
    back = lambda t: t.view(steps, n, width).transpose(0, 1).reshape(total, width)  # noqa: E731
    out = scan(side(z), side(u), h0.double().reshape(-1))
    zz, uu = (side(_packed(z)), side(_packed(u))) if packed else (side(z), side(u))
    grads = scan(zz, uu, h0.double().reshape(-1), side(g), gl.double().reshape(-1))
    both = {**grads, "h": out["h"], "last": out["last"]}
    return {k: tuple(t.view(n, width) if k in ("last", "state") else back(t) for t in v) for k, v in both.items()}


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
# 17 tiles of 32 to a sequence, two to a CTA: every other sequence starts inside one; more CTAs than SMs: a walk of many tiles
@pytest.mark.parametrize("n,steps,width,dtype", [(9, 539, 1000, "bf16"), (9, 539, 1000, "f32"), (160, 300, 64, "f32"), (40, 600, 256, "f16")])
def test_dense_tiles_and_walks(n, steps, width, dtype, packed):
    import gridnet_b200 as gb

    z, u, h0, g, gl = _inputs(steps + width, n * steps, n, width, TYPES[dtype])
    _compare(gb, z, u, h0, g, gl, None, n, packed, _dense_want(z, u, h0, g, gl, n, packed))


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
def test_ragged_walk(packed):
    """32 CTAs per SM and more than eight tiles of rows: ragged sequences as walks."""
    import gridnet_b200 as gb

    width, total = 512, 4000
    n = 32 * torch.cuda.get_device_properties(0).multi_processor_count // (width // 64) + 1
    z, u, h0, g, gl = _inputs(7, total, n, width, torch.float32)
    ends = np.concatenate([[0], np.cumsum(_lengths(7, n, total))]).tolist()
    assert max(b - a for a, b in zip(ends, ends[1:])) > 64 and ends[-1] == total
    spans = list(zip(ends, ends[1:]))
    out = scan_all(z.double(), u.double(), h0.double(), spans)
    zz, uu = (_packed(z), _packed(u)) if packed else (z.double(), u.double())
    want = {**scan_all(zz, uu, h0.double(), spans, g.double(), gl.double()), "h": out["h"], "last": out["last"]}
    _compare(gb, z, u, h0, g, gl, torch.tensor(ends, device="cuda"), n, packed, want)
