"""The gated scan and the packed copies from their definitions, in float64 on the CPU, step by step and value by value, and how far
float32 may be from them."""
import numpy as np
import torch

U = 2.0 ** -24  # half a step of float32


def pack(x, cols_from=1):
    """(codes, scales, values) of a numpy array, groups of 32 along what is behind the first ``cols_from`` dimensions."""
    shape = x.shape
    rows = int(np.prod(shape[:cols_from], dtype=np.int64))
    flat = np.asarray(x, np.float64).reshape(rows, int(np.prod(shape[cols_from:], dtype=np.int64)))
    cols = flat.shape[1]
    groups = (cols + 31) // 32
    codes, scales, values = np.zeros((rows, cols), np.int8), np.zeros((rows, groups), np.uint8), np.zeros((rows, cols))
    for r in range(rows):
        for g in range(groups):
            part = flat[r, 32 * g:32 * g + 32]
            finite = np.isfinite(part)
            top = np.abs(part[finite]).max(initial=0.0)
            e = -126
            while top > 125 * 2.0 ** e:
                e += 1
            scales[r, g] = e + 127
            for i, v in enumerate(part):
                at = r, 32 * g + i
                if np.isnan(v):
                    codes[at], values[at] = -128, np.nan
                elif np.isinf(v):
                    codes[at], values[at] = (127 if v > 0 else -127), v
                else:
                    codes[at] = np.clip(np.rint(v / 2.0 ** e), -63 if e == 122 else -125, 63 if e == 122 else 125)  # 64 * 2^122 is no float
                    values[at] = codes[at] * 2.0 ** e
    return codes.reshape(shape), scales.reshape(*shape[:cols_from], groups), values.reshape(shape)


def scan(z, u, h0, g=None, gl=None):
    """One sequence [steps, width] of float64 tensors. Returns {name: (value, how far float32 may be from it)}.

    A gate has eight units of U of its own: exp 4 (two units in the last place), 1 + e one, the reciprocal two, the product one. Putting
    steps together adds a rounding per product, per sum and per level of the three levels at most: sixteen units of U in all, each of the
    sum of the magnitudes of what is added, which obeys the same recurrence. So the error obeys it too.

    The exponential's argument is a product z log2(e) rounded to float32, |z log2(e)| U off, with a factor that is itself off by a
    quarter U: together no more than z being 1.3 |z| U off. A gate moved by d changes a by a n d, n by -a n d."""
    a, n = torch.sigmoid(z), torch.sigmoid(-z)
    term = torch.where(n == 0, 0.0, n * u)
    T = z.shape[0]
    moved = torch.where(z.isinf(), 0.0, 1.3 * U * z.abs())
    h, mag, err = h0.clone(), h0.abs(), torch.zeros_like(h0)
    before, hs, hmag, herr = [], [], [], []
    for t in range(T):
        before.append((h, mag, err))
        reset = a[t] == 0
        move = torch.where((a[t] * n[t] == 0), 0.0, a[t] * n[t] * moved[t] * (mag + u[t].abs()))
        h = torch.where(reset, term[t], a[t] * h + term[t])
        mag = torch.where(reset, term[t].abs(), a[t] * mag + term[t].abs())
        err = torch.where(reset, 0.0, a[t] * err) + 16 * U * mag + move
        hs.append(h)
        hmag.append(mag)
        herr.append(err)
    out = {"last": (h, err)}
    stack = lambda xs: torch.stack(xs) if xs else z.new_zeros(0, z.shape[1])  # noqa: E731
    out["h"] = (stack(hs), stack(herr))
    if g is None:
        return out
    c, cmag, cerr = gl.clone(), gl.abs(), torch.zeros_like(gl)
    dzs, dus = [], []
    for t in reversed(range(T)):
        dh, dmag = g[t] + c, g[t].abs() + cmag
        derr = cerr + U * dmag
        hb, hbm, hbe = before[t]
        w = a[t] * n[t]
        d = torch.where(w == 0, 0.0, hb - u[t])
        dmagn = torch.where(w == 0, 0.0, hbm + u[t].abs())
        # w = 0: the gradient is 0 by definition, with nothing to round, also where the state (and so its bound) is not finite
        dzs.append((torch.where(w == 0, 0.0, w * d * dh), torch.where(w == 0, 0.0, w * (dmagn * (derr + (20 * U + moved[t]) * dmag) + hbe * dmag))))
        dus.append((n[t] * dh, n[t] * (derr + (10 * U + moved[t]) * dmag)))
        c, cmag = torch.where(a[t] == 0, 0.0, a[t] * dh), torch.where(a[t] == 0, 0.0, a[t] * dmag)
        cerr = torch.where(a[t] == 0, 0.0, a[t] * derr) + 16 * U * cmag + n[t] * moved[t] * cmag
    for name, xs in (("gate", dzs), ("value", dus)):
        out[name] = stack([v for v, _ in xs[::-1]]), stack([e for _, e in xs[::-1]])
    out["state"] = c, cerr
    return out


def scan_all(z, u, h0, spans, g=None, gl=None):
    """Over rows [total, width] with a (start, end) per sequence; rows of none of them: zeros."""
    out = {}
    for i, (lo, hi) in enumerate(spans):
        part = scan(z[lo:hi], u[lo:hi], h0[i], None if g is None else g[lo:hi], None if g is None else gl[i])
        for name, (v, e) in part.items():
            if name not in out:
                shape = (len(spans) if name in ("last", "state") else z.shape[0], z.shape[1])
                out[name] = torch.zeros(shape, dtype=torch.float64), torch.zeros(shape, dtype=torch.float64)
            at = i if name in ("last", "state") else slice(lo, hi)
            out[name][0][at], out[name][1][at] = v, e
    return out


def assert_within(got, want, tol, what, dtype=torch.float32):
    """``tol`` plus half a step of the output's type, and of the smallest number that it tells apart."""
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if dtype != torch.float32:
        tol = tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol)
    tol = tol + (2.0 ** -25 if dtype == torch.float16 else 1e-37)
    bad = ~((got - want).abs() <= tol) & ~(got.isnan() & want.isnan()) & ~((got == want) & want.isinf())
    if bad.any():
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {i}: {got[i]!r}, want {want[i]!r} +- {tol[i]:.3e}")
