"""The gated scan and the 8-bit activation checkpoints of this package as cases that can be timed, with their plain forms in
elementary torch operations.

A case is a dict of plain values; ``listed()`` names the fixed ones, ``draw(rng)`` gives more of the same ranges,
``prepare(case, seed)`` makes the inputs on the GPU, ``run(state)`` is one pass (through the package where ``own`` is true,
else the plain form), ``work(case)`` the bytes and operations that a pass cannot do without, ``exact(case, seed)`` what the
definitions give in 64 bits.

    scan   h_t = s(gate_t) h_{t-1} + s(-gate_t) value_t, s the logistic function; a step whose s(-gate_t) is 0 does not look at its value
    pack   groups of 32 values of a row share a power of two 2^e, the smallest with |value| <= 125 * 2^e for all finite ones and
           e >= -126; a value is held as value / 2^e rounded to a whole number (half to even); infinities and NaN are held as such
    norm   LayerNorm over the whole grid of a sample; the backward pass takes the input as its packed copy gives it
"""
import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _scan(name, kind, n, steps, width, dtype, packed=False, ragged=False):
    case = dict(kind=kind, n=n, steps=steps, width=width, dtype=dtype, packed=packed, ragged=ragged)
    return dict(case, name=name) if name else case


def _pack(name, rows, width, dtype):
    case = dict(kind="pack", rows=rows, width=width, dtype=dtype)
    return dict(case, name=name) if name else case


def _norm(name, batch, grid):
    case = dict(kind="norm", batch=batch, m=grid[0], n=grid[1], k=grid[2], dtype="f32")
    return dict(case, name=name) if name else case


def listed():
    return [
        # -- the recurrence one step at a time, as a program that answers while frames come in does
        # one stream, the plane of a 32^3 grid: launch and latency
        _scan("step one", "step", 1, 1, 1024, "f32"),
        # many streams at once, the plane of a 64^3 grid
        _scan("step batch", "step", 512, 1, 4096, "bf16"),
        # -- a whole sequence without gradients: one long recording, read at once
        _scan("read long", "read", 1, 65536, 256, "bf16"),
        # -- training: outputs, last state and all gradients
        # the smallest call worth a kernel: eight short clips
        _scan("train short", "train", 8, 16, 1024, "f32"),
        # an ordinary large batch
        _scan("train", "train", 8, 2048, 4096, "f32"),
        # clips of very different lengths end to end, some empty, with masked steps; a width that fills no vector evenly
        _scan("train ragged", "train", 37, 300, 1000, "bf16", ragged=True),
        # gate and value kept in 8 bits for the backward pass; a length one over a power of two
        _scan("train packed", "train", 4, 4097, 1024, "f32", packed=True),
        # -- packing and unpacking alone
        # the activations of the 64^3 network at its benchmark batch
        _pack("pack 64^3", 64, 64 * 64 * 64, "f32"),
        # rows that are odd in every way
        _pack("pack odd", 1003, 2049, "bf16"),
        # -- the whole-grid norm, forward and backward, with its input kept in 8 bits
        # the MNIST-shaped model's mini-batch
        _norm("norm 32^3", 8, (32, 32, 32)),
        # a grid that is not a cube, the odd last batch of a data set
        _norm("norm ragged", 37, (40, 56, 72)),
        # the ImageNet-shaped grid on the share of the batch that one of eight GPUs gets
        _norm("norm 128^3", 32, (128, 128, 128)),
    ]


def _log_int(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _width(rng, lo, hi):
    """Odd now and then, else a multiple of 4."""
    w = _log_int(rng, lo, hi)
    return w if rng.random() < 0.3 else max(4, w // 4 * 4)


def draw(rng):
    kind = rng.choice(["step", "read", "train", "train", "train", "pack", "norm", "norm"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind == "step":
        return _scan(None, kind, _log_int(rng, 1, 512), 1, _width(rng, 64, 4096), dtype)
    if kind == "pack":
        width = _width(rng, 64, 1 << 18)
        return _pack(None, _log_int(rng, 1, max(2, (1 << 24) // width)), width, dtype)
    if kind == "norm":
        grid = tuple(4 * _log_int(rng, 2, 32) for _ in range(3))
        return _norm(None, _log_int(rng, 1, max(2, min(128, (1 << 26) // (grid[0] * grid[1] * grid[2])))), grid)
    width = _width(rng, 16, 4096)
    steps = _log_int(rng, 1, max(2, min(65536, (1 << 25) // width)))
    n = _log_int(rng, 1, max(2, min(64, (1 << 25) // (width * steps))))
    return _scan(None, kind, n, steps, width, dtype, kind == "train" and rng.random() < 0.5, rng.random() < 0.4)


def _offsets(case, g):
    """Where ragged sequences start and end: lengths from 0 to three times the mean, empty ones among them."""
    n, total = case["n"], case["n"] * case["steps"]
    cuts = torch.rand(n - 1, generator=g)
    cuts[n // 2:n // 2 + n // 8] = cuts[n // 2:n // 2 + 1]  # equal cuts: sequences of no steps
    cuts = (cuts * (total + 1)).long().clamp_(max=total).sort().values
    return torch.cat([torch.zeros(1, dtype=torch.long), cuts, torch.full((1,), total)])


def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    dtype = _TYPES[case["dtype"]]
    g = torch.Generator(device=device).manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=g, device=device)  # noqa: E731
    state = {"case": case}
    if case["kind"] == "pack":
        # activations: rows of different scale, a few values far out
        x = randn(case["rows"], case["width"])
        x *= torch.exp(randn(case["rows"], 1))
        x *= torch.where(torch.rand(x.shape, generator=g, device=device) < 0.001, 20.0, 1.0)
        state["x"] = x.to(dtype)
        return state
    if case["kind"] == "norm":
        grid = (case["m"], case["n"], case["k"])
        state["x"] = (randn(case["batch"], *grid) * 1.5 + 0.2).requires_grad_(True)
        state["gamma"] = (1 + 0.1 * randn(*grid)).requires_grad_(True)
        state["beta"] = (0.1 * randn(*grid)).requires_grad_(True)
        state["grad"] = randn(case["batch"], *grid)
        return state
    n, steps, width = case["n"], case["steps"], case["width"]
    shape = (n, width) if case["kind"] == "step" else (n * steps, width) if case["ragged"] else (n, steps, width)
    # gates as a trained recurrence has them: memories from a step to a few hundred, by channel
    gate = randn(*shape) + 2.0 + 1.5 * randn(width)
    value = randn(*shape)
    if case["ragged"]:
        # masked steps: the state is held whatever the value says
        held = torch.rand(shape[0], generator=g, device=device) < 0.02
        gate[held] = float("inf")
        value[held] = float("nan")
        state["offsets"] = _offsets(case, torch.Generator().manual_seed(seed)).to(device)
    train = case["kind"] == "train"
    state["gate"] = gate.to(dtype).requires_grad_(train)
    state["value"] = value.to(dtype).requires_grad_(train)
    state["state"] = randn(n, width).requires_grad_(train)
    if train:
        state["grad"] = randn(*shape).to(dtype)
        state["grad_last"] = randn(n, width)
    return state


# ---- plain forms

def _plain_packed(x, rows):
    """What the packed copy of ``x`` stands for, in float32; groups of 32 along what is behind the first ``rows`` dimensions."""
    shape = x.shape
    x = x.float().reshape(shape[:rows].numel(), -1)
    width = x.shape[1]
    groups = (width + 31) // 32
    x = torch.nn.functional.pad(x, (0, groups * 32 - width)).view(x.shape[0], groups, 32)
    finite = torch.isfinite(x)
    mantissa, exponent = torch.frexp(torch.where(finite, x, 0.0).abs().amax(-1, keepdim=True))
    e = (exponent - 7 + (mantissa > 125 / 128).int()).clamp(min=-126)
    scale = torch.ldexp(torch.ones_like(mantissa), e)
    held = torch.round(torch.ldexp(x, -e)) * scale
    return torch.where(finite, held, x).view(x.shape[0], -1)[:, :width].reshape(shape)


def _plain_affine_scan(a, b):
    """x_t = a_t x_{t-1} + b_t along dimension -2 from x = 0, by doubling."""
    k, steps = 1, a.shape[-2]
    while k < steps:
        b = torch.cat([b[..., :k, :], torch.addcmul(b[..., k:, :], a[..., k:, :], b[..., :-k, :])], -2)
        a = torch.cat([a[..., :k, :], a[..., k:, :] * a[..., :-k, :]], -2)
        k *= 2
    return b


def _plain_starts(offsets, total):
    """Per step: whether it begins a sequence; and the sequences that have steps, with their first and last one."""
    some = offsets[1:] > offsets[:-1]
    first, last = offsets[:-1], offsets[1:] - 1
    begins = torch.zeros(total + 1, dtype=torch.bool, device=offsets.device)
    begins[torch.where(some, first, total)] = True
    return begins[:total, None], some[:, None], first.clamp(max=total - 1), last.clamp(min=0)


def _plain_scan(s):
    """(h, last) in float32."""
    z, u, h0 = s["gate"].detach().float(), s["value"].detach().float(), s["state"].detach()
    a, n = torch.sigmoid(z), torch.sigmoid(-z)
    b = torch.where(n == 0, 0.0, n * u)
    if "offsets" not in s:
        b = torch.cat([b[:, :1] + a[:, :1] * h0[:, None], b[:, 1:]], 1)
        h = _plain_affine_scan(a, b)
        return h, h[:, -1]
    total = z.shape[0]
    begins, some, first, last = _plain_starts(s["offsets"], total)
    b = b.index_add(0, first, torch.where(some, a[first] * h0, 0.0))
    h = _plain_affine_scan(torch.where(begins, 0.0, a), b)
    return h, torch.where(some, h[last], h0)


def _plain_scan_backward(s):
    """The gradients of gate, value and state in float32."""
    z, u, h0 = s["gate"].detach(), s["value"].detach(), s["state"].detach()
    if s["case"]["packed"]:
        rows = 1 if "offsets" in s else 2
        z, u = _plain_packed(z, rows), _plain_packed(u, rows)
    z, u, g, gl = z.float(), u.float(), s["grad"].float(), s["grad_last"]
    a, n = torch.sigmoid(z), torch.sigmoid(-z)
    h, _ = _plain_scan({**s, "gate": z, "value": u})
    # c_t = a_t (g_t + c_{t+1}), from behind the end to the start
    if "offsets" not in s:
        before = torch.cat([h0[:, None], h[:, :-1]], 1)
        g = torch.cat([g[:, :-1], g[:, -1:] + gl[:, None]], 1)
        c = _plain_affine_scan(a.flip(-2), (a * g).flip(-2)).flip(-2)
        dh = g + torch.cat([c[:, 1:], torch.zeros_like(c[:, :1])], 1)
        d0 = c[:, 0]
    else:
        total = z.shape[0]
        begins, some, first, last = _plain_starts(s["offsets"], total)
        before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
        before = torch.where(begins, 0.0, before).index_add(0, first, torch.where(some, h0, 0.0))
        g = g.index_add(0, last, torch.where(some, gl, 0.0))
        ends = torch.cat([begins[1:], torch.ones_like(begins[:1])])  # the step after it begins another sequence
        c = _plain_affine_scan(torch.where(ends, 0.0, a).flip(0), (a * g).flip(0)).flip(0)
        dh = g + torch.where(ends, 0.0, torch.cat([c[1:], torch.zeros_like(c[:1])]))
        d0 = torch.where(some, c[first], gl)
    dz = torch.where(a * n == 0, 0.0, a * n * (before - u) * dh)
    return dz, n * dh, d0


def _plain_norm(s):
    x, gamma, beta, g = s["x"].detach(), s["gamma"].detach(), s["beta"].detach(), s["grad"]
    dims = (1, 2, 3)
    mean = x.mean(dims, keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean(dims, keepdim=True) + 1e-5)
    y = (x - mean) * rstd * gamma + beta
    p, q = (_plain_packed(x, 1) - mean) * rstd, gamma * g
    gx = rstd * (q - q.mean(dims, keepdim=True) - p * (q * p).mean(dims, keepdim=True))
    return {"y": y, "x": gx, "gamma": (g * p).sum(0), "beta": g.sum(0)}


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        import gridnet_b200 as gb

        if kind == "pack":
            return gb.unpack_activations(gb.pack_activations(state["x"]))
        if kind == "step":
            h, last = gb.gated_scan_step(state["gate"], state["value"], state["state"])
            return {"h": h, "last": last}
        if kind == "read":
            h, last = gb.gated_scan(state["gate"], state["value"], state["state"], state.get("offsets"))
            return {"h": h, "last": last}
        if kind == "train":
            leaves = state["gate"], state["value"], state["state"]
            h, last = gb.gated_scan(*leaves, state.get("offsets"), packed=case["packed"])
            grads = torch.autograd.grad([h, last], leaves, [state["grad"], state["grad_last"]])
            return {"h": h.detach(), "last": last.detach(), "gate": grads[0], "value": grads[1], "state": grads[2]}
        leaves = state["x"], state["gamma"], state["beta"]
        y = gb.PackedGridNormOp.apply(*leaves, 1e-5)
        grads = torch.autograd.grad(y, leaves, state["grad"])
        return {"y": y.detach(), "x": grads[0], "gamma": grads[1], "beta": grads[2]}
    if kind == "pack":
        return _plain_packed(state["x"], 1).to(state["x"].dtype)
    if kind == "norm":
        return _plain_norm(state)
    dtype = state["gate"].dtype
    if kind == "step":
        z = state["gate"].float()
        a, n = torch.sigmoid(z), torch.sigmoid(-z)
        last = a * state["state"] + torch.where(n == 0, 0.0, n * state["value"].float())
        return {"h": last.to(dtype), "last": last}
    h, last = _plain_scan(state)
    out = {"h": h.to(dtype), "last": last}
    if kind == "train":
        dz, du, d0 = _plain_scan_backward(state)
        out |= {"gate": dz.to(dtype), "value": du.to(dtype), "state": d0}
    return out


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "pack":
        values = case["rows"] * case["width"]
        return {"bytes": 2 * size * values, "flops": 4 * values}
    if case["kind"] == "norm":
        voxels = case["m"] * case["n"] * case["k"]
        values = case["batch"] * voxels
        # inputs, their gradients and those of the outputs; gamma and beta and theirs
        return {"bytes": 4 * (4 * values + 4 * voxels), "flops": 20 * values}
    values, states = case["n"] * case["steps"] * case["width"], case["n"] * case["width"]
    if case["kind"] == "train":
        # gate, value and the output's gradient read, the output and two gradients written; four states
        return {"bytes": 6 * size * values + 16 * states, "flops": 25 * values}
    return {"bytes": 3 * size * values + 8 * states, "flops": 8 * values}


# ---- the definitions in 64 bits, step by step

def _exact_packed(x, rows):
    x = x.double()
    flat = x.reshape(x.shape[:rows].numel(), -1)
    out = flat.clone()
    for rest in (0, 1):  # the whole groups, then what is left behind them
        whole = flat.shape[1] // 32 * 32
        part = flat[:, :whole].unflatten(1, (-1, 32)) if not rest else flat[:, None, whole:]
        if not part.numel():
            continue
        finite = part.abs() < float("inf")
        top = part.abs().masked_fill(~finite, 0).amax(-1, keepdim=True)
        step = torch.exp2(torch.ceil(torch.log2((top / 125).clamp(min=2.0 ** -126))))
        # the logarithm's rounding next to a power of two
        step = torch.where(125 * step / 2 >= top, (step / 2).clamp(min=2.0 ** -126), step)
        step = torch.where(125 * step < top, step * 2, step)
        held = torch.where(finite, torch.round(part / step) * step, part)
        if rest:
            out[:, whole:] = held[:, 0]
        else:
            out[:, :whole] = held.flatten(1)
    return out.reshape(x.shape)


def _exact_scan(z, u, g, h0, gl):
    """One sequence [..., steps, width] at a time; with g also the gradients."""
    a, n = 1 / (1 + torch.exp(-z)), 1 / (1 + torch.exp(z))
    b = torch.where(n == 0, 0.0, n * u)
    h, before, hs = h0, [], []
    for t in range(z.shape[-2]):
        before.append(h)
        h = a[..., t, :] * h + b[..., t, :]
        hs.append(h)
    hs = torch.stack(hs, -2) if hs else z
    if g is None:
        return hs, h
    dh, dhs, c = None, [], gl
    for t in reversed(range(z.shape[-2])):
        dh = g[..., t, :] + c
        dhs.append(dh)
        c = a[..., t, :] * dh
    dhs = torch.stack(dhs[::-1], -2) if dhs else z
    before = torch.stack(before, -2) if before else z
    return hs, h, torch.where(a * n == 0, 0.0, a * n * (before - u) * dhs), n * dhs, c


def exact(case, seed):
    if case.get("ragged") and case["n"] * case["steps"] > 60000:
        return None  # one step of one sequence after the other: minutes
    s = prepare(case, seed)
    wide = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if case["kind"] == "pack":
        return _exact_packed(s["x"], 1).to(torch.float64)
    if case["kind"] == "norm":
        x, gamma, g = wide["x"].flatten(1), wide["gamma"].flatten(), wide["grad"].flatten(1)
        var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
        r = (var + 1e-5).rsqrt()
        y = torch.addcmul(wide["beta"].flatten(), (x - mean) * r, gamma)
        p = (_exact_packed(s["x"].detach(), 1).flatten(1) - mean) * r
        q = g * gamma
        gx = r * (q - (q.sum(1, keepdim=True) + p * (q * p).sum(1, keepdim=True)) / x.shape[1])
        grid = s["gamma"].shape
        return {"y": y.view(s["x"].shape), "x": gx.view(s["x"].shape), "gamma": (g * p).sum(0).view(grid), "beta": g.sum(0).view(grid)}
    z, u, h0 = wide["gate"], wide["value"], wide["state"]
    if case["kind"] == "step":
        h, last = _exact_scan(z[:, None], u[:, None], None, h0, None)
        return {"h": h[:, 0], "last": last}
    ends = s["offsets"].tolist() if case["ragged"] else None
    parts = [slice(a, b) for a, b in zip(ends, ends[1:])] if ends else [slice(None)]
    # ragged: one sequence after the other, its state a row; else all at once
    row = (lambda t, i: t[i]) if ends else (lambda t, i: t)
    join = (lambda ts: torch.cat(ts)) if ends else (lambda ts: ts[0])
    rows = (lambda ts: torch.stack(ts)) if ends else (lambda ts: ts[0])
    done = [_exact_scan(z[p], u[p], None, row(h0, i), None) for i, p in enumerate(parts)]
    out = {"h": join([d[0] for d in done]), "last": rows([d[1] for d in done])}
    if case["kind"] == "train":
        if case["packed"]:
            lead = 1 if ends else 2
            z, u = _exact_packed(s["gate"].detach(), lead), _exact_packed(s["value"].detach(), lead)
        done = [_exact_scan(z[p], u[p], wide["grad"][p], row(h0, i), row(wide["grad_last"], i)) for i, p in enumerate(parts)]
        out |= {"gate": join([d[2] for d in done]), "value": join([d[3] for d in done]), "state": rows([d[4] for d in done])}
    return out
