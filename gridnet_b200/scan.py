"""The gated cell along a sequence. The gated grid updates a cell by ``h <- s(gate) h + (1 - s(gate)) value``
(gridnet/backend_torch.py:241-265, s the logistic function) with gate and value from the cell's neighbours, iteration after iteration. Where gate
and value do not depend on the state - frames, read-out planes, tokens - the steps of a whole sequence can be taken at once:
:func:`gated_scan`; :func:`gated_scan_step` takes one, and :class:`GatedRecurrence` is a layer of it. The reference has no sequences.
"""
from __future__ import annotations

import functools

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from ._lib import GridnetB200Error, check, lib
from .backend_cuda import _Op, has_tangent
from .packed import DTYPES, GROUP, check_written, dtype_id, keeps_packed, on_device, refuse_overlap, stream_of, written


def _rows(t: torch.Tensor, lead: int) -> torch.Tensor:
    """``t`` as [..., width] with ``lead`` dimensions in front and the values of a step side by side: a view where there is one."""
    if t.dim() != lead + 1:
        t = t.reshape(*t.shape[:lead], t.shape[lead:].numel())
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _strides(t: torch.Tensor):
    """Distances of sequences (0: ragged) and of steps."""
    return t.stride()[:2] if t.dim() == 3 else (0, t.stride(0))


def _ptr(t):
    return None if t is None else t.data_ptr()


def _nbytes(t) -> int:
    return 0 if t is None else t.numel()


def _scratch(nbytes: int, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


@functools.lru_cache(maxsize=512)
def _sizes(device: int, *size):
    """Bytes of what a forward pass leaves, and of scratch: forward, backward, backward from packed copies."""
    with torch.cuda.device(device):
        work = lib.gn_gated_scan_workspace_bytes
        return int(lib.gn_gated_scan_bounds_bytes(*size)), int(work(*size, 0, 0)), int(work(*size, 1, 0)), int(work(*size, 1, 1))


def _check_scan(gate, value, state, offsets):
    """Returns (sequences, steps of each (0: ragged), rows in all)."""
    for name, t in (("gate", gate), ("value", value)):
        if not t.is_cuda:
            raise GridnetB200Error(f"{name} must be a CUDA tensor")
        dtype_id(t, name)
    assert gate.shape == value.shape, f"{value.shape=} invalid for {gate.shape=}"
    assert gate.dtype == value.dtype, f"mismatching dtypes: {gate.dtype=} {value.dtype=}"
    assert gate.device == value.device, f"mismatching devices: {gate.device=} {value.device=}"
    lead = 2 if offsets is None else 1
    assert gate.dim() > lead, f"{gate.shape=}: " + ("[batch, steps, ...]" if offsets is None else "[rows, ...] with offsets")
    assert gate.shape[lead:].numel() > 0, f"{gate.shape=}: steps of no values"
    if offsets is None:
        n, steps, total = gate.shape[0], gate.shape[1], gate.shape[0] * gate.shape[1]
    else:
        assert offsets.dim() == 1 and offsets.shape[0] >= 1, f"{offsets.shape=}: one more than there are sequences"
        assert offsets.dtype in (torch.int32, torch.int64), f"{offsets.dtype=}: int32 or int64"
        n, steps, total = offsets.shape[0] - 1, 0, gate.shape[0]
    if state is not None:
        assert state.shape == (n, *gate.shape[lead:]), f"{state.shape=} invalid for {gate.shape=} and {n} sequences"
        assert state.dtype == torch.float32, f"{state.dtype=}: states are float32"
        assert state.device == gate.device, f"mismatching devices: {gate.device=} {state.device=}"
    return n, steps, total


def _device_offsets(offsets, total: int, device):
    """Offsets as the kernels read them. Those that come from the host are looked at; those on the device are not (a value out of place there
    is taken as the nearest possible)."""
    if not offsets.is_cuda:
        o = offsets.tolist()
        assert o[0] == 0 and o[-1] == total and all(a <= b for a, b in zip(o, o[1:])), f"offsets rise from 0 to {total}: got {o[:4]} ... {o[-1]}"
    else:
        assert offsets.device == device, f"mismatching devices: {offsets.device=} {device=}"
    return offsets.to(device=device, dtype=torch.int64).contiguous()


def _packed_at(total: int, width: int):
    """Codes of the gate, of the value, scales of the gate, of the value in one allocation: where each starts, and the end."""
    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    codes, scales = up(total * width), up(total * ((width + GROUP - 1) // GROUP))
    return 0, codes, 2 * codes, 2 * codes + scales, 2 * (codes + scales)


def _packed_places(memory: torch.Tensor, total: int, width: int):
    """Addresses of the gate's codes and scales and the value's."""
    base, at = memory.data_ptr(), _packed_at(total, width)
    return base, base + at[2], base + at[1], base + at[3]


def _forward(gate, value, state, offsets, kept_packed: bool, need_grad: bool):
    """(h, last), and what the backward pass needs: the tensors to save and the sizes."""
    n, steps, total = _check_scan(gate, value, state, offsets)
    dtype, dev = DTYPES[gate.dtype], gate.device
    lead = 2 if offsets is None else 1
    z, u = _rows(gate, lead), _rows(value, lead)
    width = z.shape[-1]
    s = None if state is None else state.contiguous()
    offsets = None if offsets is None else _device_offsets(offsets, total, dev)
    size = (n, steps, total, width, dtype, lead & 1)
    left, scratch = _sizes(dev.index, *size)[:2]
    h = torch.empty(gate.shape, dtype=gate.dtype, device=dev)
    last = torch.empty((n, *gate.shape[lead:]), dtype=torch.float32, device=dev)
    codes, bounds, packed = (None,) * 4, None, None
    if need_grad and kept_packed:
        packed = torch.empty(max(1, _packed_at(total, width)[-1]), dtype=torch.uint8, device=dev)
        codes = _packed_places(packed, total, width)
    elif need_grad:
        bounds = _scratch(left, dev)
    work = _scratch(scratch, dev)
    with on_device(dev):
        check(lib.gn_gated_scan_forward(z.data_ptr(), u.data_ptr(), _ptr(s), _ptr(offsets), h.data_ptr(), last.data_ptr(), *codes,
                                        _ptr(bounds), n, steps, total, width, *_strides(z), *_strides(u), dtype, _ptr(work), scratch,
                                        stream_of(gate)))
    if packed is not None:
        return h, last, (packed, None, s, offsets, None), size
    return h, last, (z, u, s, offsets, bounds), size


class GatedScanOp(_Op):
    """``GatedScanOp.apply(gate, value, state, offsets, packed)``: :func:`gated_scan` as an autograd op."""

    @staticmethod
    def forward(ctx, gate, value, state, offsets, packed: bool):
        h, last, kept, ctx.size = _forward(gate, value, state, offsets, packed, any(ctx.needs_input_grad[:3]))
        ctx.set_materialize_grads(False)
        ctx.shape, ctx.dtype = gate.shape, gate.dtype
        ctx.save_for_backward(*kept)
        return h, last

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_h, grad_last):
        z, u, s, offsets, bounds = ctx.saved_tensors
        size, dev, packed = ctx.size, z.device, u is None
        grad_h = torch.zeros(ctx.shape, dtype=ctx.dtype, device=dev) if grad_h is None else grad_h.contiguous()
        grad_last = None if grad_last is None else grad_last.contiguous()
        dz, du = torch.empty(ctx.shape, dtype=ctx.dtype, device=dev), torch.empty(ctx.shape, dtype=ctx.dtype, device=dev)
        ds = torch.empty_like(s) if s is not None and ctx.needs_input_grad[2] else None
        if packed:
            z_at, z_scales, u_at, u_scales = _packed_places(z, size[2], size[3])
            strides = (0, 0, 0, 0)
        else:
            z_at, u_at, z_scales, u_scales = z.data_ptr(), u.data_ptr(), None, None
            strides = (*_strides(z), *_strides(u))
        scratch = _sizes(dev.index, *size)[2 + packed]
        work = _scratch(scratch, dev)
        with on_device(dev):
            check(lib.gn_gated_scan_backward(z_at, u_at, z_scales, u_scales, _ptr(s), _ptr(offsets), _ptr(bounds),
                                             grad_h.data_ptr(), _ptr(grad_last), dz.data_ptr(), du.data_ptr(), _ptr(ds), *size[:4], *strides,
                                             size[4], _ptr(work), scratch, stream_of(z)))
        return dz, du, ds, None, None


def gated_scan(gate: torch.Tensor, value: torch.Tensor, state: torch.Tensor | None = None, offsets: torch.Tensor | None = None,
               packed: bool | None = None):
    """The gated cell along sequences, s the logistic function:

        h_t = s(gate_t) * h_{t-1} + s(-gate_t) * value_t

    ``gate`` and ``value`` are [batch, steps, ...], or [rows, ...] with ``offsets`` [n + 1] (int32 or int64): sequence i is rows
    ``offsets[i]`` to ``offsets[i + 1] - 1``, empty ones allowed, and rows of no sequence get zeros. float32, bfloat16 or float16;
    the recurrence itself is float32. ``state`` [n, ...] (float32) is the state ahead of the first step, zeros without. Returns
    ``(h, last)``: h like gate, and the state behind the last step, float32.

    A step whose s(-gate) is 0 (gate = inf) holds the state and does not look at its value, one whose s(gate) is 0
    (gate = -inf) takes its value and does not look at the state. Differentiable once in gate, value and state, backward only: tensors with a
    tangent of torch.autograd.forward_ad are refused. ``packed``: keep gate and value in 8 bits for the backward pass, which then takes the
    gradients at the packed copies; default as :func:`keep_packed` says. Groups of 32 neighbouring values of a step share a scale, so gates that
    hold or reset are best infinite.

    Offsets on the host are copied to the device, which a graph capture does not allow, and refused unless they rise from 0 to the number of
    rows; those on the device are not looked at, and may leave out rows ahead of the first sequence and behind the last. A step's values have to lie
    side by side, otherwise they are copied; steps and sequences may lie anywhere, so the halves of a wider projection are read where they are."""
    if offsets is not None and not isinstance(offsets, torch.Tensor):
        offsets = torch.as_tensor(offsets, dtype=torch.int64)
    if not (torch.is_grad_enabled() and (gate.requires_grad or value.requires_grad or (state is not None and state.requires_grad))
            or has_tangent(gate, value, state)):
        return _forward(gate, value, state, offsets, False, False)[:2]
    return GatedScanOp.apply(gate, value, state, offsets, keeps_packed() if packed is None else bool(packed))


def gated_scan_step(gate: torch.Tensor, value: torch.Tensor, state: torch.Tensor, out_state: torch.Tensor | None = None):
    """One step of :func:`gated_scan` without gradients: ``gate`` and ``value`` [batch, ...], ``state`` [batch, ...] float32. Returns
    ``(h, new_state)``; ``out_state`` (which may be ``state``, and otherwise shares no memory with the inputs) receives the new state, which
    autograd sees as a change in place."""
    for name, t in (("gate", gate), ("value", value), ("state", state)):
        if not t.is_cuda:
            raise GridnetB200Error(f"{name} must be a CUDA tensor")
    dtype = dtype_id(gate, "gate")
    shape, dev = gate.shape, gate.device
    assert len(shape) >= 2 and shape == value.shape == state.shape, f"{value.shape=} {state.shape=} invalid for {gate.shape=}"
    assert gate.dtype == value.dtype, f"mismatching dtypes: {gate.dtype=} {value.dtype=}"
    assert state.dtype == torch.float32, f"{state.dtype=}: states are float32"
    assert dev == value.device == state.device, f"mismatching devices: {gate.device=} {value.device=} {state.device=}"
    z, u, s = _rows(gate, 1), _rows(value, 1), state.contiguous()
    rows, width = z.shape
    assert width > 0, f"{gate.shape=}: steps of no values"
    given = out_state is not None
    if not given:
        out_state = torch.empty_like(s)
    else:
        assert out_state.shape == shape and out_state.dtype == torch.float32 and out_state.device == dev, (
            f"{out_state.shape=} {out_state.dtype=} {out_state.device=} invalid for a state of {state.shape}")
        if not out_state.is_contiguous():
            raise GridnetB200Error("out_state must be contiguous")
        check_written(out_state, "out_state")
        refuse_overlap(out_state, "out_state", gate=z, value=u)
        if out_state.data_ptr() != s.data_ptr():
            refuse_overlap(out_state, "out_state", state=s.view(rows, width))
    h = torch.empty(shape, dtype=gate.dtype, device=dev)
    with on_device(dev):
        check(lib.gn_gated_scan_step(z.data_ptr(), u.data_ptr(), s.data_ptr(), h.data_ptr(), out_state.data_ptr(), rows, width, z.stride(0),
                                     u.stride(0), dtype, stream_of(gate)))
    if given:
        written(out_state)
    return h, out_state


class GatedRecurrence(nn.Module):
    """A layer of :func:`gated_scan`: gate and value are one linear map of the input (plain torch, as in ``Readout``), and
    ``remember_bias`` is the gates' first bias, as in the gated MNIST model (gridnet/scripts/train_mnist.py:36-44).

    ``forward(x, state=None, offsets=None)``: x [batch, steps, in_features], or [rows, in_features] with offsets; returns (h, last).
    ``step(x, state, out_state=None)``: one step of x [batch, in_features], without gradients."""

    def __init__(self, in_features: int, features: int, device, dtype: torch.dtype = torch.float32, remember_bias: float = 1.0):
        super().__init__()
        self.features = features
        self.proj = nn.Linear(in_features, 2 * features, device=device, dtype=dtype)
        with torch.no_grad():
            self.proj.bias[:features].fill_(remember_bias)

    def forward(self, x: torch.Tensor, state: torch.Tensor | None = None, offsets: torch.Tensor | None = None):
        gate, value = self.proj(x).chunk(2, -1)
        return gated_scan(gate, value, state, offsets)

    @torch.no_grad()
    def step(self, x: torch.Tensor, state: torch.Tensor, out_state: torch.Tensor | None = None):
        gate, value = self.proj(x).chunk(2, -1)
        return gated_scan_step(gate, value, state, out_state)
