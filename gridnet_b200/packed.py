"""Activations in 8 bits: what a backward pass needs, kept in a quarter (float32) or half (16 bits) of the memory.

Groups of 32 values of a row share a power of two 2^e, the smallest with ``|x| <= 125 * 2^e`` (e >= -126); a value is held as
``x / 2^e`` rounded to a whole number, half to even, in a signed byte. 127, -127 and -128 are +inf, -inf and NaN, so what is not finite
stays what it is and does not touch its neighbours. 33 bytes hold 32 values, and a value is off by at most half a 2^e (up to a whole one beyond
63.5 * 2^122, the largest floats). A group has the precision of its largest: values that mark something are best infinite, a finite 1e30 leaves its neighbours none. The
reference has no counterpart: it keeps float32 between the passes.

:func:`pack_activations` / :func:`unpack_activations` are the two directions; :func:`keep_packed` has the norms, scans, steps and loops of this
package keep packed copies for their backward passes.
"""
from __future__ import annotations

import contextlib
from typing import NamedTuple

import torch

from ._lib import GridnetB200Error, check, lib

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # gn_dtype
GROUP = 32

_keep_packed = False


def keep_packed(enabled: bool) -> bool:
    """Whether differentiated float32 calls keep 8-bit copies of activations for their backward passes, and compute their gradients at those copies:
    the input of :class:`GridNorm`; the input of a step (:class:`Gridnet`, :class:`GatedGridnet`, with and without per-block normalisation);
    of the loops of the models the input and every step's output; and, whatever the type, gate and value of :func:`gated_scan`. Steps and loops then
    run their inner iterations again, from the copies, and keep none of them (:func:`keep_forward_stash`). Outputs are the same with and without.
    Off by default. Holds for forward passes that start afterwards; a backward pass goes by what its forward pass kept. Returns the previous
    setting."""
    global _keep_packed
    previous, _keep_packed = _keep_packed, bool(enabled)
    return previous


def keeps_packed() -> bool:
    return _keep_packed


class PackedActivations(NamedTuple):
    """``codes``: a signed byte per value, in the shape of the tensor; ``scales``: a byte per group, the row dimensions and the groups of a
    row; ``dtype``: the tensor's type."""
    codes: torch.Tensor
    scales: torch.Tensor
    dtype: torch.dtype

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()


def dtype_id(t: torch.Tensor, name: str) -> int:
    if t.dtype not in DTYPES:
        raise GridnetB200Error(f"unsupported dtype {t.dtype} of {name}: float32, bfloat16 and float16 only")
    return DTYPES[t.dtype]


_HERE = contextlib.nullcontext()


def on_device(device: torch.device):
    """``torch.cuda.device(device)``, but nothing where that is the current one already (1.5 us)."""
    return _HERE if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)


def stream_of(t: torch.Tensor) -> int:
    return torch._C._cuda_getCurrentRawStream(t.device.index)


def check_written(t: torch.Tensor, name: str) -> None:
    """What torch asks of a tensor that is written in place."""
    if t.requires_grad and torch.is_grad_enabled():
        raise GridnetB200Error(f"{name} requires a gradient: what is written in place here has none")


def overlaps(out: torch.Tensor, t: torch.Tensor) -> bool:
    """Whether ``out``, contiguous, has bytes of ``t``, which is [rows, values] with the values of a row side by side and rows at any
    distance."""
    rows, row = t.shape[0], t.shape[1] * t.element_size()
    lo, nbytes, base = out.data_ptr(), out.numel() * out.element_size(), t.data_ptr()
    if not rows or not row or not nbytes or base >= lo + nbytes:
        return False
    distance = t.stride(0) * t.element_size()
    # the first row that ends behind the start of out
    first = max(0, (lo - row - base) // distance + 1) if distance else 0
    return first < rows and base + first * distance < lo + nbytes and base + first * distance + row > lo


def refuse_overlap(out: torch.Tensor, name: str, **inputs: torch.Tensor) -> None:
    """The kernels read and write in no order that a caller could count on."""
    for other, t in inputs.items():
        if overlaps(out, t):
            raise GridnetB200Error(f"{name} shares memory with {other}")


# After the library has written to a tensor of the caller's: autograd counts it like an in-place operation of torch's own
written = torch.autograd.graph.increment_version


def pack_activations(x: torch.Tensor, rows: int = 1) -> PackedActivations:
    """The packed copy of ``x`` (float32, bfloat16 or float16, on a CUDA device). The first ``rows`` dimensions count rows (a sample, a
    step of a sequence); groups of 32 run along the others taken together and never across a row's end."""
    if not x.is_cuda:
        raise GridnetB200Error("x must be a CUDA tensor")
    dtype = dtype_id(x, "x")
    assert 0 <= rows <= x.dim(), f"{rows=} invalid for {x.shape=}"
    x = x.contiguous()
    nrows, cols = x.shape[:rows].numel(), x.shape[rows:].numel()
    codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scales = torch.empty((*x.shape[:rows], (cols + GROUP - 1) // GROUP), dtype=torch.uint8, device=x.device)
    with on_device(x.device):
        check(lib.gn_pack8(x.data_ptr(), codes.data_ptr(), scales.data_ptr(), nrows, cols, dtype, stream_of(x)))
    return PackedActivations(codes, scales, x.dtype)


def unpack_activations(packed: PackedActivations, out: torch.Tensor | None = None) -> torch.Tensor:
    """What the packed copy stands for, in the tensor's own type or in ``out``'s (contiguous, any of the three types; no memory of the
    copy's), rounded to it. Autograd sees a change in place of ``out``."""
    codes, scales, dtype = packed
    for name, t in (("codes", codes), ("scales", scales)):
        if not t.is_cuda:
            raise GridnetB200Error(f"{name} must be a CUDA tensor")
        if not t.is_contiguous():
            raise GridnetB200Error(f"{name} must be contiguous")
    assert codes.dtype == torch.int8 and scales.dtype == torch.uint8, f"{codes.dtype=} {scales.dtype=}: int8 and uint8"
    assert codes.device == scales.device, f"mismatching devices: {codes.device=} {scales.device=}"
    rows = scales.dim() - 1
    nrows, cols = codes.shape[:rows].numel(), codes.shape[rows:].numel()
    assert 0 <= rows <= codes.dim() and scales.shape == (*codes.shape[:rows], (cols + GROUP - 1) // GROUP), (
        f"{scales.shape=} invalid for {codes.shape=}")
    given = out is not None
    if not given:
        out = torch.empty(codes.shape, dtype=dtype, device=codes.device)
    assert out.shape == codes.shape, f"{out.shape=} invalid for {codes.shape=}"
    assert out.device == codes.device, f"mismatching devices: {codes.device=} {out.device=}"
    if not out.is_contiguous():
        raise GridnetB200Error("out must be contiguous")
    check_written(out, "out")
    if given:
        refuse_overlap(out, "out", codes=codes.view(1, -1), scales=scales.view(1, -1))
    with on_device(codes.device):
        check(lib.gn_unpack8(codes.data_ptr(), scales.data_ptr(), out.data_ptr(), nrows, cols, dtype_id(out, "out"), stream_of(codes)))
    if given:
        written(out)
    return out
