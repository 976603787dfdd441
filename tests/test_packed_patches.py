"""Loops on the register-patch kernels with 8-bit copies: which copies are made and how often they are unpacked, without a GPU (the kernels
are left out)."""
import contextlib

import pytest
import torch

import gridnet_b200.backend_cuda as bc
from gridnet_b200 import patch_loop
from gridnet_b200.packed import PackedActivations


class _NoKernels:
    def __getattr__(self, name):
        return lambda *args: 1 if name == "gn_step_stats_partials" else 0


@pytest.fixture()
def counted(monkeypatch):
    """Names of what is packed and unpacked, in order; and how many unpacked grids are held at most."""
    packs, unpacks, alive, most = [], [], set(), [0]

    class Grid(torch.Tensor):
        def __del__(self):
            alive.discard(id(self))

    def pack(x, rows=1):
        packs.append(len(packs))
        return PackedActivations(x.new_full((1,), len(packs) - 1), x.new_zeros(1), torch.float32)

    def unpack(p, out=None):
        unpacks.append(int(p.codes))
        t = torch.zeros(1, 8, 8, 8).as_subclass(Grid)
        alive.add(id(t))
        most[0] = max(most[0], len(alive))
        return t

    monkeypatch.setattr(bc, "pack_activations", pack)
    monkeypatch.setattr(bc, "unpack_activations", unpack)
    monkeypatch.setattr(bc, "keeps_packed", lambda: True)
    monkeypatch.setattr(patch_loop, "lib", _NoKernels())
    monkeypatch.setattr(patch_loop.gridnet_cuda, "backward", lambda *args: None)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: type("S", (), {"cuda_stream": 0}))
    return packs, unpacks, most


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("outer", [1, 2, 6])
def test_each_copy_is_made_and_unpacked_once(counted, outer, residual):
    packs, unpacks, most = counted
    plist = [(torch.zeros(27, 8, 8, 8), torch.zeros(8, 8, 8), torch.zeros(8, 8, 8))]
    norm, x = torch.ones(8, 8, 8), torch.zeros(1, 8, 8, 8)
    y, saved = bc._patch_forward(plist, norm, norm, x, 2, outer, 8, "silu", 1e-5, residual, True)
    # the input and every step's output; with residual nothing reads the last one's
    needed = outer + (0 if residual else 1)
    assert len(packs) == needed
    bc._loop_backward(plist, norm, norm, saved, torch.zeros_like(x), 2, outer, 8, "silu", residual)
    assert unpacks == list(reversed(range(needed)))  # once each, as the steps are walked back
    assert most[0] == 1
