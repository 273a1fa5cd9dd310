"""The attention block takes projections of the cache's device only (host-only stand-ins: one
GPU or none is needed)."""

import types

import pytest
import torch

import mlxl3_amd
from mlxl3_amd import kv


def linear(device, loaded=False):
    """What Exl3Linear says of itself: its tensors' device, or the one it was loaded to."""
    made = types.SimpleNamespace(in_features=64, out_features=64, k=4, cb=0, handle=None)
    if loaded:
        made.trellis, made.device = None, torch.device(device)
    else:
        made.trellis = types.SimpleNamespace(device=torch.device(device))
    return made


@pytest.mark.parametrize("loaded", [False, True])
@pytest.mark.parametrize("other", range(4))
def test_projections_of_one_device(loaded, other):
    parts = [linear("cuda:1" if i == other else "cuda:0", loaded) for i in range(4)]
    with pytest.raises(mlxl3_amd.Exl3Error, match="is on cuda"):
        mlxl3_amd.Exl3Attention(*parts)


@pytest.mark.parametrize("loaded", [False, True])
def test_projections_of_the_caches_device(monkeypatch, loaded):
    monkeypatch.setattr(kv, "_device_tensor", lambda t, *a: t)
    block = mlxl3_amd.Exl3Attention(*(linear("cuda:1", loaded) for _ in range(4)))
    cpu = torch.device("cpu")
    cache, batch = types.SimpleNamespace(device=cpu), types.SimpleNamespace(kv_lens=torch.zeros(1))
    with pytest.raises(mlxl3_amd.Exl3Error, match="projections is on cuda:1, expected cpu"):
        block(torch.zeros(1, 64, dtype=torch.float16), cache, batch)


def test_a_projection_loaded_to_the_device_that_was_current():
    """"cuda" without a number names no device to compare."""
    parts = [linear("cuda" if i == 1 else "cuda:1", True) for i in range(4)]
    mlxl3_amd.Exl3Attention(*parts)
