"""The attention block's own workspaces under threads, without a GPU: the launch is replaced by
one that tells who is inside."""

import threading
import types

import pytest
import torch

import mlxl3_amd
from mlxl3_amd import kv


@pytest.fixture
def block(monkeypatch):
    """(block, call, launches): call(stream) runs a forward as if on that stream; launches holds
    for each one the workspace and how many others were inside with the same."""
    stream = threading.local()
    launches, inside, guard = [], {}, threading.Lock()
    waiting = threading.Barrier(2)

    def launch(device, entry, *args):
        space = args[-2]
        with guard:
            inside[space] = inside.get(space, 0) + 1
        try:
            waiting.wait(0.3)  # both threads are in a launch at once, or that never happens
            met = True
        except threading.BrokenBarrierError:
            met = False
        with guard:
            launches.append((space, inside[space], met))
            inside[space] -= 1

    lib = types.SimpleNamespace(exl3_linear_output_dtype=lambda *a: 9, exl3_attn_block_workspace_bytes=lambda *a: 4096,
                                exl3_attn_block_forward=None)
    monkeypatch.setattr(kv, "load_library", lambda: lib)
    monkeypatch.setattr(kv, "_device_tensor", lambda t, *a: t)
    monkeypatch.setattr(kv, "_stream_ptr", lambda device: stream.at)
    monkeypatch.setattr(kv, "_launch", launch)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    linear = lambda n: types.SimpleNamespace(in_features=64, out_features=n, k=4, cb=0, handle=None, trellis=torch.zeros(1))
    made = mlxl3_amd.Exl3Attention(linear(64), linear(64), linear(64), linear(64))
    cache = types.SimpleNamespace(device=torch.device("cpu"), head_dim=64, handle=None)
    batch = types.SimpleNamespace(kv_lens=torch.zeros(1), _attended=lambda rows: None)

    def call(at):
        stream.at = at
        made(torch.zeros(1, 64, dtype=torch.float16), cache, batch)

    return made, call, launches


def together(*works):
    threads = [threading.Thread(target=w) for w in works]
    for t in threads:
        t.start()
    for t in threads:
        t.join()


def test_two_threads_on_one_stream_take_turns(block):
    """One call's launches are in the stream before the next one's: each overwrites the space
    for q, k and v of the last."""
    _, call, launches = block
    together(lambda: call(7), lambda: call(7))
    assert len(launches) == 2 and launches[0][0] == launches[1][0]
    assert [n for _, n, _ in launches] == [1, 1] and not any(met for *_, met in launches)


def test_two_threads_on_two_streams_do_not_wait(block):
    _, call, launches = block
    together(lambda: call(7), lambda: call(8))
    assert launches[0][0] != launches[1][0]
    assert [n for _, n, _ in launches] == [1, 1] and all(met for *_, met in launches)


def test_kept_workspaces_are_bounded(block, monkeypatch):
    """A program that makes streams for ever does not keep a workspace for each."""
    made, call, launches = block
    monkeypatch.setattr(kv, "_launch", lambda *a: None)
    for at in range(500):
        call(at)
    assert len(made._ws) <= 64
