"""Calls on tensors of another device than the current one: every launch is made on
the stream of the tensors' device, with that device as the current one (a launch
takes the current device's kernels).  Devices, streams and the library are stubs, so
this runs without a GPU."""

import contextlib

import pytest
import torch

from probjax_amd import attention as A
from probjax_amd import hip_attention as hip
from probjax_amd import masks, native

CURRENT, THEIRS = 3, 0


class _Library:
    def __init__(self, calls, state):
        self.calls, self.state = calls, state

    def __getattr__(self, name):
        if name.endswith(("_size", "_bytes")):
            return lambda *a: 64

        def entry(*args):
            self.calls.append((name, self.state["current"], args[-1]))
            return 0

        return entry


@pytest.fixture
def calls(monkeypatch):
    calls, state = [], {"current": CURRENT}

    @contextlib.contextmanager
    def device(index):
        was, state["current"] = state["current"], index
        yield
        state["current"] = was

    lib = _Library(calls, state)
    monkeypatch.setattr(native, "load", lambda: lib)
    monkeypatch.setattr(hip, "_on_device", lambda *ts: torch.device("cpu", THEIRS))
    monkeypatch.setattr(hip, "_gpu", lambda *ts: THEIRS)
    monkeypatch.setattr(hip, "_workspace_size", lambda *a: 64)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: state["current"], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 1000 + i, raising=False)
    yield calls
    assert state["current"] == CURRENT


def _bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def test_launches_on_the_tensors_device(calls):
    q, k, w = _bf16(2, 3, 4, 64), _bf16(2, 9, 2, 64), torch.zeros((2, 2, 9))
    lse, o = torch.zeros((2, 4, 3)), _bf16(2, 3, 4, 64)
    latent, cache = _bf16(2, 1, 4, 64), _bf16(2, 9, 64)
    wk = _bf16(4, 64, 64)
    for call in (
        lambda: A.attention_with_key_weights(q, k, k, w, mask=masks.CausalMask()),
        lambda: A.attention_with_key_weights(q, k, k, w),
        lambda: A.tree_attention(q, k, k, parents=[-1, 0, 0]),
        lambda: A.evict_keys(k, k, w, 4),
        lambda: A.rotary(q, None, torch.arange(3)),
        lambda: hip.flash_attention_fwd(q, k, k, sm_scale=0.1),
        lambda: hip.flash_attention_bwd(q, k, k, o, o, lse, sm_scale=0.1),
        lambda: hip.splitkv_decode(q, k, k, sm_scale=0.1),
        lambda: hip.mla_decode(latent, cache, sm_scale=0.1),
        lambda: hip.empty_rows(lse, k, o, grad=False),
        lambda: hip.zero_empty_rows(lse, o, o),
        lambda: hip.mla_project(cache, wk, wk, width=64),
        lambda: hip.mla_project_bwd(cache, wk, wk, _bf16(2, 9, 4, 64), _bf16(2, 9, 4, 64)),
    ):
        before = len(calls)
        call()
        assert len(calls) > before
    assert {(device, stream) for _, device, stream in calls} == {(THEIRS, 1000 + THEIRS)}, calls
    assert len({name for name, *_ in calls}) >= 13
