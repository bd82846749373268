"""attn_verify_q8's workspace of a cache on another device than the current one: a call
that is being captured there must not share one with eager calls (no GPU: the devices
are stand-ins)."""
from __future__ import annotations

import contextlib
from types import SimpleNamespace

import pytest
import torch

from dflash_mlx import kv8


@pytest.mark.parametrize("current", [0, 1])
@pytest.mark.parametrize("capturing", [(False, False), (False, True), (True, False), (True, True)])
def test_a_capture_on_the_cache_s_device(monkeypatch, current, capturing):
    now = [current]

    @contextlib.contextmanager
    def device(d):
        before, now[0] = now[0], d.index
        yield
        now[0] = before

    empty = torch.empty
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[now[0]])
    monkeypatch.setattr(torch, "empty", lambda n, dtype, device: empty(n, dtype=dtype))
    monkeypatch.setattr(kv8._lib, "stream_handle", lambda dev: 7)
    monkeypatch.setattr(kv8, "attn_verify_q8_workspace_bytes", lambda *a: 4096)
    cache = object.__new__(kv8.QuantizedKVCache)
    cache.B, cache.Hkv, cache.Smax, cache.device = 2, 4, 128, SimpleNamespace(index=1)
    cache._ws_bytes, cache._workspaces = {}, {}
    a, b = (kv8._verify_workspace(cache, 4, 16) for _ in range(2))
    assert now[0] == current and (a[:32] == 0).all()
    if capturing[1]:
        assert a is not b and not cache._workspaces
    else:
        assert a is b and cache._workspaces[7] is a
