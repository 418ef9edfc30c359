"""Caches and scales on another device than the tables are refused before anything is launched. CPU: the tables pass for
device tensors, the others lie on another device (meta)."""
import pytest
import torch

from kitchen_amd import _lib, kv


@pytest.mark.parametrize("wrong", ["cache", "k_scale", "v_scale"])
def test_caches_elsewhere(monkeypatch, wrong):
    called = []
    monkeypatch.setattr(_lib, "call", lambda name, *args: called.append(name))
    monkeypatch.setattr(_lib, "stream_of_device", lambda dev: 0)
    monkeypatch.setattr(kv, "_device_of", lambda t, what: t.device)
    monkeypatch.setattr(kv, "_kv_scratch", lambda pages, n, dev, stream: (torch.zeros(1), 4))
    table, lens, refs = (torch.zeros(n, dtype=torch.int32) for n in ((2, 3), 2, 5))

    def there(what):
        return "meta" if what == wrong else "cpu"

    cache = torch.zeros((1, 5, 2, 16, 64), dtype=torch.int8, device=there("cache"))
    ks, vs = (torch.zeros((1, 5, 2, 16), device=there(what)) for what in ("k_scale", "v_scale"))
    with pytest.raises(ValueError, match="must be on cpu"):
        kv.kv_fork(cache, cache, table, lens, refs, [0], [1], ks, vs)
    with pytest.raises(ValueError, match="must be on cpu"):
        kv.kv_compact(cache, cache, table, refs, ks, vs)
    assert not called
