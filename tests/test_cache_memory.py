"""What cache_write may write to, without a GPU: caches two of whose elements share memory are refused, others are not."""
import contextlib

import pytest
import torch

from memarch_amd import _lib, attention, kv_cache

F8 = torch.float8_e4m3fn


@pytest.fixture
def launched(monkeypatch):
    names = []
    monkeypatch.setattr(_lib, "call", lambda *a: names.append(a[0]))
    for mod in (attention, kv_cache):
        monkeypatch.setattr(mod, "_check_same", lambda *a: None)
        monkeypatch.setattr(mod, "_On", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(kv_cache, "_stream", lambda dev: 0)
    return names


def _mem(*shape):
    return torch.zeros(*shape, dtype=torch.uint8).view(F8)


def _write(kc, vc, scales=None):
    pages, page, h, d = kc.shape
    x = torch.zeros(2, h, d, dtype=torch.bfloat16)
    scales = scales or [torch.zeros(pages, page // 8, h) for _ in range(2)]
    kv_cache.cache_write(x, x, kc, vc, *scales, torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32))


def test_elements_that_share_memory_are_refused(launched):
    shape = (4, 16, 2, 64)
    good = _mem(*shape)
    for bad in (_mem(4, 16, 1, 64).expand(shape), _mem(1, 16, 2, 64).expand(shape),          # heads, pages that are one
                _mem(4 * 16 * 128 + 64).as_strided(shape, (2048, 128, 32, 1)),                # heads that run into each other
                _mem(8 * 16 * 128).as_strided(shape, (1024, 128, 64, 1))):                    # pages that do
        for pair in ((bad, good), (good, bad)):
            with pytest.raises(ValueError, match="share memory"):
                _write(*pair)
    with pytest.raises(ValueError, match="same memory"):
        _write(good, good)
    one = torch.zeros(4, 2, 2)
    with pytest.raises(ValueError, match="same memory"):
        _write(good, _mem(*shape), [one, one])
    assert not launched


def test_other_layouts_are_written(launched):
    both = _mem(4, 2, 16, 2, 64)                        # keys and values side by side in a page
    heads = _mem(2, 4, 2, 16, 64)                       # heads outside slots
    wide = _mem(4, 16, 2, 2, 128)                       # slices of everything
    layers = _mem(16, 4, 2, 3, 2, 64)                   # slots outside pages, one layer of several
    pairs = [(both[:, 0], both[:, 1]), (heads[0].transpose(1, 2), heads[1].transpose(1, 2)),
             (wide[:, :, 0, :, 64:], wide[:, :, 1, :, :64]), (wide[1:3, :8, :, 0, :64], wide[1:3, 8:, :, 1, :64]),
             (layers[:, :, 0, 1].transpose(0, 1), layers[:, :, 1, 1].transpose(0, 1)),
             (_mem(1, 16, 1, 64).expand(1, 16, 1, 64), _mem(1, 16, 1, 64)), (_mem(0, 16, 2, 64), _mem(0, 16, 2, 64))]
    for kc, vc in pairs:
        _write(kc, vc)
    assert launched == ["mce_cache_write"] * len(pairs)


def test_reading_takes_shared_memory(launched):
    """Pages and heads that are one may be read."""
    shared = _mem(4, 16, 1, 64).expand(4, 16, 2, 64)
    s = torch.zeros(4, 2, 2)
    kv_cache.cache_read(shared, shared, s, s, torch.zeros(2, 3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), 5)
    assert launched == ["mce_cache_read"]
