"""Announced reloads that are invalidated while they are being encrypted."""
from __future__ import annotations

import time

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from conftest import det_bytes  # noqa: E402
from test_prepare_gpu import check, layer_inputs  # noqa: E402


@pytest.fixture(scope="module")
def nl():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from secure_infer_b200 import native_layerwise
    s = native_layerwise.Session(0, det_bytes("prepare-key", 16), det_bytes("prepare-salt", 4))
    yield native_layerwise
    s.close()


def test_what_was_invalidated_under_encryption_is_no_miss(nl):
    """80 MB take the host some milliseconds to encrypt, the invalidations come meanwhile."""
    host, cache, mapping = layer_inputs(nl, 8, 160, 6, 11)
    small, small_cache, small_mapping = layer_inputs(nl, 2, 3, 7, 12)
    t = nl.NativeTransfer("none", layers=8)
    before = nl.prefetch_stats()
    for wait in (0.0002, 0.0004, 0.0007, 0.001, 0.0015):
        assert t.prepare_layer((host, mapping), 8, layer=6)
        time.sleep(wait)
        nl._native.lib().secure_infer_invalidate_transfer_prefetches()
        t.layer = 7
        t.single_layer_kv_transfer((small, small_mapping), small_cache)
        t.wait_for_layer_load(7)
        check(small, small_cache, small_mapping)
    assert nl.prefetch_stats() == before
    # What is announced now still counts, beside what is stale.
    assert t.prepare_layer((host, mapping), 8, layer=6)
    t.layer = 7
    t.single_layer_kv_transfer((small, small_mapping), small_cache)
    t.wait_for_layer_load(7)
    assert nl.prefetch_stats()["missing"] == before["missing"] + 1
    t.layer = 6
    t.single_layer_kv_transfer((host, mapping), cache)
    t.wait_for_layer_load(6)
    check(host, cache, mapping)
    assert nl.prefetch_stats()["ready"] == before["ready"] + 320
