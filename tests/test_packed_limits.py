"""The sizes that packed attention takes, without a GPU: what its header says is accepted is."""
import os

import pytest

from memarch_amd import _lib


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.SERVE_LIB_PATH):
        pytest.skip("libmce_serve.so not built")
    return _lib.load_serve()


@pytest.mark.parametrize("nseq,n,hq,hkv,d,window,sinks", [
    (4096, 2 ** 20, 32, 32, 128, 4096, 15000), (4096, 2 ** 20, 32, 32, 128, 4096, 16384), (4096, 2 ** 20, 32, 32, 128, 4096, 2 ** 20),
    (4096, 65536, 16, 16, 8, 100, 65536), (10 ** 5, 2 ** 27, 8, 2, 64, 1024, 2 ** 20), (10 ** 6, 2 ** 27, 2, 2, 64, 1024, 1000)])
def test_many_first_tokens_of_many_sequences(lib, nseq, n, hq, hkv, d, window, sinks):
    """All sequences together have no more key blocks than keys / 128 and one each, however many first tokens one could have:
    the limits are those of mce_pack.h, and the workspace does not grow with sequences times first tokens."""
    assert hq * (n // 128 + nseq + 2) < 2 ** 24 and hkv * (n // 128 + nseq + 2) < 2 ** 23 - 2 ** 11 and nseq * sinks // 128 < 2 ** 31
    need = lib.mce_pack_bwd_ws_bytes(nseq, n, n, hq, hkv, d, window, sinks)
    few = lib.mce_pack_bwd_ws_bytes(nseq, n, n, hq, hkv, d, window, 1)
    parts = 2 * 128 * d * 4
    assert 8 * n * hq <= need <= few + (2048 + hkv * (n // 128 + nseq + 2)) * parts
