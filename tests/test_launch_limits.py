"""Calls whose launch would hold 2^32 threads are refused, those just below are not (CPU: nothing is launched)."""
import ctypes

import pytest

import femtochat_amd._lib as L

FAKE = 0x10000  # an aligned address; nothing is read before the checks fail


def _last():
    return L.lib().fc_last_error().decode()


@pytest.mark.parametrize("V", [1, 259, 2048])
@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_sequences_of_a_small_vocabulary(V, temperature):
    """A workgroup of 1024 threads for each of them."""
    n = ctypes.c_size_t(7)
    fits, beyond = (L.VerifyDesc(B, 1, V, L.FC_F32, 0, 0, 0, temperature) for B in (2 ** 22 - 1, 2 ** 22))
    assert L.lib().fc_verify_workspace_bytes(fits, ctypes.byref(n)) == L.FC_OK and n.value == 0
    assert L.lib().fc_verify_workspace_bytes(beyond, ctypes.byref(n)) == L.FC_ERR_UNSUPPORTED and "sequences" in _last()
    st = L.lib().fc_verify_drafts(beyond, FAKE, None, FAKE, FAKE, None, None, FAKE, FAKE, FAKE, None, 0, None)
    assert st == L.FC_ERR_UNSUPPORTED


def test_sequences_of_a_large_vocabulary():
    """256 threads to a chunk: the limit on logits comes first."""
    n = ctypes.c_size_t(0)
    assert L.lib().fc_verify_workspace_bytes(L.VerifyDesc(2 ** 22, 1, 2049, L.FC_F32, 0, 0, 0, 1.0), ctypes.byref(n)) == L.FC_OK


@pytest.mark.parametrize("B,Hkv,G,N,fits", [
    (16384, 1024, 1, 1, False), (16383, 1024, 1, 1, True), (16384, 512, 2, 1, True), (16384, 1, 16, 64, True),
    (32768, 512, 1, 1, False), (65535, 256, 1, 1, True),
])
def test_rows_of_attention(B, Hkv, G, N, fits):
    """A workgroup of 256 threads for a sequence's KV head and sixteen of its rows, or 32."""
    n = ctypes.c_size_t(0)
    d = L.CacheDesc(16, Hkv, B, 1, 4, 16, 1, L.FC_CACHE_I8)
    o = L.CachedAttnOptions(Hkv * G, N, -1, 0, 0.0, None)
    st = L.lib().fc_cached_attn_workspace_bytes(d, o, ctypes.byref(n))
    assert st == (L.FC_OK if fits else L.FC_ERR_UNSUPPORTED), _last()
    if not fits:
        assert "workgroups" in _last()
        c = L.Cache(FAKE, FAKE, FAKE, FAKE, FAKE)
        assert L.lib().fc_cached_attn(d, c, o, FAKE, FAKE, FAKE, None, None, None, 0, None) == L.FC_ERR_UNSUPPORTED
