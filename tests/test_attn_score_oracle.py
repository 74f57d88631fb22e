"""Capped, biased and prefix-masked attention on the CPU: the oracle against the
plain attention oracle and against differences, and the refusals of the host side
(no kernel is launched)."""
import ctypes

import numpy as np
import pytest
import torch

import femtochat_amd as F
import femtochat_amd._lib as L
from oracle import attention_ref as R
from oracle import attention_score as S


def _qkv(seed, B=2, T=7, H=4, Hkv=2, D=16):
    rng = np.random.default_rng(seed)
    return [rng.standard_normal(s) for s in ((B, T, H, D), (B, T, Hkv, D), (B, T, Hkv, D), (B, T, H, D))]


@pytest.mark.parametrize("window", [(-1, 0), (3, 0), (2, 2), (4, -2)])
@pytest.mark.parametrize("documents", [False, True])
def test_without_options_it_is_plain_attention(window, documents):
    Q, K, V, _ = _qkv(1)
    pos = np.array([[0, 1, 2, 0, 1, 0, 1], [3, 4, 0, 1, 2, 3, 4]], np.int32) if documents else None
    for a, b in zip(S.forward(Q, K, V, window, pos), R.forward(Q, K, V, window, pos)):
        np.testing.assert_allclose(a, b, rtol=1e-12, atol=1e-12)


def test_the_prefix_mask_by_hand():
    seen = S.visible(5, (-1, 0), None, np.array([3, 0]))
    assert seen[0].astype(int).tolist() == [[1, 1, 1, 0, 0], [1, 1, 1, 0, 0], [1, 1, 1, 0, 0], [1, 1, 1, 1, 0], [1, 1, 1, 1, 1]]
    assert (seen[1] == np.tril(np.ones((5, 5), bool))).all()
    pos, pre = np.array([[0, 1, 2, 0, 1]]), np.array([[2, 2, 2, 2, 2]])
    assert S.visible(5, (-1, 0), pos, pre)[0].astype(int).tolist() == [
        [1, 1, 0, 0, 0], [1, 1, 0, 0, 0], [1, 1, 1, 0, 0], [0, 0, 0, 1, 1], [0, 0, 0, 1, 1]]
    # the window still cuts on the left, and a prefix past the row's end ends there
    assert S.visible(4, (1, 0), None, np.array([9]))[0].astype(int).tolist() == [[1, 1, 1, 1], [1, 1, 1, 1], [0, 1, 1, 1], [0, 0, 1, 1]]


@pytest.mark.parametrize("softcap,bias,prefix", [(2.0, False, False), (0.0, True, False), (1.5, True, True)])
def test_gradients_against_differences(softcap, bias, prefix):
    Q, K, V, dO = _qkv(2, B=1, T=5, H=2, Hkv=1)
    how = dict(softcap=softcap, slopes=np.array([0.3, 0.05]) if bias else None, prefix=np.array([3]) if prefix else None)
    grads = S.backward(dO, Q, K, V, (-1, 0), **how)
    rng = np.random.default_rng(3)
    for n, (x, g) in enumerate(zip((Q, K, V), grads)):
        for _ in range(12):
            at = tuple(rng.integers(0, s) for s in x.shape)
            args, h = [Q, K, V], 1e-6
            f = []
            for sign in (1, -1):
                args[n] = x.copy()
                args[n][at] += sign * h
                f.append((S.forward(*args, (-1, 0), **how)[0] * dO).sum())
            # truncation 1e-12 of third derivatives of order 1, rounding 1e-15 / h
            assert abs((f[0] - f[1]) / (2 * h) - g[at]) < 1e-7


ROOM = ctypes.create_string_buffer(4096)
AT = (ctypes.addressof(ROOM) + 255) & ~255  # host memory: only checks look at it


def _desc(mode=L.FC_MODE_FAST):
    t = L.FC_BF16 if mode == L.FC_MODE_FAST else L.FC_F32
    return L.AttnDesc(64, 4, 2, 16, 1, -1, 0, mode, t, t, t, t, 0)


@pytest.mark.parametrize("score,status", [
    (L.AttnScore(-1.0, 0, None, None), L.FC_ERR_INVALID_ARGUMENT),
    (L.AttnScore(float("nan"), 0, None, None), L.FC_ERR_INVALID_ARGUMENT),
    (L.AttnScore(float("inf"), 0, None, None), L.FC_ERR_INVALID_ARGUMENT),
    (L.AttnScore(4097.0, 0, None, None), L.FC_ERR_INVALID_ARGUMENT),
    (L.AttnScore(0.0009, 0, None, None), L.FC_ERR_INVALID_ARGUMENT),
    (L.AttnScore(0.0, 0, AT + 2, None), L.FC_ERR_INVALID_ARGUMENT),
    (L.AttnScore(0.0, 0, None, AT + 1), L.FC_ERR_INVALID_ARGUMENT),
])
def test_bad_scores(score, status):
    lib, d = L.lib(), _desc()
    n = ctypes.c_size_t(0)
    assert lib.fc_attn_score_fwd(ctypes.byref(d), score, AT, AT, AT, None, AT, AT, AT, None, 0, None) == status
    assert lib.fc_attn_score_bwd(ctypes.byref(d), score, *[AT] * 7, None, *[AT] * 3, AT, 1 << 20, None) == status
    assert lib.fc_attn_score_workspace_bytes(ctypes.byref(d), score, L.FC_PASS_FORWARD, 0, ctypes.byref(n)) == status


@pytest.mark.parametrize("score", [L.AttnScore(30.0, 0, None, None), L.AttnScore(0.0, 0, AT, None), L.AttnScore(0.0, 0, None, AT)])
def test_exact_mode_is_refused(score):
    lib, d = L.lib(), _desc(L.FC_MODE_EXACT)
    assert lib.fc_attn_score_fwd(ctypes.byref(d), score, AT, AT, AT, None, AT, AT, AT, None, 0, None) == L.FC_ERR_UNSUPPORTED
    assert lib.fc_attn_score_bwd(ctypes.byref(d), score, *[AT] * 7, None, *[AT] * 3, AT, 1 << 20, None) == L.FC_ERR_UNSUPPORTED


def test_the_calls_checks_still_hold():
    lib, d, score = L.lib(), _desc(), L.AttnScore(30.0, 0, None, None)
    assert lib.fc_attn_score_fwd(ctypes.byref(d), score, AT, None, AT, None, AT, AT, AT, None, 0, None) == L.FC_ERR_INVALID_ARGUMENT
    assert lib.fc_attn_score_bwd(ctypes.byref(d), score, *[AT] * 7, None, *[AT] * 3, AT, 16, None) == L.FC_ERR_WORKSPACE
    assert lib.fc_attn_score_bwd(ctypes.byref(d), score, *[AT] * 7, None, *[AT] * 3, None, 0, None) == L.FC_ERR_WORKSPACE


@pytest.mark.parametrize("T,B,positions,parts", [(1, 1, 0, 1), (333, 3, 0, 2), (333, 3, 1, 2), (2048, 1, 0, 8), (40000, 2, 1, 1)])
def test_scores_need_their_tables_and_parts_in_the_workspace(T, B, positions, parts):
    """A prefix: per 32 queries two upper bounds, and the lower ones where positions do not
    bring them.  Any score: the float32 parts of a split dK/dV where there are few key tiles."""
    lib = L.lib()
    d = L.AttnDesc(64, 4, 2, T, B, -1, 0, L.FC_MODE_FAST, *[L.FC_BF16] * 4, 0)
    got = []
    for score in (None, L.AttnScore(1.0, 0, None, None), L.AttnScore(0.0, 0, None, AT)):
        n = ctypes.c_size_t(0)
        assert lib.fc_attn_score_workspace_bytes(ctypes.byref(d), score, L.FC_PASS_BACKWARD, positions, ctypes.byref(n)) == 0
        got.append(n.value)
    room = lambda n: (n + 255) // 256 * 256  # noqa: E731
    split = 2 * room(parts * B * T * 2 * 64 * 4) if parts > 1 else 0
    n128 = B * -(-T // 128)
    order = 2 * room(n128 * 4) if positions and n128 * 4 <= 640 else 0  # small query grids take no work order
    assert got[1] - got[0] == split - order
    assert got[2] - got[1] == room(B * -(-T // 32) * 8) * (1 if positions else 2)


def test_the_causal_workspace_serves_every_window():
    lib = L.lib()
    n = ctypes.c_size_t(0)
    for T in (1, 130, 500, 1500, 4000, 9000):
        for H, Hkv in ((1, 1), (8, 1), (16, 4), (6, 3)):
            for positions in (0, 1):
                sizes = []
                for window in ((-1, 0), (0, 0), (100, 0), (700, 50), (T, T), (5, -9)):
                    d = L.AttnDesc(64, H, Hkv, T, 2, *window, L.FC_MODE_FAST, *[L.FC_BF16] * 4, 0)
                    assert lib.fc_attn_score_workspace_bytes(ctypes.byref(d), L.AttnScore(1.0, 0, None, None), L.FC_PASS_BACKWARD,
                                                             positions, ctypes.byref(n)) == 0
                    sizes.append(n.value)
                assert max(sizes) == sizes[0], (T, H, Hkv, positions, sizes)


def test_python_refusals():
    x = torch.zeros(1, 4, 2, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="HIP device"):
        F.attention(x, x, x, (-1, 0), softcap=30.0)
    with pytest.raises(TypeError, match="unexpected"):
        F.attention(x, x, x, (-1, 0), softcaps=30.0)


def _parts_bytes(T, B, H, Hkv, D, window, positions=0):
    """What a capped score adds to the backward's workspace beside the plain one's (the work
    order aside, which a score may do without)."""
    lib, got = L.lib(), []
    d = L.AttnDesc(D, H, Hkv, T, B, *window, L.FC_MODE_FAST, *[L.FC_BF16] * 4, 0)
    for score in (None, L.AttnScore(1.0, 0, None, None)):
        n = ctypes.c_size_t(0)
        assert lib.fc_attn_score_workspace_bytes(ctypes.byref(d), score, L.FC_PASS_BACKWARD, positions, ctypes.byref(n)) == 0
        got.append(n.value)
    return got[1] - got[0]


@pytest.mark.parametrize("T,B,H,Hkv,D", [(8192, 1, 64, 4, 128), (14000, 1, 64, 4, 128), (16384, 1, 128, 1, 128), (50000, 1, 32, 1, 128),
                                         (128, 440, 16, 1, 128), (6000, 9, 64, 1, 128), (4096, 1, 16, 8, 128), (1, 1, 64, 1, 16),
                                         (16384, 1, 32, 8, 128), (32768, 1, 32, 8, 128), (32768, 8, 64, 4, 128), (8192, 8, 32, 4, 128)])
def test_the_parts_of_a_split_are_bounded(T, B, H, Hkv, D):
    """At most 256 MB of float32 parts, whatever the problem's size."""
    for window in ((-1, 0), (1024, 0), (600, 300)):
        assert _parts_bytes(T, B, H, Hkv, D, window) <= (256 << 20) + 512
