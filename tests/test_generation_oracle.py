"""Text generation on the CPU: the oracle against closed forms and the training
attention's oracle, planted mistakes, the index arithmetic under sanitizers, and the
refusals of the host side (no kernel is launched)."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

import femtochat_amd as F
import femtochat_amd._lib as L
from oracle import attention_score as S
from oracle import generation as G

ROOT = Path(__file__).resolve().parents[1]


# ---- the oracle -----------------------------------------------------------------


def test_e4m3_is_torchs():
    x = np.concatenate([np.linspace(-448, 448, 20001), np.linspace(-0.05, 0.05, 20001)]).astype(np.float32)
    assert (G.round_e4m3(x) == torch.from_numpy(x).to(torch.float8_e4m3fn).float().numpy()).all()


@pytest.mark.parametrize("kind,step", [("bf16", 2.0 ** -8), ("int8", 0.5 / 127), ("fp8", 2.0 ** -4)])
def test_quantised_values_are_half_a_step_off(kind, step):
    x = np.random.default_rng(1).standard_normal((200, 64)).astype(np.float32)
    y, a = G.held(x, kind), np.abs(x).max(-1, keepdims=True)
    # int8: half a step of the head's scale; fp8: half a unit of the value, or of the smallest step 2^-9 a/448
    room = step * (a if kind == "int8" else np.maximum(np.abs(x), 2.0 ** -6 * a / 448 if kind == "fp8" else 0.0))
    assert (np.abs(y - x) <= room * (1 + 1e-5)).all()


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_heads_without_a_scale(kind):
    x = np.zeros((5, 16), np.float32)
    x[1] = 2.0 ** -110
    x[2, 3], x[3, 5], x[4] = np.inf, np.nan, np.linspace(-1, 1, 16)
    y = G.held(x, kind)
    assert (y[:2] == 0).all() and np.isnan(y[2:4]).all() and abs(y[4, -1] - 1) < 1e-6


@pytest.mark.parametrize("left,softcap,bias", [(-1, 0.0, False), (3, 0.0, False), (-1, 2.0, True), (2, 1.5, True)])
def test_a_run_is_the_training_attentions_last_rows(left, softcap, bias):
    rng = np.random.default_rng(2)
    T, H, Hkv, D, N = 9, 4, 2, 16, 4
    Q, K, V = (rng.standard_normal((1, T, h, D)) for h in (H, Hkv, Hkv))
    slopes = np.array([0.5, 0.25, 0.125, 0.0625]) if bias else None
    O = S.forward(Q, K, V, (left, 0), softcap=softcap, slopes=slopes)[0][0, -N:]
    got = G.attend(Q[0, -N:], K[0], V[0], T - N, N, left, None, softcap, slopes)
    np.testing.assert_allclose(got, O, rtol=1e-12, atol=1e-12)


def test_a_tree_is_its_paths():
    """Each node's row is the last row of its root-to-node path run alone."""
    rng = np.random.default_rng(3)
    n, H, Hkv, D, parents = 6, 2, 1, 16, [-1, 0, 0, 1, 1, 2, 5, -1]
    N = len(parents)
    Q, K, V = rng.standard_normal((N, H, D)), rng.standard_normal((n + N, Hkv, D)), rng.standard_normal((n + N, Hkv, D))
    for left in (-1, 2, 7):
        got = G.attend(Q, K, V, n, N, left, parents, 0.0, [0.3, 0.1])
        for i, line in enumerate(G.lineage(parents, N)):
            rows = list(range(n)) + [n + j for j in line]
            alone = G.attend(Q[line], K[rows], V[rows], n, len(line), left, None, 0.0, [0.3, 0.1])
            np.testing.assert_allclose(got[i], alone[-1], rtol=1e-12)
    # what a wrong mask would do
    assert not np.allclose(G.attend(Q, K, V, n, N, -1, None)[3], G.attend(Q, K, V, n, N, -1, parents)[3])


def test_parents_that_are_no_tree():
    assert G.lineage([-1, 0, 5, 2, 1], 5) == [[0], [0, 1], None, None, [0, 1, 4]]
    assert G.lineage([-2, 0], 2) == [None, None] and G.lineage([0], 1) == [None]


def _emitted(verify, p0, draw_token, grid):
    """The distribution of the first token behind the root, over a grid of the random numbers."""
    out = np.zeros(len(p0))
    for weight, tokens, us in grid:
        out[verify(tokens, us)] += weight
    return out


def test_draws_keep_the_targets_distribution():
    """Over the drafted token, its u on a grid and the exact distribution of what is drawn instead."""
    rng = np.random.default_rng(4)
    V = 5
    x, d = rng.standard_normal((2, V)) * 2, rng.standard_normal((1, V)) * 2
    p, q = G.softmax(x[0], 0.7), G.softmax(d[0], 0.7)
    M, got = 400, np.zeros(V)
    for y in range(V):
        for k in range(M):
            for u0 in (np.arange(50) + 0.5) / 50:
                path, token = G.verify(x, [0, y], [u0, (k + 0.5) / M], d, temperature=0.7)
                got[y if len(path) == 2 else token] += q[y] / (M * 50)
    assert np.abs(got - p).max() < 2 * (1 / M + 1 / 50)  # the grids' steps
    assert np.abs(q - p).max() > 0.1


def test_candidates_keep_the_targets_distribution():
    rng = np.random.default_rng(5)
    V, M = 6, 40
    x = np.tile(rng.standard_normal(V) * 1.5, (4, 1))
    p, got, grid = G.softmax(x[0], 1.0), np.zeros(V), (np.arange(M) + 0.5) / M
    for a in grid:
        for b in grid:
            for u0 in grid:
                path, token = G.verify(x, [0, 2, 4, 2], [u0, a, b, 0.0], parents=[-1, 0, 0, 0])  # the second 2 is never taken
                assert path in ([0], [0, 1], [0, 2])
                got[[token, 2, 4][path[-1]]] += M ** -3.0
    assert np.abs(got - p).max() < 3 / M


def test_a_mistaken_rule_is_seen():
    """Testing a second candidate against p itself, not against what is left, moves the distribution."""
    p = np.array([0.5, 0.3, 0.2])
    right = np.array([p[0], (1 - p[0]) * min(1, p[1] / (1 - p[0])), 0])
    wrong = np.array([p[0], (1 - p[0]) * p[1], 0])
    assert abs(right[1] - p[1]) < 1e-12 and abs(wrong[1] - p[1]) > 0.1


def test_walks_by_hand():
    x = np.log(np.array([[0.1, 0.6, 0.3], [0.2, 0.2, 0.6], [0.5, 0.4, 0.1]]))
    assert G.verify(x, [0, 1, 2], [0.0, 0.59, 0.5]) == ([0, 1, 2], 0)
    assert G.verify(x, [0, 1, 2], [0.5, 0.61, 0.5]) == ([0], 2)        # 1 is struck: 0.1, 0.3 -> 0.5 of 0.4
    assert G.verify(x, [0, 1, 2], [0.2, 0.61, 0.5]) == ([0], 0)
    assert G.verify(x, [0, 1, 2], [0.95, 0.1, 0.7], count=2) == ([0, 1], 2)
    assert G.verify(x, [0, 1, 1], [0.0] * 3, temperature=0) == ([0, 1], 2)
    assert G.verify(x, [0, 2, 1], [0.0] * 3, parents=[-1, 0, 0], temperature=0) == ([0, 2], 0)
    assert G.verify(x, [0, 1, 2], [0.0] * 3, count=0) == ([], -1)
    x[1, 0] = np.nan
    assert G.verify(x, [0, 1, 2], [0.0] * 3) == ([0, 1], -1)


# ---- index arithmetic under sanitizers -------------------------------------------


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_cache_index_arithmetic_under_sanitizers(tmp_path):
    """Pages, places, slots and masks (csrc/cache_index.hpp) over lengths, tables and trees of any values."""
    exe = tmp_path / "harness"
    r = subprocess.run(["g++", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-g", "-O1", "-std=c++17", "-Wall", "-Werror",
                        str(ROOT / "tests" / "sanitize" / "cache_harness.cpp"), "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300, env={"PATH": "/usr/bin:/bin"})
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout + r.stderr


# ---- refusals ---------------------------------------------------------------------

FAKE = 0x10000  # an aligned address; nothing is read before the checks fail


def _cache_desc(**kw):
    return L.CacheDesc(**{**dict(D=64, Hkv=2, B=2, layers=1, pages=2, page_size=64, max_pages=0, type=L.FC_CACHE_I8), **kw})


def _cache(**kw):
    return L.Cache(**{**dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, table=None), **kw})


def _last():
    return L.lib().fc_last_error().decode()


BAD_CACHES = [
    (dict(D=24), {}, "head_dim"), (dict(D=144), {}, "head_dim"), (dict(Hkv=0), {}, "positive"), (dict(B=-1), {}, "positive"),
    (dict(type=0), {}, "type"), (dict(type=4), {}, "type"), (dict(page_size=40), {}, "multiple of 16"),
    (dict(page_size=48, max_pages=2), dict(table=FAKE), "power of two"), (dict(pages=3), {}, "one page"),
    (dict(max_pages=-1), {}, "max_pages"), (dict(page_size=1 << 29), {}, "2^28"), (dict(max_pages=1 << 23), dict(table=FAKE), "2^28"),
    ({}, dict(k=None), "null"), ({}, dict(v_scale=None), "scales"), (dict(max_pages=2), {}, "table"), ({}, dict(k=FAKE + 8), "aligned"),
    ({}, dict(k_scale=FAKE + 4), "aligned"),
]


@pytest.mark.parametrize("d,c,what", BAD_CACHES, ids=[f"{b[0]}{b[1]}" for b in BAD_CACHES])
def test_bad_caches_are_refused(d, c, what):
    lib, d, c = L.lib(), _cache_desc(**d), _cache(**c)
    o = L.CachedAttnOptions(4, 1, -1, 0, 0.0, None)
    for st in (lib.fc_cache_write(d, c, FAKE, FAKE, L.FC_BF16, 4, FAKE, None, None),
               lib.fc_cache_read(d, c, FAKE, FAKE, L.FC_BF16, 4, None, None, None),
               lib.fc_cache_keep(d, c, 4, FAKE, FAKE, None, None),
               lib.fc_cached_attn(d, c, o, FAKE, FAKE, FAKE, None, None, None, 0, None)):
        assert st in (L.FC_ERR_INVALID_ARGUMENT, L.FC_ERR_UNSUPPORTED) and what in _last(), _last()


def test_null_and_unaligned_pointers_are_refused():
    lib, d, c = L.lib(), _cache_desc(), _cache()
    assert lib.fc_cache_write(None, c, FAKE, FAKE, 1, 4, FAKE, None, None) == L.FC_ERR_INVALID_ARGUMENT
    assert lib.fc_cache_write(d, None, FAKE, FAKE, 1, 4, FAKE, None, None) == L.FC_ERR_INVALID_ARGUMENT
    for args in ((None, FAKE, 1, 4, FAKE), (FAKE, FAKE, 1, 4, None), (FAKE + 2, FAKE, 1, 4, FAKE), (FAKE, FAKE, 7, 4, FAKE),
                 (FAKE, FAKE, 1, 0, FAKE), (FAKE, FAKE, 1, 4, FAKE + 1)):
        assert lib.fc_cache_write(d, c, *args, None, None) == L.FC_ERR_INVALID_ARGUMENT, args
    assert lib.fc_cache_keep(d, c, 4, None, FAKE, None, None) == L.FC_ERR_INVALID_ARGUMENT
    assert lib.fc_cache_keep(d, c, 4, FAKE, FAKE + 2, None, None) == L.FC_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("kw,what", [
    (dict(H=3), "multiple of Hkv"), (dict(N=0), "1 to 64"), (dict(N=65), "1 to 64"), (dict(left=-2), "left"), (dict(tree=3), "tree"),
    (dict(softcap=-1.0), "softcap"), (dict(softcap=5000.0), "softcap"), (dict(softcap=float("nan")), "softcap"), (dict(slopes=FAKE + 2), "aligned"),
    (dict(tree=1), "parents"),
])
def test_bad_options_are_refused(kw, what):
    o = L.CachedAttnOptions(**{**dict(H=4, N=2, left=-1, tree=0, softcap=0.0, slopes=None), **kw})
    st = L.lib().fc_cached_attn(_cache_desc(), _cache(), o, FAKE, FAKE, FAKE, None, None, FAKE, 1 << 40, None)
    assert st in (L.FC_ERR_INVALID_ARGUMENT, L.FC_ERR_UNSUPPORTED) and what in _last(), _last()


def test_workspaces_and_layers():
    lib, n = L.lib(), ctypes.c_size_t(7)
    o = L.CachedAttnOptions(4, 1, -1, 0, 0.0, None)
    assert lib.fc_cached_attn_workspace_bytes(_cache_desc(), o, ctypes.byref(n)) == L.FC_OK and n.value == 0  # 64 tokens: one part
    big = _cache_desc(page_size=4096)
    assert lib.fc_cached_attn_workspace_bytes(big, o, ctypes.byref(n)) == L.FC_OK and n.value > 0
    st = lib.fc_cached_attn(big, _cache(), o, FAKE, FAKE, FAKE, None, None, FAKE, n.value - 1, None)
    assert st == L.FC_ERR_WORKSPACE
    assert lib.fc_cached_attn(big, _cache(), o, FAKE, FAKE, FAKE, None, None, FAKE + 16, n.value, None) == L.FC_ERR_WORKSPACE
    assert lib.fc_cached_attn(_cache_desc(layers=2), _cache(), o, FAKE, FAKE, FAKE, None, None, None, 0, None) == L.FC_ERR_INVALID_ARGUMENT
    assert "one layer" in _last()
    assert lib.fc_cached_attn(_cache_desc(), _cache(), o, FAKE, FAKE + 8, FAKE, None, None, None, 0, None) == L.FC_ERR_INVALID_ARGUMENT


def _verify_desc(**kw):
    return L.VerifyDesc(**{**dict(B=2, N=4, V=100, dtype=L.FC_F32, index_type=1, tree=0, has_draft=1, temperature=1.0), **kw})


@pytest.mark.parametrize("kw,what", [
    (dict(B=0), "positive"), (dict(N=65), "64 nodes"), (dict(V=0), "positive"), (dict(dtype=3), "dtype"), (dict(index_type=2), "index_type"),
    (dict(tree=3), "tree"), (dict(tree=1), "draft_logits"), (dict(temperature=-1.0), "temperature"), (dict(temperature=1e-5), "temperature"),
    (dict(temperature=float("nan")), "temperature"), (dict(B=60000, N=64, V=100000), "too many"), (dict(V=1 << 27), "vocabulary"),
])
def test_bad_verifications_are_refused(kw, what):
    n = ctypes.c_size_t(0)
    d = _verify_desc(**kw)
    assert L.lib().fc_verify_workspace_bytes(d, ctypes.byref(n)) in (L.FC_ERR_INVALID_ARGUMENT, L.FC_ERR_UNSUPPORTED)
    assert what in _last(), _last()
    st = L.lib().fc_verify_drafts(d, FAKE, FAKE, FAKE, FAKE, FAKE if d.tree else None, None, FAKE, FAKE, FAKE, FAKE, 1 << 40, None)
    assert st in (L.FC_ERR_INVALID_ARGUMENT, L.FC_ERR_UNSUPPORTED) and what in _last()


def test_verification_pointers_and_workspace():
    lib, d, n = L.lib(), _verify_desc(V=2048), ctypes.c_size_t(0)
    assert lib.fc_verify_workspace_bytes(d, ctypes.byref(n)) == L.FC_OK and n.value == 0
    d = _verify_desc(V=2049)
    assert lib.fc_verify_workspace_bytes(d, ctypes.byref(n)) == L.FC_OK and n.value > 0
    ok = [FAKE, FAKE, FAKE, FAKE, None, None, FAKE, FAKE, FAKE, FAKE, n.value, None]
    for at in (0, 1, 2, 3, 6, 7, 8):
        args = list(ok)
        args[at] = None
        assert lib.fc_verify_drafts(d, *args) == L.FC_ERR_INVALID_ARGUMENT, at
    for at, p in ((0, FAKE + 2), (2, FAKE + 4), (3, FAKE + 1), (4, FAKE), (6, FAKE + 2)):
        args = list(ok)
        args[at] = p
        assert lib.fc_verify_drafts(d, *args) == L.FC_ERR_INVALID_ARGUMENT, at
    for at, p in ((9, None), (10, n.value - 1), (9, FAKE + 128)):
        args = list(ok)
        args[at] = p
        assert lib.fc_verify_drafts(d, *args) == L.FC_ERR_WORKSPACE, at


def test_the_host_side_refuses_before_any_launch():
    with pytest.raises(ValueError, match="HIP device"):
        c = F.kv_cache(2, 100, 2, 64, torch.int8, device="cpu")
        F.cache_read(c, None, 4)
    assert c.k.shape == (2, 2, 112, 64) and c.capacity == 112
    paged = F.kv_cache(3, 100, 2, 64, page=32, pool=10, layers=5, device="cpu")
    assert paged.k.shape == (5, 10, 2, 32, 64) and paged.capacity == 128 and paged.k_scale is None
    assert paged.pages.tolist() == [[0, 1, 2, 3], [4, 5, 6, 7], [8, 9, -1, -1]]
    assert paged.layer(2).k.shape == (10, 2, 32, 64)
    for bad in (dict(page=24), dict(page=8), dict(pool=3), dict(layers=0)):
        with pytest.raises(ValueError):
            F.kv_cache(2, 100, 2, 64, device="cpu", **bad)
    with pytest.raises(TypeError):
        F.kv_cache(2, 100, 2, 64, torch.float16, device="cpu")
    with pytest.raises(ValueError, match="one layer"):
        c.layer(0)
    with pytest.raises(ValueError, match="HIP device"):
        F.verify_drafts(torch.zeros(1, 2, 8), torch.zeros(1, 2, dtype=torch.int64), torch.zeros(1, 2))
