"""GPU parity of the cache, its attention and the verification of drafted tokens against
the oracle (oracle/generation.py).

Tolerances.  Codes and scales are float32 operations that the oracle repeats: equal.
Attention: a score is a float32 sum of D <= 128 products, within 127 2^-24 of the sum of
their magnitudes, below 14 in units of the score here (q and k near 2 and 1.2 in size,
divided by sqrt(D)): 1.1e-4; the exponential (2^-22), the scales' and the cap's roundings
(30 2^-21) add under 5e-5.  So p is within 1.6e-4 of itself, its sum too, and O within
3.2e-4 of the largest value of its column; P as two bf16 values adds 2^-16.  O's rounding
to bf16 is 2^-8 of it.  Verification: whole numbers, equal."""
import numpy as np
import pytest
import torch

import femtochat_amd as F
from oracle import generation as G

pytestmark = pytest.mark.gpu
KINDS = {"bf16": torch.bfloat16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}
O_ROOM, O_HALF_STEP = 4e-4, 2.0 ** -8


def _dev(gpu, *arrays):
    out = [None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(gpu) for a in arrays]
    return out if len(out) > 1 else out[0]


def _junk(cache):
    """Fills a cache with what is no number: nothing of it may reach a result."""
    for t in (cache.k, cache.v):
        t.view(torch.uint8).fill_(0x7F)  # bf16 and e4m3 NaN; int8 127
        if t.dtype == torch.bfloat16:
            t.fill_(float("nan"))
    for t in (cache.k_scale, cache.v_scale):
        if t is not None:
            t.fill_(float("nan"))
    return cache


def _shuffled(cache, seed):
    """The same cache with its pages handed out in a random order."""
    if cache.pages is None:
        return cache
    P = cache.k.shape[-4]
    order = torch.from_numpy(np.random.default_rng(seed).permutation(P)[:cache.pages.numel()].astype(np.int32))
    cache.pages.copy_(order.view(cache.pages.shape))
    return cache


def _where(cache, b, t):
    """(page, place) of sequence b's token t."""
    S = cache.k.shape[-2]
    return (b, t) if cache.pages is None else (int(cache.pages[b, t // S]), t % S)


def _values(rng, *shape, dtype=torch.bfloat16):
    return (1.2 * torch.from_numpy(rng.standard_normal(shape, dtype=np.float32))).to(dtype)


# ---- write, read, keep --------------------------------------------------------------


@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("kind,source,page", [("int8", torch.bfloat16, None), ("fp8", torch.float32, 16), ("bf16", torch.float32, 32),
                                              ("int8", torch.float32, 64), ("fp8", torch.bfloat16, None), ("bf16", torch.bfloat16, None)])
def test_written_tokens_read_back(gpu, kind, source, page, D):
    rng = np.random.default_rng(D)
    B, T, Hkv, layers, lengths, counts = 3, 21, 3, 2, np.array([0, 5, 43], np.int32), np.array([21, 0, 13], np.int32)
    cache = _shuffled(_junk(F.kv_cache(B, 64, Hkv, D, KINDS[kind], layers=layers, page=page, device=gpu)), D)
    before = [None if t is None else t.clone() for t in cache[:4]]
    K, V = (_values(rng, layers, B, T, Hkv, D, dtype=source) for _ in range(2))
    K[0, 0, 0, 0], V[1, 2, 3, 1] = 0.0, 2.0 ** -120
    K[1, 0, 4, 2, 3], V[0, 0, 5, 0, 1], V[0, 0, 6, 0, 0] = float("inf"), float("nan"), 1e30
    n, c = _dev(gpu, lengths, counts)
    F.cache_write_(cache, K.to(gpu), V.to(gpu), n, c)
    for x, now, scale, old, old_scale in ((K, cache.k, cache.k_scale, *before[0::2]), (V, cache.v, cache.v_scale, *before[1::2])):
        codes, scales = G.quantise(x.float().numpy(), kind)
        want, wants = old.float().cpu().numpy(), None if scales is None else old_scale.cpu().numpy()
        for b in range(B):
            for t in range(counts[b]):
                p, at = _where(cache, b, int(lengths[b]) + t)
                want[:, p, :, at] = codes[:, b, t]
                if scales is not None:
                    wants[:, p, :, at] = scales[:, b, t]
        np.testing.assert_array_equal(now.float().cpu().numpy(), want)
        if scales is not None:
            np.testing.assert_array_equal(scale.cpu().numpy(), wants)
    for dtype in (torch.float32, torch.bfloat16):
        for x, y in zip((K, V), F.cache_read(cache, n, T, c, dtype=dtype)):
            want = torch.from_numpy(G.held(x.float().numpy(), kind)) * (torch.arange(T)[:, None, None] < torch.from_numpy(counts)[:, None, None, None])
            np.testing.assert_array_equal(np.where(torch.isnan(want) & (torch.arange(T)[:, None, None] >= torch.from_numpy(counts)[:, None, None, None]), 0.0,
                                                   want.to(dtype).float().numpy()), y.float().cpu().numpy())


def test_tokens_beyond_the_capacity_and_on_bad_pages(gpu):
    """They are not written and read as NaN; the pool's other rows keep their values."""
    rng = np.random.default_rng(1)
    cache = F.kv_cache(2, 32, 2, 64, torch.int8, page=16, pool=5, device=gpu)
    cache.pages.copy_(torch.tensor([[3, -1], [7, 1]], dtype=torch.int32))
    K, V = (_values(rng, 2, 20, 2, 64).to(gpu) for _ in range(2))
    F.cache_write_(cache, K, V, _dev(gpu, np.array([0, 14], np.int32)))
    assert (cache.k[[0, 2, 4]] == 0).all() and (cache.v_scale[[0, 2, 4]] == 0).all()
    k, _ = F.cache_read(cache, None, 40, dtype=torch.float32)
    held = torch.from_numpy(G.held(K.float().cpu().numpy(), "int8"))
    assert torch.equal(k[0, :16].cpu(), held[0, :16]) and torch.isnan(k[0, 16:]).all()
    assert torch.isnan(k[1, :16]).all() and torch.equal(k[1, 16:32].cpu(), held[1, 2:18]) and torch.isnan(k[1, 32:]).all()
    for n in (-5, 32, 33, 2 ** 31 - 1, -2 ** 31):  # lengths that leave no room, or are none
        fresh = F.kv_cache(1, 32, 2, 64, torch.int8, device=gpu)
        F.cache_write_(fresh, K[:1], V[:1], _dev(gpu, np.array([n], np.int32)))
        assert int((fresh.k_scale != 0).sum()) == (40 if n < 0 else 0)  # (below 0 is 0)


@pytest.mark.parametrize("kind,page,D", [("bf16", None, 16), ("int8", 16, 128), ("fp8", 32, 48), ("int8", None, 80)])
def test_kept_paths_move_to_the_front(gpu, kind, page, D):
    rng = np.random.default_rng(5)
    B, N, Hkv, layers = 5, 12, 3, 2
    cache = _shuffled(F.kv_cache(B, 60, Hkv, D, KINDS[kind], layers=layers, page=page, device=gpu), 3)
    K, V = (_values(rng, layers, B, 60, Hkv, D).to(gpu) for _ in range(2))
    F.cache_write_(cache, K, V, torch.zeros(B, dtype=torch.int32, device=gpu))
    lengths, kept = np.array([0, 7, 30, 48, 13], np.int32), np.array([12, 1, 4, 6, 0], np.int32)
    path = np.full((B, N), -1, np.int32)
    for b in range(B):
        path[b, :kept[b]] = np.sort(rng.choice(N, kept[b], replace=False))
    path[1, 0], path[2, :4] = 0, [0, 1, 2, 3]
    before = F.cache_read(cache, None, 60, dtype=torch.float32)
    F.cache_keep_(cache, *_dev(gpu, lengths, path, kept))
    for old, new in zip(before, F.cache_read(cache, None, 60, dtype=torch.float32)):
        want = old.clone()
        for b in range(B):
            for j in range(kept[b]):
                want[:, b, lengths[b] + j] = old[:, b, lengths[b] + path[b, j]]
        assert torch.equal(new, want)


def test_a_path_of_all_nodes_over_many_layers_and_bad_entries(gpu):
    """64 nodes, each moved by one; entries that are no nodes move nothing."""
    cache = F.kv_cache(1, 80, 2, 64, torch.int8, layers=3, device=gpu)
    K = _values(np.random.default_rng(6), 3, 1, 80, 2, 64).to(gpu)
    F.cache_write_(cache, K, K, _dev(gpu, np.array([0], np.int32)))
    old = F.cache_read(cache, None, 80, dtype=torch.float32)[0]
    F.cache_keep_(cache, *_dev(gpu, np.array([10], np.int32), np.arange(1, 65, dtype=np.int32)[None], np.array([63], np.int32)))
    new = F.cache_read(cache, None, 80, dtype=torch.float32)[0]
    assert torch.equal(new[:, :, 10:73], old[:, :, 11:74]) and torch.equal(new[:, :, :10], old[:, :, :10])
    F.cache_keep_(cache, *_dev(gpu, np.array([10], np.int32), np.array([[-1, 99, 2 ** 31 - 1, -2 ** 31]], np.int32), np.array([9], np.int32)))
    assert torch.equal(F.cache_read(cache, None, 80, dtype=torch.float32)[0], new)


# ---- attention ----------------------------------------------------------------------


def _tree(rng, N):
    return np.array([-1] + [int(rng.integers(0, i)) for i in range(1, N)], np.int32)


def _filled(gpu, rng, kind, lengths, counts, N, Hkv, D, capacity, page):
    """A cache of junk that holds the sequences, and what it holds of them (float32)."""
    B = len(lengths)
    cache = _shuffled(_junk(F.kv_cache(B, capacity, Hkv, D, KINDS[kind], page=page, device=gpu)), 7)
    T = max(1, max(int(n) + int(c) for n, c in zip(lengths, counts)))
    K, V = _values(rng, B, T, Hkv, D), _values(rng, B, T, Hkv, D)
    F.cache_write_(cache, K.to(gpu), V.to(gpu), torch.zeros(B, dtype=torch.int32, device=gpu),
                   _dev(gpu, np.asarray(lengths, np.int32) + np.asarray(counts, np.int32)))
    return cache, G.held(K.float().numpy(), kind), G.held(V.float().numpy(), kind)


def _check(O, want, V):
    """O (N, H, D) against the oracle's; V (keys, Hkv, D)."""
    O = O.double().cpu().numpy()
    assert (np.isnan(O) == np.isnan(want)).all()
    most = np.repeat(np.abs(V).max(0) if len(V) else np.zeros(V.shape[1:]), O.shape[1] // V.shape[1], 0)
    over = np.abs(O - want) - O_HALF_STEP * np.abs(want) - O_ROOM * most[None]
    assert np.nanmax(over, initial=-1.0) <= 0, (np.nanmax(over), np.nanmax(np.abs(O - want)))


def _compare(gpu, rng, kind, lengths, counts, N, H, Hkv, D, capacity, page=None, left=-1, softcap=0.0, bias=False, tree="run", ragged=True):
    B = len(lengths)
    cache, K, V = _filled(gpu, rng, kind, lengths, counts, N, Hkv, D, capacity, page)
    Q = (2.0 * torch.from_numpy(rng.standard_normal((B, N, H, D), dtype=np.float32))).bfloat16()
    slopes = (2.0 ** (-8.0 * (np.arange(H) + 1) / H)).astype(np.float32) if bias else None
    parents = None if tree == "run" else _tree(rng, N) if tree == "one" else np.stack([_tree(rng, N) for _ in range(B)])
    n, c, up, sl = (_dev(gpu, a) for a in (np.asarray(lengths, np.int32), np.asarray(counts, np.int32) if ragged else None, parents, slopes))
    O = F.cached_attention(Q.to(gpu), cache, n, (left, 0), counts=c, parents=up, softcap=softcap, slopes=sl)
    for b in range(B):
        m = int(lengths[b]) + int(counts[b])
        want = G.attend(Q[b].double().numpy(), K[b, :m], V[b, :m], int(lengths[b]), int(counts[b]), left,
                        None if parents is None else parents if parents.ndim == 1 else parents[b], softcap, slopes)
        _check(O[b], want, V[b, :m])
    return O


@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("kind", list(KINDS))
def test_single_tokens_of_ragged_sequences(gpu, kind, D):
    lengths = [0, 1, 15, 16, 31, 32, 33, 127, 200]
    _compare(gpu, np.random.default_rng(D), kind, lengths, [1] * 8 + [0], 1, 6, 2, D, 256, page=16 if D % 32 else None)


@pytest.mark.parametrize("N,H,Hkv,tree", [(2, 4, 4, "run"), (5, 8, 2, "each"), (13, 8, 8, "each"), (16, 4, 1, "one"), (17, 2, 2, "run"),
                                          (31, 6, 2, "each"), (64, 4, 2, "each"), (64, 1, 1, "run"), (33, 16, 2, "one")])
@pytest.mark.parametrize("kind,D,page", [("bf16", 128, 32), ("int8", 128, None), ("fp8", 64, 16), ("bf16", 64, None), ("int8", 96, 64)])
def test_runs_and_trees(gpu, kind, D, page, N, H, Hkv, tree):
    rng = np.random.default_rng(N + D)
    lengths = [0, 3, 29, 64, 130]
    _compare(gpu, rng, kind, lengths, [N, max(1, N // 2), N, 1, N], N, H, Hkv, D, 224, page, tree=tree)


@pytest.mark.parametrize("left", [0, 1, 5, 31, 64, 1000])
@pytest.mark.parametrize("softcap,bias", [(0.0, False), (30.0, True)])
def test_windows_caps_and_biases(gpu, left, softcap, bias):
    rng = np.random.default_rng(left)
    for kind, tree, N in (("int8", "each", 9), ("bf16", "run", 40), ("fp8", "each", 1)):
        _compare(gpu, rng, kind, [0, 2, 63, 100, 333], [N] * 5, N, 4, 2, 64, 400, 16, left, softcap, bias, tree, ragged=False)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("N,H,Hkv,D", [(1, 8, 1, 128), (1, 2, 1, 48), (7, 4, 2, 64), (32, 4, 2, 128)])
def test_long_sequences_in_parts(gpu, kind, N, H, Hkv, D):
    """Enough tiles for several slots per sequence, and a batch of very unlike lengths."""
    rng = np.random.default_rng(N)
    _compare(gpu, rng, kind, [5000, 3, 1234], [N, N, 1], N, H, Hkv, D, 5120, 64, tree="each", ragged=True)
    _compare(gpu, rng, kind, [9000], [N], N, H, Hkv, D, 9088, None, left=700, tree="run", ragged=False)


def test_many_sequences(gpu):
    """More sequences than a wave has lanes: each with a workgroup of its own, in parts, and
    several to a share."""
    rng = np.random.default_rng(8)
    lengths = rng.integers(0, 700, 150)
    _compare(gpu, rng, "int8", lengths, rng.integers(0, 3, 150), 2, 2, 1, 64, 768, 64, tree="run")
    _compare(gpu, rng, "fp8", rng.integers(0, 1500, 150), rng.integers(0, 3, 150), 2, 2, 1, 64, 1600, 64, tree="run")
    _compare(gpu, rng, "int8", rng.integers(0, 90, 300), rng.integers(0, 3, 300), 2, 20, 2, 32, 768, 64, tree="run")  # (more than a CU has room for)
    lengths = np.where(rng.integers(0, 20, 150) > 0, rng.integers(0, 40, 150), 1500)
    _compare(gpu, rng, "bf16", lengths, rng.integers(0, 4, 150), 3, 64, 8, 32, 1600, 16, tree="each")


def test_thousands_of_sequences(gpu):
    """A line far longer than the shares' least, whose beginning takes many chunks of lengths."""
    rng = np.random.default_rng(40)
    B, Hkv, H, D, T = 5000, 1, 3, 16, 1024
    cache = F.kv_cache(B, 1600, Hkv, D, torch.int8, device=gpu)
    lengths = torch.from_numpy(np.where(rng.integers(0, 50, B) > 0, rng.integers(0, 60, B), 1023).astype(np.int32))
    K, V = (1.2 * torch.randn(B, T, Hkv, D, generator=torch.Generator().manual_seed(i)) for i in (1, 2))
    F.cache_write_(cache, K.to(gpu), V.to(gpu), torch.zeros(B, dtype=torch.int32, device=gpu))
    Q = (2.0 * torch.from_numpy(rng.standard_normal((B, 1, H, D), dtype=np.float32))).bfloat16()
    O = F.cached_attention(Q.to(gpu), cache, lengths.to(gpu))
    assert torch.isfinite(O).all()
    for b in [0, 63, 64, B - 1] + rng.integers(0, B, 20).tolist() + torch.nonzero(lengths == 1023)[:20, 0].tolist():
        n = int(lengths[b])
        Kh, Vh = (G.held(x[b:b + 1, :n + 1].numpy(), "int8")[0] for x in (K, V))
        _check(O[b], G.attend(Q[b].double().numpy(), Kh, Vh, n, 1), Vh)


def test_scores_that_grow_along_the_keys(gpu):
    """References move, upwards by far, and a first key may be all there is."""
    rng = np.random.default_rng(9)
    cache, K, V = _filled(gpu, rng, "bf16", [600], [3], 3, 1, 64, 640, None)
    grow = np.linspace(0.0, 30.0, K.shape[1], dtype=np.float32)[None, :, None, None]
    Kb = torch.from_numpy(K * (0.05 + grow)).bfloat16()
    F.cache_write_(cache, Kb.to(gpu), torch.from_numpy(V).bfloat16().to(gpu), torch.zeros(1, dtype=torch.int32, device=gpu))
    Q = torch.from_numpy(rng.standard_normal((1, 3, 2, 64), dtype=np.float32)).bfloat16()
    for sign in (1.0, -1.0):
        O = F.cached_attention((sign * Q).to(gpu), cache, _dev(gpu, np.array([600], np.int32)))
        want = G.attend(sign * Q[0].double().numpy(), Kb[0].double().numpy(), V[0], 600, 3)
        # scores up to 8 sqrt(64) 30 1.2 / 8: their roundings are 30 times the others
        assert np.abs(O[0].double().cpu().numpy() - want).max() < 2.0 ** -8 * np.abs(want).max() + 30 * O_ROOM * np.abs(V).max()


@pytest.mark.parametrize("N,H", [(1, 2), (3, 12)])
def test_scores_far_below_zero(gpu, N, H):
    """Every score of a row near -4e32: equal ones share, and a smaller one has nothing."""
    D, n = 16, 900
    cache = F.kv_cache(1, 1600, 1, D, torch.bfloat16, device=gpu)
    K, V = torch.full((1, n + N, 1, D), 1e16), torch.randn(1, n + N, 1, D)
    K[0, :n // 2] = 2e16
    F.cache_write_(cache, K.to(gpu), V.to(gpu), torch.zeros(1, dtype=torch.int32, device=gpu))
    Q = torch.full((1, N, H, D), -1e16, dtype=torch.bfloat16, device=gpu)
    O = F.cached_attention(Q, cache, _dev(gpu, np.array([n], np.int32)))[0]
    Kh, Vh = G.held(K.numpy(), "bf16")[0], G.held(V.numpy(), "bf16")[0]
    _check(O, G.attend(Q[0].double().cpu().numpy(), Kh, Vh, n, N), Vh)


@pytest.mark.parametrize("H,n,capacity", [(4, 90, 128), (12, 90, 128), (12, 1100, 1600)])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_what_a_node_does_not_see_does_not_reach_it(gpu, value, H, n, capacity):
    """Keys and values that are no numbers at siblings, before the window and behind the sequence."""
    rng = np.random.default_rng(10)
    N, Hkv, D = 6, 2, 64
    parents = np.array([-1, 0, 0, 1, 2, 4], np.int32)
    for kind, left in (("bf16", -1), ("bf16", 20), ("int8", -1), ("fp8", 20)):
        cache, K, V = _filled(gpu, rng, kind, [n], [N], N, Hkv, D, capacity, 16)
        Kb, Vb = (_values(rng, 1, n + N, Hkv, D).float() for _ in range(2))
        Kb[0, n + 3, 0, 5], Vb[0, n + 3, :, 7] = value, value  # node 3: only its own row sees it
        if left > 0:
            Kb[0, :60], Vb[0, 3:n - left] = value, value     # (the root sees from n - 20 on)
        F.cache_write_(cache, Kb.to(gpu), Vb.to(gpu), torch.zeros(1, dtype=torch.int32, device=gpu))
        Q = (2.0 * torch.from_numpy(rng.standard_normal((1, N, H, D), dtype=np.float32))).bfloat16()
        O = F.cached_attention(Q.to(gpu), cache, _dev(gpu, np.array([n], np.int32)), (left, 0), parents=_dev(gpu, parents))[0]
        Kh, Vh = G.held(Kb.numpy(), kind)[0], G.held(Vb.numpy(), kind)[0]
        clean_k, clean_v = np.where(np.isfinite(Kh), Kh, 0.0), np.where(np.isfinite(Vh), Vh, 0.0)
        want = G.attend(Q[0].double().numpy(), clean_k, clean_v, n, N, left, parents)
        others = [0, 1, 2, 4, 5]
        _check(O[others], want[others], clean_v)
        assert not torch.isfinite(O[3, :, 7]).any()
        if kind == "bf16":  # KV head 1's keys are numbers: its queries' other columns are too, and the column is what was put there
            assert torch.isfinite(O[3, H // 2:, :7]).all()
            assert torch.equal(O[3, H // 2:, 7].float().cpu(), torch.full((H // 2,), value)) or (
                np.isnan(value) and torch.isnan(O[3, H // 2:, 7]).all())


def test_nodes_that_are_no_trees_and_lie_beyond_the_capacity(gpu):
    rng = np.random.default_rng(11)
    cache, K, V = _filled(gpu, rng, "int8", [27], [5], 5, 1, 32, 32, 16)
    Q = torch.from_numpy(rng.standard_normal((1, 5, 2, 32), dtype=np.float32)).bfloat16()
    n = _dev(gpu, np.array([20], np.int32))
    for parents in ([-1, 0, 2, 1, 7], [-1, 0, -2, 2, 0], [0, 0, 1, 1, 1], [-1, 2 ** 31 - 1, -2 ** 31, 0, 0]):
        O = F.cached_attention(Q.to(gpu), cache, n, parents=_dev(gpu, np.array(parents, np.int32)))
        _check(O[0], G.attend(Q[0].double().numpy(), K[0, :25], V[0, :25], 20, 5, -1, parents), V[0])
    # capacity 32: nodes from place 32 on were not written, nor can their rows be
    F.cache_write_(cache, _values(rng, 1, 5, 1, 32).to(gpu), _values(rng, 1, 5, 1, 32).to(gpu), _dev(gpu, np.array([29], np.int32)))
    for length, good in ((29, 3), (32, 0), (33, 0), (2 ** 31 - 1, 0)):
        O = F.cached_attention(Q.to(gpu), cache, _dev(gpu, np.array([length], np.int32)))
        assert torch.isfinite(O[0, :good]).all() and torch.isnan(O[0, good:]).all(), length
    cache.pages[0, 0] = 99  # not in the pool
    O = F.cached_attention(Q.to(gpu), cache, n, (2, 0))  # keys from 18 on: on the second page
    assert torch.isfinite(O).all()
    assert torch.isnan(F.cached_attention(Q.to(gpu), cache, n)).all()


def test_rows_of_a_cache_past_32_bits(gpu):
    """A pool of more than 2^32 bytes; the sequences' pages at its ends."""
    rng = np.random.default_rng(12)
    P, Hkv, S, D, N = 280000, 2, 64, 128, 3
    cache = F.KVCache(torch.zeros(P, Hkv, S, D, dtype=torch.int8, device=gpu), torch.zeros(P, Hkv, S, D, dtype=torch.int8, device=gpu),
                      torch.zeros(P, Hkv, S, device=gpu), torch.zeros(P, Hkv, S, device=gpu),
                      torch.tensor([[P - 1, 0, P - 7], [3, P // 2, P - 2]], dtype=torch.int32, device=gpu))
    assert cache.k.numel() > 2 ** 32
    lengths = np.array([150, 100], np.int32)
    K, V = (_values(rng, 2, 153, Hkv, D) for _ in range(2))
    F.cache_write_(cache, K.to(gpu), V.to(gpu), torch.zeros(2, dtype=torch.int32, device=gpu))
    Q = (2.0 * torch.from_numpy(rng.standard_normal((2, N, 4, D), dtype=np.float32))).bfloat16()
    O = F.cached_attention(Q.to(gpu), cache, _dev(gpu, lengths))
    for b, n in enumerate(lengths):
        Kh, Vh = (G.held(x[b, :n + N].float().numpy(), "int8") for x in (K, V))
        _check(O[b], G.attend(Q[b].double().numpy(), Kh, Vh, int(n), N), Vh)
    path, kept = np.array([[0, 2, -1], [1, 2, -1]], np.int32), np.array([2, 2], np.int32)
    F.cache_keep_(cache, *_dev(gpu, lengths, path, kept))
    k, _ = F.cache_read(cache, _dev(gpu, lengths), 2, dtype=torch.float32)
    for b in range(2):
        assert np.array_equal(k[b].cpu().numpy(), G.held(K[b, lengths[b] + path[b, :2]].float().numpy(), "int8"))


def test_types_streams_and_workspaces(gpu):
    rng = np.random.default_rng(13)
    cache, K, V = _filled(gpu, rng, "int8", [700, 50], [2, 2], 2, 2, 64, 1600, 64)
    n = _dev(gpu, np.array([700, 50], np.int32))
    Q = (2.0 * torch.from_numpy(rng.standard_normal((2, 2, 4, 64), dtype=np.float32))).bfloat16().to(gpu)
    O = F.cached_attention(Q, cache, n)
    assert torch.equal(F.cached_attention(Q.float(), cache, n), O.float())
    half = F.cached_attention(Q.half(), cache, n)
    assert half.dtype == torch.float16 and torch.equal(half, F.cached_attention(Q.half().bfloat16(), cache, n).half())
    shifted = torch.empty(Q.numel() + 1, dtype=Q.dtype, device=gpu)[1:].view(Q.shape)
    shifted.copy_(Q)
    assert torch.equal(F.cached_attention(shifted, cache, n), O)
    nbytes = F.cached_attention_workspace_bytes(Q, cache)
    ws = torch.full((nbytes,), 255, dtype=torch.uint8, device=gpu)  # NaN wherever it would be read
    assert torch.equal(F.cached_attention(Q, cache, n, workspace=ws), O)
    with pytest.raises(ValueError, match="workspace"):
        F.cached_attention(Q, cache, n, workspace=ws[1:])
    # two calls at a time on two streams, each with its own workspace
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = [[] for _ in streams]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, r in zip(streams, results):
            with torch.cuda.stream(s):
                r.append(F.cached_attention(Q, cache, n))
    torch.cuda.synchronize()
    assert all(torch.equal(x, O) for r in results for x in r)


def test_captured_and_replayed(gpu):
    """A step in a graph; lengths, tokens and the cache change between its replays."""
    rng = np.random.default_rng(14)
    B, N, H, Hkv, D, V = 2, 3, 4, 2, 64, 1000
    caches = [F.kv_cache(B, 2048, Hkv, D, torch.int8, page=64, layers=2, device=gpu) for _ in range(2)]
    n = torch.full((B,), 900, dtype=torch.int32, device=gpu)
    K, V_, Q = (torch.from_numpy(rng.standard_normal((B, N, h, D), dtype=np.float32)).bfloat16().to(gpu) for h in (Hkv, Hkv, H))
    logits = (3 * torch.from_numpy(rng.standard_normal((B, N, V), dtype=np.float32))).to(gpu)
    tokens, u = torch.from_numpy(rng.integers(0, V, (B, N))).to(gpu), torch.rand(B, N, device=gpu)
    prefill = [_values(rng, 2, B, 2048, Hkv, D).to(gpu) for _ in range(2)]
    for c in caches:
        F.cache_write_(c, *prefill, torch.zeros(B, dtype=torch.int32, device=gpu))

    def step(cache, lengths):
        out = []
        for i in range(2):
            F.cache_write_(cache.layer(i), K, V_, lengths)
            out.append(F.cached_attention(Q, cache.layer(i), lengths))
        path, kept, token = F.verify_drafts(logits, tokens, u)
        F.cache_keep_(cache, lengths, path, kept)
        return out + [path, kept, token]

    step(caches[0], n)
    torch.cuda.synchronize()
    graph, static = torch.cuda.CUDAGraph(), n.clone()
    with torch.cuda.graph(graph):
        captured = step(caches[0], static)
    for c in caches:
        F.cache_write_(c, *prefill, torch.zeros(B, dtype=torch.int32, device=gpu))
    for k in range(4):
        x = torch.randn(1000, 1000, device=gpu).sum()  # the program's own work between the replays
        lengths = torch.tensor([5 + 300 * k, 1800 - 400 * k], dtype=torch.int32, device=gpu)
        K.normal_()
        u.uniform_()
        logits.normal_(0, 3)
        static.copy_(lengths)
        graph.replay()
        eager = step(caches[1], lengths)
        torch.cuda.synchronize()
        assert torch.isfinite(x)
        for got, want in zip(captured, eager):
            assert torch.equal(got, want), k
        for got, want in zip(F.cache_read(caches[0], None, 2048), F.cache_read(caches[1], None, 2048)):
            assert torch.equal(got, want), k


# ---- verification -------------------------------------------------------------------


def _verified(gpu, logits, tokens, u, draft=None, parents=None, counts=None, temperature=1.0, index=torch.int64, off=0, **kw):
    def place(x):
        y = torch.empty(x.numel() + off, dtype=x.dtype, device=gpu)[off:].view(x.shape)
        y.copy_(x)
        return y

    got = F.verify_drafts(place(logits), torch.from_numpy(tokens).to(index).to(gpu), _dev(gpu, u),
                          draft_logits=None if draft is None else place(draft), parents=_dev(gpu, parents), counts=_dev(gpu, counts),
                          temperature=temperature, **kw)
    return [x.cpu().numpy() for x in got]


def _agree(got, logits, tokens, u, draft=None, parents=None, counts=None, temperature=1.0):
    path, kept, token = got
    B, N = tokens.shape
    x, d = logits.double().numpy(), None if draft is None else draft.double().numpy()
    for b in range(B):
        want, after = G.verify(x[b], tokens[b], u[b].astype(np.float64), None if d is None else d[b],
                               None if parents is None else parents if parents.ndim == 1 else parents[b],
                               None if counts is None else int(counts[b]), temperature)
        assert path[b].tolist() == want + [-1] * (N - len(want)) and kept[b] == len(want) and token[b] == after, b


@pytest.mark.parametrize("V", [1, 2, 7, 259, 8191, 8192, 8193, 32768, 50257])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [1.0, 0.6, 0.0])
def test_runs_against_the_oracle(gpu, V, dtype, temperature):
    """Draws with the drafts' distribution, and the same runs as candidates."""
    rng = np.random.default_rng(V)
    B, N = 12, 6
    logits = torch.from_numpy(2.5 * rng.standard_normal((B, N, V), dtype=np.float32)).to(dtype)
    draft = (logits[:, :-1].float() + 0.7 * torch.from_numpy(rng.standard_normal((B, N - 1, V), dtype=np.float32))).to(dtype)
    q = G.softmax(draft.double().numpy(), temperature or 1.0)
    tokens = np.zeros((B, N), np.int64)
    for b in range(B):
        for i in range(N - 1):
            tokens[b, i + 1] = rng.choice(V, p=q[b, i]) if temperature else int(np.argmax(draft[b, i].float().numpy()))
    u = rng.random((B, N)).astype(np.float32)
    u[0], u[1], u[2, 0] = 0.0, 1.0 - 2.0 ** -24, 0.0
    counts = np.array([N, N, N, 1, 2, 0, N, N, 5, 4, 3, N], np.int32)
    for d in (draft, None):
        for c in (None, counts):
            got = _verified(gpu, logits, tokens, u, d, None, c, temperature, index=torch.int32 if c is None else torch.int64)
            _agree(got, logits, tokens, u, d if temperature else None, None, c, temperature)


@pytest.mark.parametrize("V,dtype", [(5, torch.float32), (259, torch.bfloat16), (32768, torch.bfloat16), (50257, torch.float32)])
@pytest.mark.parametrize("N", [1, 2, 9, 32, 64])
@pytest.mark.parametrize("temperature", [1.3, 0.0])
def test_trees_of_candidates_against_the_oracle(gpu, V, dtype, N, temperature):
    rng = np.random.default_rng(N + V)
    B = 6
    logits = torch.from_numpy(2.5 * rng.standard_normal((B, N, V), dtype=np.float32)).to(dtype)
    parents = np.stack([_tree(rng, N) for _ in range(B)])
    best = np.argsort(-logits.float().numpy(), -1, kind="stable")[..., :8]
    tokens = rng.integers(0, V, (B, N))
    for b in range(B):
        for i in range(1, N):  # the parents' best tokens, with repetitions among siblings
            tokens[b, i] = best[b, parents[b, i], min(V - 1, int(rng.integers(0, 4)))]
    u = rng.random((B, N)).astype(np.float32)
    counts = np.array([N, max(1, N // 2), 0, N, N, 1], np.int32)
    for up, c in ((parents, None), (parents, counts), (parents[0], counts)):
        got = _verified(gpu, logits, tokens, u, None, up, c, temperature)
        _agree(got, logits, tokens, u, None, up, c, temperature)


@pytest.mark.parametrize("B", [2, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_row_of_many_parts(gpu, dtype, B):
    """More parts of the drawn row than a wave's registers hold, and draws from all over it, by the
    last workgroup to arrive and in a launch of its own."""
    rng = np.random.default_rng(31)
    N, V = 3, 199999
    logits = torch.from_numpy(0.5 * rng.standard_normal((B, N, V), dtype=np.float32)).to(dtype)
    draft = torch.from_numpy(0.5 * rng.standard_normal((B, N - 1, V), dtype=np.float32)).to(dtype)
    tokens = rng.integers(0, V, (B, N))
    u = rng.random((B, N)).astype(np.float32)
    u[:, 0] = np.linspace(0.02, 0.98, B)
    for d in (draft, None):
        _agree(_verified(gpu, logits, tokens, u, d), logits, tokens, u, d, None, None, 1.0)


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_off_a_16_byte_boundary(gpu, dtype, off):
    rng = np.random.default_rng(off)
    B, N, V = 5, 4, 9001
    logits = torch.from_numpy(2.0 * rng.standard_normal((B, N, V), dtype=np.float32)).to(dtype)
    draft = torch.from_numpy(2.0 * rng.standard_normal((B, N - 1, V), dtype=np.float32)).to(dtype)
    tokens, u = rng.integers(0, V, (B, N)), rng.random((B, N)).astype(np.float32)
    _agree(_verified(gpu, logits, tokens, u, draft, off=off), logits, tokens, u, draft)


def test_equal_distributions_filtered_logits_and_ties(gpu):
    """p = q keeps every draft; -infinity is never drawn; the lowest of equal logits is the largest."""
    rng = np.random.default_rng(20)
    B, N, V = 8, 5, 9000
    logits = torch.from_numpy(2.0 * rng.standard_normal((B, N, V), dtype=np.float32))
    logits[:, :, ::3] = -float("inf")
    tokens = 3 * rng.integers(0, V // 3, (B, N)) + 1
    u = rng.random((B, N)).astype(np.float32)
    path, kept, token = _verified(gpu, logits, tokens, u, logits[:, :-1].contiguous())
    assert (kept == N).all() and (token % 3 != 0).all()
    got = _verified(gpu, logits, tokens - 1, u)  # candidates of probability 0
    assert (got[1] == 1).all()
    _agree(got, logits, tokens - 1, u)
    flat = torch.zeros(B, N, V)
    flat[:, :, 5] = flat[:, :, 4000] = flat[:, :, 8999] = 1.5
    got = _verified(gpu, flat, np.full((B, N), 5), u, temperature=0.0)
    assert (got[1] == N).all() and (got[2] == 5).all()
    # one value holds all of p
    sure = torch.full((B, N, V), -200.0)
    sure[:, :, 77] = 10.0
    _agree(_verified(gpu, sure, np.full((B, N), 77), u), sure, np.full((B, N), 77), u)
    _agree(_verified(gpu, sure, np.full((B, N), 78), u), sure, np.full((B, N), 78), u)


@pytest.mark.parametrize("temperature", [1.0, 0.0])
def test_rows_without_probabilities_and_foreign_tokens(gpu, temperature):
    rng = np.random.default_rng(21)
    B, N, V = 6, 3, 10000
    logits = torch.from_numpy(rng.standard_normal((B, N, V), dtype=np.float32))
    tokens = np.zeros((B, N), np.int64)
    for i in range(1, N):
        tokens[:, i] = logits[:, i - 1].argmax(-1).numpy()
    u = np.zeros((B, N), np.float32)
    logits[0, 0, 9999], logits[1, 1, 3], logits[2, 2] = float("nan"), float("inf"), -float("inf")
    tokens[3, 1], tokens[4, 2] = V, -1
    got = _verified(gpu, logits, tokens, u, temperature=temperature)
    _agree(got, logits, tokens, u, temperature=temperature)
    assert got[2][:3].tolist() == [-1, -1, -1] and got[1].tolist() == [1, 2, 3, 1, 2, 3]
    for parents in ([-1, 2, 1], [-1, -1, 0], [-1, -7, 2 ** 31 - 1], [5, 0, 0]):  # nodes that hang on nothing are never reached
        up = np.array(parents, np.int32)
        path, kept, _ = _verified(gpu, logits, tokens, u, parents=up, temperature=temperature)
        reach = [i for i in range(1, N) if parents[i] == 0]
        assert set(path[5].tolist()) <= {0, -1, *reach}


def test_the_same_bits_again_and_a_callers_workspace(gpu):
    rng = np.random.default_rng(22)
    B, N, V = 16, 5, 32768
    logits = torch.from_numpy(2.0 * rng.standard_normal((B, N, V), dtype=np.float32)).to(gpu)
    draft = logits[:, 1:].contiguous()
    tokens, u = torch.from_numpy(rng.integers(0, V, (B, N))).to(gpu), torch.rand(B, N, device=gpu)
    first = F.verify_drafts(logits, tokens, u, draft_logits=draft)
    n = F.verify_drafts_workspace_bytes(logits, tokens, u, draft_logits=draft)
    ws = torch.full((n,), 255, dtype=torch.uint8, device=gpu)
    for _ in range(3):
        for a, b in zip(first, F.verify_drafts(logits, tokens, u, draft_logits=draft, workspace=ws)):
            assert torch.equal(a, b)


# ---- a run of them together -----------------------------------------------------------


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("tree", [False, True])
def test_generating_text_with_drafted_tokens(gpu, kind, tree):
    """A two-layer model's steps: prompts written, trees (or runs) drafted, attended to,
    verified and kept.  At every step each layer's attention is that of the text so far
    (read from the cache), the verification is the oracle's on the same logits, and the cache
    holds the accepted tokens' keys and values and nothing else."""
    rng = np.random.default_rng(30)
    B, H, Hkv, D, N, vocab, steps, width = 3, 4, 2, 32, 6, 50, 8, 64
    cache = _shuffled(_junk(F.kv_cache(B, 128, Hkv, D, KINDS[kind], layers=2, page=16, device=gpu)), 1)
    g = torch.Generator().manual_seed(31)
    table = torch.randn(vocab, width, generator=g)
    proj = [{n: torch.randn(width, h * D, generator=g) / 8 for n, h in (("q", H), ("k", Hkv), ("v", Hkv))} for _ in range(2)]
    back = [torch.randn(H * D, width, generator=g) / 8 for _ in range(2)]
    sin, cos = F.rotary_embeddings(256, D)
    sin, cos = sin.to(gpu), cos.to(gpu)
    table, back, proj = table.to(gpu), [w.to(gpu) for w in back], [{n: w.to(gpu) for n, w in p.items()} for p in proj]
    slopes = _dev(gpu, np.array([0.5, 0.25, 0.125, 0.0625], np.float32))
    windows, cap = [(-1, 0), (20, 0)], 15.0

    def heads(x, w, h):
        return (x @ w).view(x.shape[0], x.shape[1], h, D).bfloat16()

    def layer_inputs(i, x, positions):
        q, k, v = heads(x, proj[i]["q"], H), heads(x, proj[i]["k"], Hkv), heads(x, proj[i]["v"], Hkv)
        return F.attention_prologue(q, (sin, cos), positions), F.attention_prologue(k, (sin, cos), positions), v

    # prompts, of odd lengths, padded: attention over the batch, keys and values into the cache
    prompt_lengths = np.array([7, 19, 1], np.int32)
    T = int(prompt_lengths.max())
    text = [rng.integers(0, vocab, n).tolist() for n in prompt_lengths]
    ids = torch.zeros(B, T, dtype=torch.int64)
    for b in range(B):
        ids[b, :len(text[b]) - 1] = torch.tensor(text[b][:-1], dtype=torch.int64)
    counts = _dev(gpu, prompt_lengths - 1)  # the last token is the first step's node 0
    lengths = torch.zeros(B, dtype=torch.int32, device=gpu)
    x = table[ids.to(gpu)]
    for i in range(2):
        q, k, v = layer_inputs(i, x, None)
        F.cache_write_(cache.layer(i), k, v, lengths, counts)
        O = F.attention(q, k, v, windows[i], softcap=cap, slopes=slopes)
        x = x + O.float().reshape(B, T, H * D) @ back[i]
    lengths += counts
    kept_total = 0
    for step in range(steps):
        parents = _tree(rng, N) if tree else np.arange(-1, N - 1, dtype=np.int32)
        lines = G.lineage(parents, N)
        depth = np.array([len(l) - 1 for l in lines])
        nodes = rng.integers(0, vocab, (B, N))
        nodes[:, 0] = [t[-1] for t in text]
        counts_now = np.array([N, N - 1, N if step % 2 else 1], np.int32)
        up, c = _dev(gpu, parents) if tree else None, _dev(gpu, counts_now)
        positions = (lengths[:, None] + _dev(gpu, depth.astype(np.int32))).contiguous()
        x = table[torch.from_numpy(nodes).to(gpu)]
        for i in range(2):
            q, k, v = layer_inputs(i, x, positions)
            F.cache_write_(cache.layer(i), k, v, lengths, c)
            O = F.cached_attention(q, cache.layer(i), lengths, windows[i], counts=c, parents=up, softcap=cap, slopes=slopes)
            Kc, Vc = F.cache_read(cache.layer(i), None, 128, lengths + c, dtype=torch.float32)
            for b in range(B):
                n, m = int(lengths[b]), int(counts_now[b])
                assert n == len(text[b]) - 1
                held = (Kc[b, :n + m].cpu().numpy(), Vc[b, :n + m].cpu().numpy())
                want = G.attend(q[b].double().cpu().numpy(), *held, n, m, windows[i][0], parents, cap, slopes.cpu().numpy())
                _check(O[b], want, held[1])
            x = x + O.float().reshape(B, N, H * D) @ back[i]
        logits = (x @ table.T * 0.5).contiguous()
        # drafts: some of them the model's own best tokens
        if step % 3 != 2:
            best = logits.argmax(-1).cpu().numpy()
            for b in range(B):
                nodes[b, 1] = best[b, 0]
        u = rng.random((B, N)).astype(np.float32)
        T_ = [1.0, 0.0, 0.7][step % 3]
        path, kept, token = F.verify_drafts(logits, torch.from_numpy(nodes).to(gpu), _dev(gpu, u), parents=up, counts=c, temperature=T_)
        _agree([t.cpu().numpy() for t in (path, kept, token)], logits.cpu(), nodes, u, None, parents if tree else None, counts_now, T_)
        before = F.cache_read(cache, lengths, N, c, dtype=torch.float32)
        F.cache_keep_(cache, lengths, path, kept)
        after = F.cache_read(cache, lengths, N, kept, dtype=torch.float32)
        for b in range(B):
            line = path[b, :int(kept[b])].tolist()
            assert line in [l for l in lines]
            for old, new in zip(before, after):
                assert torch.equal(new[:, b, :len(line)], old[:, b, line])
            text[b] += nodes[b, line[1:]].tolist() + [int(token[b])]
            kept_total += len(line)
        lengths += kept
    assert kept_total > B * steps  # drafts were accepted


# ---- refusals -----------------------------------------------------------------------------


def test_refusals(gpu):
    cache = F.kv_cache(2, 64, 2, 32, torch.int8, device=gpu)
    n = torch.zeros(2, dtype=torch.int32, device=gpu)
    K = torch.zeros(2, 3, 2, 32, dtype=torch.bfloat16, device=gpu)
    Q = torch.zeros(2, 3, 4, 32, dtype=torch.bfloat16, device=gpu)
    for call in (lambda: F.cache_write_(cache, K, K[:, :2], n), lambda: F.cache_write_(cache, K, K, n[:1]),
                 lambda: F.cache_write_(cache, K.half(), K.half(), n), lambda: F.cache_write_(cache, K, K.float(), n),
                 lambda: F.cache_write_(cache, K, K, n.long()), lambda: F.cache_write_(cache, K.transpose(1, 2), K, n),
                 lambda: F.cache_write_(cache, K, K, None), lambda: F.cache_write_(cache, K, K, n, n.float()),
                 lambda: F.cache_write_(cache._replace(k_scale=None), K, K, n), lambda: F.cache_write_(cache._replace(v=cache.k[:1]), K, K, n),
                 lambda: F.cache_write_(cache._replace(k=cache.k.float()), K, K, n),
                 lambda: F.cache_write_(cache._replace(pages=n), K, K, n), lambda: F.cache_read(cache, n, -1),
                 lambda: F.cache_read(cache, n, 3, dtype=torch.float16), lambda: F.cache_keep_(cache, n, n, n),
                 lambda: F.cached_attention(Q, cache, n, (3, 1)), lambda: F.cached_attention(Q, cache, n, (-2, 0)),
                 lambda: F.cached_attention(Q[:, :, :3], cache, n), lambda: F.cached_attention(Q, cache, n.cpu()),
                 lambda: F.cached_attention(Q, cache, n, parents=n), lambda: F.cached_attention(Q, cache, n, slopes=n.float()),
                 lambda: F.cached_attention(torch.zeros(2, 65, 4, 32, dtype=torch.bfloat16, device=gpu), cache, n),
                 lambda: F.cached_attention(torch.zeros(2, 3, 3, 32, dtype=torch.bfloat16, device=gpu), cache, n),
                 lambda: F.cached_attention(Q, cache, n, softcap=-1.0), lambda: F.cached_attention(Q.double(), cache, n),
                 lambda: F.cached_attention(Q.transpose(0, 1), cache, n),
                 lambda: F.cached_attention(Q, F.kv_cache(2, 64, 2, 32, torch.int8, layers=2, device=gpu), n)):
        with pytest.raises((ValueError, TypeError, F._lib.AttentionError)):
            call()
    x, t, u = torch.zeros(2, 3, 50, device=gpu), torch.zeros(2, 3, dtype=torch.int64, device=gpu), torch.zeros(2, 3, device=gpu)
    up = torch.tensor([-1, 0, 0], dtype=torch.int32, device=gpu)
    for call in (lambda: F.verify_drafts(x, t, u, draft_logits=x[:, 1:].contiguous(), parents=up), lambda: F.verify_drafts(x, t, None),
                 lambda: F.verify_drafts(x, t, u, draft_logits=x), lambda: F.verify_drafts(x, t, u, draft_logits=x[:, 1:].bfloat16()),
                 lambda: F.verify_drafts(x, t.float(), u), lambda: F.verify_drafts(x, t, u.double()),
                 lambda: F.verify_drafts(x, t, u, temperature=-1.0), lambda: F.verify_drafts(x.half(), t, u),
                 lambda: F.verify_drafts(x, t[:, :2], u), lambda: F.verify_drafts(x, t, u, parents=up[:2]),
                 lambda: F.verify_drafts(x, t, u, counts=up), lambda: F.verify_drafts(x[:, :, ::2], t, u)):
        with pytest.raises((ValueError, TypeError, F._lib.AttentionError)):
            call()
    F.cache_write_(cache, K[:, :0], K[:, :0], n)  # nothing to do
    assert F.cache_read(cache, n, 0)[0].shape == (2, 0, 2, 32)
    assert [v.tolist() for v in F.verify_drafts(x, t, None, temperature=0.0)[1:]] == [[3, 3], [0, 0]]
