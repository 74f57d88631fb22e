"""Values in a cache that are not finite: a node that sees one has it in that column, wherever its
key lies, and no other node or column has anything of it.

Tolerances are those of the cache's attention (a sum's float32 roundings 4e-4 of a column's largest
value, O's rounding 2^-8 of itself); what is not finite is equal."""
import numpy as np
import pytest
import torch

import femtochat_amd as F
from oracle import generation as G

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def _check(O, want, V):
    """want: the oracle's on the finite values, with what is not finite put in."""
    O = O.double().cpu().numpy()
    odd = ~np.isfinite(want)
    np.testing.assert_array_equal(np.where(odd, O, 0.0), np.where(odd, want, 0.0))
    most = np.repeat(np.abs(V).max(0), O.shape[1] // V.shape[1], 0)
    good = np.where(odd, 0.0, want)
    assert np.isfinite(O[~odd]).all()
    assert (np.abs(np.where(odd, 0.0, O) - good) <= 2.0 ** -8 * np.abs(good) + 4e-4 * most[None]).all()


def _attend_odd(Q, K, V, length, N, left, parents):
    """The oracle with values that are not finite: their sum over the keys that a node sees, in their columns."""
    H, odd = Q.shape[1], np.where(np.isfinite(V), 0.0, V)
    out = G.attend(Q, K, np.where(np.isfinite(V), V, 0.0), length, N, left, parents)
    for i, line in enumerate(G.lineage(parents, N)):
        keys = [t for t in range(length) if left < 0 or length + len(line) - 1 - t <= left]
        keys += [length + j for d, j in enumerate(line) if left < 0 or len(line) - 1 - d <= left]
        with np.errstate(invalid="ignore"):
            out[i] += np.repeat(odd[keys].sum(0), H // V.shape[1], 0)
    return out


def _inputs(rng, n, N, H, Hkv, D):
    K, V = (1.2 * torch.from_numpy(rng.standard_normal((1, n + N, Hkv, D), dtype=np.float32)) for _ in range(2))
    Q = (2.0 * torch.from_numpy(rng.standard_normal((1, N, H, D), dtype=np.float32))).bfloat16()
    return K.bfloat16().float(), V.bfloat16().float(), Q


def _tree(rng, N):
    return np.array([-1] + [int(rng.integers(0, i)) for i in range(1, N)], np.int32)


@pytest.mark.parametrize("D", [16, 48, 64, 80, 112, 128])
@pytest.mark.parametrize("N,H,Hkv", [(1, 4, 2), (6, 4, 2), (6, 24, 2), (40, 2, 1)])
@pytest.mark.parametrize("n,capacity,page", [(90, 144, 16), (700, 784, None), (1300, 2048, 64)])
def test_values_that_are_not_finite_anywhere_in_a_sequence(gpu, n, capacity, page, N, H, Hkv, D):
    """In the first tiles, in the middle, at the last token and at nodes; one workgroup, eight waves, and parts."""
    rng = np.random.default_rng(n + N + D)
    K, V, Q = _inputs(rng, n, N, H, Hkv, D)
    parents = _tree(rng, N)
    for left in (-1, n // 2):
        X = V.clone()
        for value, t, h, d in ((INF, 0, 0, 1), (-INF, n // 2 - 7, Hkv - 1, 2), (NAN, n // 3, 0, 3), (INF, n - 1, 0, D - 1), (-INF, 33, 0, 5),
                               (INF, n - 20, 0, 5), (INF, 70, 0, 7), (INF, n - 2, 0, 7), (-INF, n + N // 2, 0, 0), (NAN, n + N - 1, 0, 9)):
            X[0, t, h, d] = value
        cache = F.kv_cache(1, capacity, Hkv, D, torch.bfloat16, page=page, device=gpu)
        cache.v.fill_(NAN)  # (behind the nodes)
        F.cache_write_(cache, K.to(gpu), X.to(gpu), torch.zeros(1, dtype=torch.int32, device=gpu))
        O = F.cached_attention(Q.to(gpu), cache, torch.tensor([n], dtype=torch.int32, device=gpu), (left, 0),
                               parents=torch.from_numpy(parents).to(gpu))[0]
        _check(O, _attend_odd(Q[0].double().numpy(), K[0].double().numpy(), X[0].double().numpy(), n, N, left, parents),
               np.where(np.isfinite(X[0].numpy()), X[0].numpy(), 0.0))


@pytest.mark.parametrize("n,capacity", [(300, 512), (3000, 4096)])
@pytest.mark.parametrize("value", [INF, -INF])
def test_an_infinity_whose_share_is_next_to_nothing(gpu, value, n, capacity):
    """Its key's score lies hundreds below the row's largest, before or behind it: 2^-400 of an infinity is one."""
    rng = np.random.default_rng(n)
    N, H, Hkv, D = 2, 2, 1, 64
    K, V, Q = _inputs(rng, n, N, H, Hkv, D)
    Q[:] = 4.0  # scores: half the sum of a key's values
    K[:] = K / 16
    for far in (3, n - 2):
        X, Y = V.clone(), K.clone()
        X[0, far, 0, 11] = value
        Y[0, far] = -8.0  # a score of -256, 370 in base 2
        cache = F.kv_cache(1, capacity, Hkv, D, torch.bfloat16, device=gpu)
        F.cache_write_(cache, Y.to(gpu), X.to(gpu), torch.zeros(1, dtype=torch.int32, device=gpu))
        O = F.cached_attention(Q.to(gpu), cache, torch.tensor([n], dtype=torch.int32, device=gpu))[0]
        _check(O, _attend_odd(Q[0].double().numpy(), Y[0].bfloat16().double().numpy(), X[0].double().numpy(), n, N, -1, None),
               np.where(np.isfinite(X[0].numpy()), X[0].numpy(), 0.0))


@pytest.mark.parametrize("D", [16, 64, 80, 128])
@pytest.mark.parametrize("N,H,Hkv", [(6, 4, 2), (40, 2, 1)])
@pytest.mark.parametrize("n,capacity,page", [(90, 144, 16), (1300, 2048, 64)])
def test_nan_codes_of_float8(gpu, n, capacity, page, N, H, Hkv, D):
    """A caller's own float8 codes may be NaN, at keys that all see and at nodes that some do not."""
    rng = np.random.default_rng(n + D)
    K, V, Q = _inputs(rng, n, N, H, Hkv, D)
    parents = _tree(rng, N)
    cache = F.kv_cache(1, capacity, Hkv, D, torch.float8_e4m3fn, page=page, device=gpu)
    F.cache_write_(cache, K.to(gpu), V.to(gpu), torch.zeros(1, dtype=torch.int32, device=gpu))
    Kh, Vh = (G.held(x.numpy(), "fp8")[0] for x in (K, V))
    codes, size = cache.v.view(torch.uint8), cache.k.shape[-2]
    for code, t, h, d in ((0x7F, 2, 0, 1), (0xFF, n // 2, Hkv - 1, 2), (0x7F, n - 1, 0, D - 1), (0xFF, n + N // 2, 0, 3), (0x7F, n + N - 1, 0, 4)):
        p = 0 if cache.pages is None else int(cache.pages[0, t // size])
        codes[p, h, t % size, d] = code
        Vh[t, h, d] = NAN
    k = cache.k.view(torch.uint8)  # and a key's, behind the nodes
    k[0 if cache.pages is None else int(cache.pages[0, (n + N) // size]), 0, (n + N) % size, 3] = 0x7F
    for left in (-1, n // 2 - 10):
        O = F.cached_attention(Q.to(gpu), cache, torch.tensor([n], dtype=torch.int32, device=gpu), (left, 0),
                               parents=torch.from_numpy(parents).to(gpu))[0]
        _check(O, _attend_odd(Q[0].double().numpy(), Kh.astype(np.float64), Vh.astype(np.float64), n, N, left, parents),
               np.where(np.isfinite(Vh), Vh, 0.0))


def test_the_same_sums_beside_them(gpu):
    """Rows and columns without such a value have the bits that they have without any."""
    rng = np.random.default_rng(3)
    n, N, H, Hkv, D = 1500, 6, 4, 2, 128
    K, V, Q = _inputs(rng, n, N, H, Hkv, D)
    out = []
    for value in (0.0, INF):
        V[0, 40, 1, 17] = value
        cache = F.kv_cache(1, 2048, Hkv, D, torch.bfloat16, device=gpu)
        F.cache_write_(cache, K.to(gpu), V.to(gpu), torch.zeros(1, dtype=torch.int32, device=gpu))
        out.append(F.cached_attention(Q.to(gpu), cache, torch.tensor([n], dtype=torch.int32, device=gpu))[0])
    assert (out[1][:, 2:, 17] == INF).all()
    out[1][:, 2:, 17] = out[0][:, 2:, 17]
    assert torch.equal(*out)


@pytest.mark.parametrize("capacity,top", [(784, 700), (1600, 1500)])
def test_a_batch_in_which_some_sequences_have_them(gpu, capacity, top):
    """Workgroups that go from a sequence with such a value to one without: every other number has
    the bits that it has without any."""
    rng = np.random.default_rng(capacity)
    B, N, H, Hkv, D = 150, 2, 12, 2, 64
    lengths = rng.integers(1, top, B).astype(np.int32)
    T = int(lengths.max()) + N
    K, V = (1.2 * torch.from_numpy(rng.standard_normal((B, T, Hkv, D), dtype=np.float32)) for _ in range(2))
    Q = (2.0 * torch.from_numpy(rng.standard_normal((B, N, H, D), dtype=np.float32))).bfloat16().to(gpu)
    n, zero = torch.from_numpy(lengths).to(gpu), torch.zeros(B, dtype=torch.int32, device=gpu)
    out, odd = [], torch.zeros(B, N, H, D)
    for with_them in (False, True):
        if with_them:
            for b in range(0, B, 3):
                t, h, d = int(rng.integers(0, lengths[b])), int(rng.integers(0, Hkv)), int(rng.integers(0, D))
                value = (INF, -INF, NAN)[b // 3 % 3]
                V[b, t, h, d] = value
                odd[b, :, h * (H // Hkv):(h + 1) * (H // Hkv), d] = value
        cache = F.kv_cache(B, capacity, Hkv, D, torch.bfloat16, device=gpu)
        F.cache_write_(cache, K.to(gpu), V.to(gpu), zero)
        out.append(F.cached_attention(Q, cache, n).float().cpu())
    there = odd != 0
    assert torch.equal(torch.where(there, 0.0, out[1]), torch.where(there, 0.0, out[0])) and torch.isfinite(out[0]).all()
    np.testing.assert_array_equal(out[1][there].numpy(), odd[there].numpy())
