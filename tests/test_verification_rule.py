"""Mistakes planted in the oracle's verification of drafted tokens move the distribution of the
text, by more than the grids that the right rule passes (CPU)."""
import numpy as np
import pytest

from oracle import generation as G


@pytest.mark.parametrize("mistaken", [False, True])
def test_a_second_candidate_against_all_of_p(mistaken):
    """Mistaken: u < p(x) for the second candidate, not u (1 - p of the first) < p(x)."""
    rng = np.random.default_rng(5)
    V, M = 6, 40
    x = np.tile(rng.standard_normal(V) * 1.5, (4, 1))
    p, got, grid = G.softmax(x[0], 1.0), np.zeros(V), (np.arange(M) + 0.5) / M
    left = 1.0 - p[4]
    for a in grid:
        for b in grid:
            for u0 in grid:
                path, token = G.verify(x, [0, 4, 3, 4], [u0, a, b / left if mistaken else b, 0.0], parents=[-1, 0, 0, 0])
                got[[token, 4, 3][path[-1]]] += M ** -3.0
    assert (np.abs(got - p).max() < 3 / M) == (not mistaken)  # (a step of each of three grids)


@pytest.mark.parametrize("mistaken", [False, True])
def test_a_refused_draw_replaced_from_all_of_p(mistaken):
    """Mistaken: the next token behind a refusal drawn from p, not from max(p - q, 0)."""
    rng = np.random.default_rng(6)
    V, M = 5, 400
    x, d = rng.standard_normal((2, V)) * 2, rng.standard_normal((1, V)) * 2
    p, q, got = G.softmax(x[0], 1.0), G.softmax(d[0], 1.0), np.zeros(V)
    for y in range(V):
        for k in range(M):
            for u0 in (np.arange(50) + 0.5) / 50:
                path, token = G.verify(x, [0, y], [u0, (k + 0.5) / M], d)
                if mistaken and len(path) == 1:
                    token = G.draw(p, u0)
                got[y if len(path) == 2 else token] += q[y] / (M * 50)
    assert (np.abs(got - p).max() < 1 / M + 1 / 50) == (not mistaken)
