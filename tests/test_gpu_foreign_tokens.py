"""Drafted tokens outside the vocabulary, in runs with the drafts' distributions: such a node was
not drawn from them, so it ends the run and the next token is drawn from the target's own."""
import numpy as np
import pytest
import torch

import femtochat_amd as F
from oracle import generation as G

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [3, 300, 9001])
@pytest.mark.parametrize("alike", [False, True])
@pytest.mark.parametrize("foreign", [-1, 0, 2 ** 31 - 1, -2 ** 31, 2 ** 32 + 1, -2 ** 63])
def test_the_next_token_behind_a_foreign_one(gpu, V, alike, foreign):
    """foreign 0 stands for V itself; a second foreign node behind the first, and one that no one reaches."""
    rng = np.random.default_rng(V)
    B, N = 40, 4
    logits = torch.from_numpy(1.5 * rng.standard_normal((B, N, V), dtype=np.float32))
    draft = logits[:, :-1].clone() if alike else torch.from_numpy(1.5 * rng.standard_normal((B, N - 1, V), dtype=np.float32))
    if V == 3:
        logits[:] = torch.log(torch.tensor([0.5, 0.4, 0.1]))
        draft[:] = torch.log(torch.tensor([0.5, 0.4, 0.1] if alike else [0.6, 0.3, 0.1]))
    q = G.softmax(draft.double().numpy(), 1.0)
    tokens = np.zeros((B, N), np.int64)
    for b in range(B):
        for i in range(1, N):
            tokens[b, i] = rng.choice(V, p=q[b, i - 1])
        tokens[b, 1 + b % (N - 1):3 + b % (N - 1)] = foreign if foreign != 0 else V
    u = rng.random((B, N)).astype(np.float32)
    u[:, 0] = (np.arange(B) + 0.5) / B
    index = torch.int32 if abs(foreign + 0.5) < 2 ** 31 else torch.int64
    for counts in (None, rng.integers(1, N + 1, B).astype(np.int32)):
        path, kept, token = (t.tolist() for t in F.verify_drafts(
            logits.to(gpu), torch.from_numpy(tokens).to(index).to(gpu), torch.from_numpy(u).to(gpu), draft_logits=draft.to(gpu),
            counts=None if counts is None else torch.from_numpy(counts).to(gpu)))
        for b in range(B):
            want, after = G.verify(logits[b].double().numpy(), tokens[b], u[b].astype(np.float64), draft[b].double().numpy(),
                                   count=None if counts is None else int(counts[b]))
            assert (path[b], kept[b], token[b]) == (want + [-1] * (N - len(want)), len(want), after), b
