"""Drafts whose distribution is the target's: where one is refused all the same (it has no weight in
either), nothing is left of max(p - q, 0), and the next token is drawn from p."""
import numpy as np
import pytest
import torch

import femtochat_amd as F
from oracle import generation as G

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [2, 259, 2048, 2049, 9001, 50000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("spread", [0.0, 2.5, 60.0])
def test_nothing_left_of_a_residual(gpu, V, dtype, spread):
    rng = np.random.default_rng(V)
    B, N = 48, 3
    logits = torch.from_numpy(spread * rng.standard_normal((B, N, V), dtype=np.float32)).to(dtype)
    logits[:, :, V // 2] = -float("inf")
    draft = logits[:, :-1].contiguous()
    tokens = np.full((B, N), V // 2, np.int64)
    q = G.softmax(draft.double().numpy(), 0.8)
    for b in range(0, B, 2):
        tokens[b, 1] = rng.choice(V, p=q[b, 0])  # kept; its follower is refused
    u = rng.random((B, N)).astype(np.float32)
    path, kept, token = (t.tolist() for t in F.verify_drafts(
        logits.to(gpu), torch.from_numpy(tokens).to(gpu), torch.from_numpy(u).to(gpu), draft_logits=draft.to(gpu), temperature=0.8))
    for b in range(B):
        want, after = G.verify(logits[b].double().numpy(), tokens[b], u[b].astype(np.float64), draft[b].double().numpy(), temperature=0.8)
        assert len(want) == 2 - b % 2
        assert (path[b], kept[b], token[b]) == (want + [-1] * (N - len(want)), len(want), after), b
