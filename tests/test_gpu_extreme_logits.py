"""Verification of drafted tokens at logits of any finite size: what counts is their distance
from the row's largest, against the temperature."""
import numpy as np
import pytest
import torch

import femtochat_amd as F
from oracle import generation as G

pytestmark = pytest.mark.gpu
LEAST = float(torch.finfo(torch.float32).min)


def _compare(gpu, logits, draft, temperature, rng):
    B, N, V = logits.shape
    q = G.softmax((logits[:, :-1] if draft is None else draft).double().numpy(), temperature)
    tokens = np.zeros((B, N), np.int64)
    for b in range(B):
        for i in range(N - 1):
            tokens[b, i + 1] = rng.choice(V, p=q[b, i])
    u = rng.random((B, N)).astype(np.float32)
    path, kept, token = (t.tolist() for t in F.verify_drafts(
        logits.to(gpu), torch.from_numpy(tokens).to(gpu), torch.from_numpy(u).to(gpu),
        draft_logits=None if draft is None else draft.to(gpu), temperature=temperature))
    ends = set()
    for b in range(B):
        want, after = G.verify(logits[b].double().numpy(), tokens[b], u[b].astype(np.float64),
                               None if draft is None else draft[b].double().numpy(), temperature=temperature)
        assert (path[b], kept[b], token[b]) == (want + [-1] * (N - len(want)), len(want), after), b
        ends.add(len(want))
    return ends


@pytest.mark.parametrize("V", [300, 9001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size,temperature", [
    (3e9, 1.0), (-3e9, 1.0), (-1e9, 0.7), (5e7, 0.01), (-5e7, 0.01), (3e6, 2.0 ** -10), (-3e6, 2.0 ** -10), (3e10, 1.0), (-3e10, 1.0),
    (2.5e7, 2.0 ** -10), (-2.5e7, 2.0 ** -10), (3e38, 1.0), (-3e38, 2.0 ** 10), (LEAST, 1.0), (LEAST, 2.0 ** 10), (LEAST, 2.0 ** -10)])
def test_rows_of_equal_logits_of_any_size(gpu, size, temperature, dtype, V):
    """Some of a row's logits are its largest, the others a step of the type below it or at -infinity:
    p is even over the largest (q over others of them)."""
    rng = np.random.default_rng(V)
    B, N = 24, 4
    top = torch.tensor(size).to(dtype)
    if not torch.isfinite(top):
        top = torch.tensor(torch.finfo(dtype).min).to(dtype)
    low = torch.nextafter(top, torch.tensor(-float("inf"), dtype=dtype))
    if float(top - low) < 60 * temperature:  # (a step that leaves the lower ones a share: none of them)
        low = torch.tensor(-float("inf"), dtype=dtype)

    def rows(n):
        high = torch.from_numpy(rng.random((B, n, V)) < 0.4)
        high[..., 0] = True
        return torch.where(high, top, low)

    ends = set()
    for draft in (rows(N - 1), None):
        ends |= _compare(gpu, rows(N), draft, temperature, rng)
    assert len(ends) > 1


@pytest.mark.parametrize("V", [300, 9001])
@pytest.mark.parametrize("draws", [True, False])
def test_masked_logits_and_the_whole_range(gpu, V, draws):
    """The type's lowest value as a mask, and a largest logit whose distance from it is beyond float32."""
    rng = np.random.default_rng(V + 1)
    B, N = 24, 4

    def rows(n):
        x = torch.from_numpy(2.5 * rng.standard_normal((B, n, V), dtype=np.float32))
        x[:, :, ::3] = LEAST
        x[B // 2:, :, 5::7] = -LEAST
        return x

    ends = _compare(gpu, rows(N), rows(N - 1) if draws else None, 1.0, rng)
    assert len(ends) > 1
