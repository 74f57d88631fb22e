"""A caller's workspace in an order of its own dimensions."""
import pytest
import torch

import femtochat_amd as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("softcap", [0.0, 5.0])
@pytest.mark.parametrize("D", [64, 96])
def test_permuted_workspaces(gpu, softcap, D):
    A, B, T, H, Hkv = F.MFMAFast(), 2, 333, 4, 2
    g = torch.Generator().manual_seed(1)
    Q, K, V, dO = (torch.randn(B, T, h, D, generator=g).bfloat16().to(gpu) for h in (H, Hkv, Hkv, H))
    pos = (torch.arange(T, dtype=torch.int32) % 50).repeat(B, 1).to(gpu)
    got = []
    for permuted in (False, True):
        O, l, m = torch.empty_like(Q), torch.empty(B, H, T, device=gpu), torch.empty(B, H, T, device=gpu)
        grads = [torch.empty_like(x) for x in (Q, K, V)]
        how = dict(positions=pos, softcap=softcap)
        room = lambda n: torch.empty((n + 63) // 64, 64, dtype=torch.uint8, device=gpu).t() if permuted else None  # noqa: E731
        F.attention_(A, O, l, m, Q, K, V, (-1, 0), workspace=room(F.forward_workspace_bytes(A, Q, K, **how)), **how)
        F.delta_attention_(A, *grads, dO, Q, K, V, O, l, m, (-1, 0), accumulate=False,
                           workspace=room(F.backward_workspace_bytes(A, Q, K, **how)), **how)
        got.append([O, l, m] + grads)
    assert all(torch.equal(a, b) for a, b in zip(*got))
    x, t, r = torch.zeros(2, 3, 5, device=gpu), torch.zeros(2, 3, dtype=torch.int64, device=gpu), torch.zeros(2, device=gpu)
    with pytest.raises(F._lib.AttentionError):
        F.preference_loss(x, t, r, workspace=torch.empty(5, dtype=torch.float64, device=gpu))
    assert torch.equal(F.preference_loss(x, t, r, workspace=torch.empty(3, 2, dtype=torch.float64, device=gpu).t()), F.preference_loss(x, t, r))
