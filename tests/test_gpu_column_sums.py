"""The sum over a column where almost all of it is one value: the log-probability of the
likeliest token, from both of the policy loss's entry points."""
import math

import pytest
import torch

import femtochat_amd as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1000, 4000, 8192, 32768, 50257, 65533])
def test_the_likeliest_token(gpu, dtype, V):
    """One logit of 0, all others -25: lp = -log(1 + (V - 1) e^-25), up to 1e-6, of which the
    sums of 64 and more threads beside the one with the maximum are each below 2^-24.  That
    one's own further values, at most 256, may drop out of its float32 sum; each exponential
    is within 30 2^-23 of its value."""
    B, T = 1, 4
    x = torch.full((B, T, V), -25.0, dtype=dtype, device=gpu)
    tok = torch.tensor([[0, 77, V // 2, V - 1]], device=gpu)
    x.scatter_(-1, tok[..., None], 0.0)
    old, adv = torch.zeros(B, T, device=gpu), torch.ones(B, device=gpu)
    small = math.exp(-25.0)
    want, room = -math.log1p((V - 1) * small), 256 * small + 30 * 2.0 ** -23 * V * small
    lps = [torch.empty(B, T, device=gpu) for _ in range(2)]
    losses, delta = torch.empty(B, T, device=gpu), torch.empty_like(x)
    F.policy_loss_(losses, x, tok, old, adv, logprobs=lps[0])
    F.policy_loss_fused_(losses, delta, x, tok, old, adv, logprobs=lps[1])
    for lp in lps:
        assert (lp.double() - want).abs().max().item() <= room


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,off", [(1000, 0), (4000, 1), (8192, 0), (8191, 3), (32768, 0), (50257, 0), (65533, 0)])
def test_the_likeliest_tokens_own_thread(gpu, dtype, V, off):
    """The same with logits of -19, of which 4 to 8 together are below half a step beside 1:
    only the chunk of the likeliest token itself, up to 8 values with it, may lose its others."""
    B, T = 1, 5
    x = torch.empty(B * T * V + off, dtype=dtype, device=gpu)[off:].view(B, T, V).fill_(-19.0)
    tok = torch.tensor([[0, 77, V // 2, V - 2, V - 1]], device=gpu)
    x.scatter_(-1, tok[..., None], 0.0)
    old, adv = torch.zeros(B, T, device=gpu), torch.ones(B, device=gpu)
    small = math.exp(-19.0)
    want, room = -math.log1p((V - 1) * small), 8 * small + 30 * 2.0 ** -23 * V * small
    lps = [torch.empty(B, T, device=gpu) for _ in range(2)]
    losses, delta = torch.empty(B, T, device=gpu), torch.empty(B * T * V + off, dtype=dtype, device=gpu)[off:].view(B, T, V)
    F.policy_loss_(losses, x, tok, old, adv, logprobs=lps[0])
    F.policy_loss_fused_(losses, delta, x, tok, old, adv, logprobs=lps[1])
    for lp in lps:
        assert (lp.double() - want).abs().max().item() <= room
