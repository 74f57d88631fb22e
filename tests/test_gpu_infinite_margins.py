"""Pairs of answers whose margin is infinite."""
import pytest
import torch

import femtochat_amd as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("smoothing", [0.0, 0.25, 1.0])
def test_infinite_margins(gpu, smoothing):
    """A token with a logit of -inf in the chosen answer, in the rejected one, in both."""
    P, T, V, beta = 3, 2, 8, 0.1
    x = torch.zeros(2 * P, T, V)
    tok = torch.zeros(2 * P, T, dtype=torch.int64)
    for answer in (0, P + 1, 2, P + 2):
        x[answer, 1, 3], tok[answer, 1] = -float("inf"), 3
    xd = x.to(gpu).requires_grad_()
    loss, rewards = F.PreferenceLossFunction.apply(xd, tok.to(gpu), torch.zeros(2 * P, device=gpu), beta, smoothing, -1, "none")
    inf = float("inf")
    want = [0.0 if smoothing == 1.0 else inf, 0.0 if smoothing == 0.0 else inf]
    assert loss.detach()[:2].tolist() == want and torch.isnan(loss[2])
    assert rewards[[0, P + 1]].tolist() == [-inf, -inf]
    g = torch.autograd.grad(loss[:2].sum(), xd)[0].double().cpu()
    # the logistic function is 0 and 1: w = -beta (1 - e) for the first pair, beta e for the second
    for pair, w in ((0, -beta * (1 - smoothing)), (1, beta * smoothing)):
        for answer, sign in ((pair, 1), (pair + P, -1)):
            p = torch.softmax(x[answer].double(), -1)
            onehot = torch.nn.functional.one_hot(tok[answer], V)
            assert (g[answer] - sign * w * (onehot - p)).abs().max() <= 2.0 ** -20 * beta
