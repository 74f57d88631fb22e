"""The longest columns of the one-pass policy loss: the call and autograd agree on which
they are, and the results at the limit."""
import numpy as np
import pytest
import torch

import femtochat_amd as F
from oracle import answer_loss as O

from tests.test_gpu_answer_loss import CLIP, LP, _check_gradient, _dev, _logits, _policy_inputs, _tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,V,off,fits", [
    ("f32", 65533, 0, True), ("f32", 65533, 3, True), ("f32", 65534, 0, False), ("f32", 65532, 0, True), ("f32", 65532, 1, True),
    ("f32", 65536, 0, True), ("f32", 65536, 1, False), ("f32", 65537, 0, False),
    ("bf16", 131065, 0, True), ("bf16", 131065, 7, True), ("bf16", 131066, 0, False), ("bf16", 131064, 5, True),
    ("bf16", 131072, 0, True), ("bf16", 131072, 1, False), ("bf16", 131073, 0, False),
])
def test_the_longest_columns(gpu, dtype, V, off, fits):
    B, T = 1, 3
    x, xd = _logits(gpu, 13, B, T, V, dtype, off=off)
    tok = _tokens(14, B, T, V, "none")
    old, ref, adv = _policy_inputs(15, x, tok, True)
    td, od, rd, ad = _dev(gpu, tok, old, ref, adv)
    loss, g, w = O.policy(x, tok, old, adv, ref, CLIP, 0.1, dy=1.0 / 3)
    lp, _ = O.log_probs(x, tok)
    slope = (np.abs(adv)[:, None] * np.exp(lp - old) + 0.1 * np.exp(ref - lp)) / 3
    room = torch.empty(xd.numel() + off, dtype=xd.dtype, device=gpu)
    losses, delta = torch.empty(B, T, device=gpu), room[off:].view(B, T, V)
    how = dict(ref_logprobs=rd, clip=CLIP, kl=0.1)
    if fits:
        F.policy_loss_fused_(losses, delta, xd, td, od, ad, **how)
        _check_gradient(delta, g, np.abs(w) / 3 + slope, dtype)
        assert (np.abs(losses.double().cpu().numpy() - loss) <= LP * (1 + 6 * slope)).all()
    else:
        with pytest.raises(F._lib.AttentionError, match="256 KB"):
            F.policy_loss_fused_(losses, delta, xd, td, od, ad, **how)
    xd.requires_grad_()
    out = F.PolicyLossFunction.apply(xd, td, od, ad, rd, CLIP, 0.1, -1, "mean")
    assert (out.grad_fn.delta is not None) == fits  # formed beside the loss, in one pass
    got = torch.autograd.grad(out, xd)[0]
    _check_gradient(got, g, np.abs(w) / 3 + slope, dtype)
    if fits:
        assert torch.equal(got, delta)
