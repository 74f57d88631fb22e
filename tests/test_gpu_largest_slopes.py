"""Slopes up to float32's largest."""
import numpy as np
import pytest
import torch

import femtochat_amd as F
from oracle import attention_score as S

from tests.test_gpu_attn_score import _inputs, _np, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [16, 64, 96, 128])
@pytest.mark.parametrize("softcap", [0.0, 5.0])
@pytest.mark.parametrize("T", [3, 70, 900])
def test_the_largest_slopes(gpu, D, softcap, T):
    """A query sees its own key at its score and nothing else: O is V's row, dV dO's, and dQ
    and dK hold only what a float32 sum over the head dimension leaves of dP - Delta."""
    B, H = 1, 4
    host = _inputs(3, B, T, H, H, D)
    big = float(np.finfo(np.float32).max)
    how = dict(softcap=softcap, slopes=np.array([big, 2.5e38, 2.3e38, 1e30], np.float32), prefix=None)
    O, l, m, dQ, dK, dV = _run(gpu, host, (-1, 0), None, how)
    assert torch.equal(O.cpu(), host[2]) and torch.equal(dV.cpu(), host[3])
    Q, K, V, dO = (x.double().numpy() for x in host)
    _, l64, m64 = S.forward(Q, K, V, (-1, 0), None, **how)
    assert (_np(l) == l64).all()
    assert np.abs(_np(m) - m64).max() <= 2.0 ** -20 * (np.abs(m64).max() + softcap)
    # |dP - Delta| <= 2 D 2^-24 max|dO V| over the sum, times a row of K or Q over sqrt(D)
    room = 2 * D * 2.0 ** -24 * np.abs(dO).max() * np.abs(V).max() * max(np.abs(Q).max(), np.abs(K).max())
    assert np.abs(_np(dQ)).max() <= room and np.abs(_np(dK)).max() <= room
