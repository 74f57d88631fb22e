"""Scored attention where it takes the documents' work order (query grids of more than
640 workgroups), and capped dK/dV with two workgroups on a CU (512 unsplit items and
more), against the float64 oracle; the order's tables recounted from the masks."""
import numpy as np
import pytest
import torch

import femtochat_amd as F
from femtochat_amd import workloads as W
from oracle import attention_score as S

from tests.test_gpu_attn_score import A, _check, _dev, _inputs, _options, _run

pytestmark = pytest.mark.gpu


def _up(n):
    return (n + 255) // 256 * 256


def _room(B, T, H, prefix, positions, ordered):
    """Bytes of the backward's workspace without a split's parts: Delta, lse2, bounds,
    counters, the two orders, upper bounds."""
    chunks, order = _up(B * -(-T // 32) * 8), _up(B * -(-T // 128) * 4)
    return 2 * _up(B * T * H * 4) + (chunks if positions or prefix else 0) + 256 + (2 * order if ordered else 0) + (chunks if prefix else 0)


def _orders(T, window, pos, prefix):
    """(qorder, korder): items by decreasing work, ties by index."""
    left = T if window == (-1, 0) else window[0]
    lbs, ubs = S.bounds(T, window, pos, prefix)
    n = -(-T // 128)
    q, k = [], []
    for lb, ub in zip(lbs, ubs):
        lo = [int(lb[128 * t:128 * t + 128].min()) for t in range(n)]
        hi = [int(ub[128 * t:128 * t + 128].max()) for t in range(n)]
        q += [h // 64 - x // 64 + 1 for x, h in zip(lo, hi)]
        for t in range(n):
            k0, k1 = 128 * t, min(128 * t + 128, T) - 1
            last = min(T - 1, k1 + left) // 128
            first = 0 if prefix is not None else max(0, k0 - window[1]) // 128
            k.append(sum(lo[u] <= k1 and (prefix is None or hi[u] >= k0) for u in range(first, last + 1)))
    return np.argsort(-np.array(q), kind="stable"), np.argsort(-np.array(k), kind="stable")


@pytest.mark.parametrize("kind", ["prefix", "cap+prefix", "bias+prefix", "all", "cap", "bias"])
@pytest.mark.parametrize("B,T,H,Hkv,D", [(14, 300, 16, 4, 64), (11, 400, 16, 8, 128), (14, 300, 16, 4, 32), (14, 260, 16, 8, 96)])
@pytest.mark.parametrize("window", [(-1, 0), (90, 0)])
def test_documents_in_the_work_order(gpu, kind, B, T, H, Hkv, D, window):
    n128 = -(-T // 128)
    assert B * n128 * H > 640
    host = _inputs(T + D, B, T, H, Hkv, D)
    pos = W.document_positions(T, B, T, mean=110, sigma=1.0, cap=T)
    how = _options(kind, T, B, T, H, per_token=True)
    prefix = how["prefix"]
    if prefix is not None:
        prefix = how["prefix"] = (prefix % 90).astype(np.int32)
    _check(_run(gpu, host, window, pos, how), host, window, pos, how)
    if D == 96:
        return  # (its workspace begins with room for tensors off a 16-byte boundary)
    # the tables that the forward and the backward leave in their workspaces
    Q, K, V, dO = (x.to(gpu) for x in host)
    d, p = _dev(gpu, how), torch.from_numpy(pos).to(gpu)
    O, l, m = torch.empty_like(Q), torch.empty(B, H, T, device=gpu), torch.empty(B, H, T, device=gpu)
    grads = [torch.empty_like(x) for x in (Q, K, V)]
    chunks, items = _up(B * -(-T // 32) * 8), B * n128
    fws = torch.empty(F.forward_workspace_bytes(A, Q, K, positions=p, **d), dtype=torch.uint8, device=gpu)
    bws = torch.empty(F.backward_workspace_bytes(A, Q, K, positions=p, **d), dtype=torch.uint8, device=gpu)
    assert fws.data_ptr() % 256 == 0 and bws.data_ptr() % 256 == 0
    assert fws.numel() == chunks + _up(4 * items) + (chunks if prefix is not None else 0) + 256
    F.attention_(A, O, l, m, Q, K, V, window, positions=p, workspace=fws, **d)
    F.delta_attention_(A, *grads, dO, Q, K, V, O, l, m, window, positions=p, accumulate=False, workspace=bws, **d)
    qorder, korder = _orders(T, window, pos, prefix)

    def table(ws, at):
        return ws[at:at + 4 * items].view(torch.int32).cpu().numpy()

    assert np.array_equal(table(fws, chunks), qorder)
    at = 2 * _up(B * T * H * 4) + chunks + 256
    assert np.array_equal(table(bws, at), qorder) and np.array_equal(table(bws, at + _up(4 * items)), korder)


@pytest.mark.parametrize("kind", ["cap", "cap+bias", "cap+prefix", "all"])
@pytest.mark.parametrize("D", [16, 32, 48, 64])
@pytest.mark.parametrize("documents,B", [(False, 11), (True, 11), (True, 14)])
@pytest.mark.parametrize("window", [(-1, 0), (70, 0), (40, 25)])
def test_two_workgroups_on_a_cu(gpu, kind, D, documents, B, window):
    T, H = 270, 16
    assert B * -(-T // 128) * H >= 512
    host = _inputs(T + D, B, T, H, H, D)
    pos = W.document_positions(T, B, 3, mean=80, sigma=1.0, cap=T) if documents else None
    how = _options(kind, D, B, T, H, per_token=documents)
    if documents and how["prefix"] is not None:
        how["prefix"] = (how["prefix"] % 60).astype(np.int32)
    Q, K = host[0], host[1]
    given = dict(positions=pos, softcap=how["softcap"], slopes=how["slopes"], prefix=how["prefix"])
    if D != 48:  # unsplit: no parts in the workspace
        room = _room(B, T, H, how["prefix"] is not None, documents, documents and B * 3 * H > 640)
        assert F.backward_workspace_bytes(A, Q, K, **given) == room + 256
    got = _run(gpu, host, window, pos, how)
    _check(got, host, window, pos, how)
    added = _run(gpu, host, window, pos, how, grad=torch.float32, init=0.5)
    for x, y in zip(got[3:], added[3:]):  # got is rounded to bf16 once
        assert ((y - x.float() - 0.5).abs() <= 2.0 ** -8 * x.float().abs() + 1e-6).all()
