"""The operators for fine-tuning on prompts and answers: what is measured, on which inputs, in plain form and by the framework.

Three groups: attention with capped scores, a distance bias and a prefix mask (forward, forward + backward), the clipped policy
loss with a KL term, and the preference loss over pairs of answers (each with the gradient of the logits).
``run`` computes the plain form in elementary torch operations, or, with ``own``, makes the framework's calls.
"""
import math

import numpy as np
import torch

own = False
DEV = "cuda"


def listed():
    return [
        # The smallest attention call: a toy layer (2 x 16 tokens, 2 heads of 16), capped and biased, one training step
        # through autograd.  Only launches and host work count.
        dict(name="toy_capped_step", kind="attention", entry="autograd", B=2, T=16, H=2, Hkv=1, D=16, left=-1, softcap=30.0,
             bias=True, mask="plain"),
        # One layer of the training script's default model (8 heads of 64, 4 x 2048 tokens) with capped scores.
        dict(name="capped_step", kind="attention", entry="autograd", B=4, T=2048, H=8, Hkv=8, D=64, left=-1, softcap=50.0,
             bias=False, mask="plain"),
        # The headline layer (n_embed 1280, GQA 2:1, 16 x 2048 tokens) with capped scores, into buffers the caller keeps.
        dict(name="capped_gqa_step", kind="attention", entry="buffers", B=16, T=2048, H=10, Hkv=5, D=128, left=-1, softcap=50.0,
             bias=False, mask="plain"),
        # The same width with a distance bias in place of rotary positions, through autograd.
        dict(name="biased_step", kind="attention", entry="autograd", B=4, T=2048, H=8, Hkv=4, D=128, left=-1, softcap=0.0,
             bias=True, mask="plain"),
        # Packed prompt-answer documents in a long row: each document's prompt sees itself in both directions.
        dict(name="prefix_documents_step", kind="attention", entry="autograd", B=1, T=8192, H=16, Hkv=8, D=128, left=-1,
             softcap=0.0, bias=False, mask="prefix_documents"),
        # Evaluation of one prompt of odd length, capped and biased, 96-wide heads: forward only.
        dict(name="biased_eval", kind="attention", entry="forward", B=1, T=777, H=8, Hkv=4, D=96, left=-1, softcap=30.0,
             bias=True, mask="prefix"),
        # The smallest policy step: a few short answers over a byte vocabulary, fp32 logits, through autograd.
        dict(name="policy_small", kind="policy", entry="autograd", dtype="fp32", B=2, T=12, V=259, kl=0.05),
        # A policy step over 8 sampled answers of 1024 tokens, bf16 logits over a vocabulary of 2^15, through autograd.
        dict(name="policy_step", kind="policy", entry="autograd", dtype="bf16", B=8, T=1024, V=32768, kl=0.05),
        # Odd lengths, an odd vocabulary and fp32 logits: the loss and its gradient in one call, as the step's last node.
        dict(name="policy_ragged_fused", kind="policy", entry="fused", dtype="fp32", B=6, T=333, V=50257, kl=0.0),
        # The smallest preference step: two pairs of short answers, fp32 logits, through autograd.
        dict(name="preference_small", kind="preference", dtype="fp32", P=2, T=33, V=1000, smoothing=0.0),
        # A preference step over 4 pairs of 1024 tokens, bf16 logits over a vocabulary of 2^15, through autograd.
        dict(name="preference_step", kind="preference", dtype="bf16", P=4, T=1024, V=32768, smoothing=0.0),
        # Odd lengths, an odd vocabulary, fp32 logits, smoothed labels.
        dict(name="preference_ragged", kind="preference", dtype="fp32", P=3, T=377, V=50257, smoothing=0.1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["attention", "policy", "preference"], [6, 3, 3])[0]
    if kind == "attention":
        entry = rng.choices(["autograd", "buffers", "forward"], [4, 2, 3])[0]
        H = rng.choice([1, 2, 4, 6, 8, 10, 12, 16])
        Hkv = H // rng.choice([r for r in (1, 1, 2, 4, 5) if H % r == 0])
        D = rng.choices([16, 32, 48, 64, 80, 96, 112, 128], [1, 1, 1, 5, 1, 2, 1, 6])[0]
        T, B = _log(rng, 1 if entry == "forward" else 16, 8192), _log(rng, 1, 16)
        # no draw costs more than the largest above, in products or in score matrices of the plain form
        while B > 1 and (B * H * T * T > 6.0e8 or B * H * T * T * D > 8.0e10):
            B -= 1
        while B * H * T * T > 6.0e8 or B * H * T * T * D > 8.0e10:
            T = T * 3 // 4
        return dict(kind=kind, entry=entry, B=B, T=T, H=H, Hkv=Hkv, D=D,
                    left=rng.choice([-1, -1, min(T, -(-T // 512) * 128), rng.randint(0, T)]),
                    softcap=rng.choice([0.0, 15.0, 30.0, 50.0, round(rng.uniform(10.0, 100.0), 2)]),
                    bias=rng.choice([True, False]), mask=rng.choice(["plain", "documents", "prefix", "prefix_documents"]))
    dtype = rng.choice(["bf16", "fp32"])
    V = rng.choice([8192, 32768, _log(rng, 50, 50257), 50257, 50304])
    rows = _log(rng, 4, min(8192, (1 << 28) // V))
    if kind == "policy":
        B = _log(rng, 1, min(64, rows))
        return dict(kind=kind, entry=rng.choice(["autograd", "fused"]), dtype=dtype, B=B, T=max(1, rows // B), V=V,
                    kl=rng.choice([0.0, 0.01, 0.05, 0.2]))
    P = _log(rng, 1, max(1, min(32, rows // 2)))
    return dict(kind=kind, dtype=dtype, P=P, T=max(1, rows // (2 * P)), V=V, smoothing=rng.choice([0.0, 0.0, 0.1]))


# ---- inputs ---------------------------------------------------------------------------------------------------------

CLIP = (0.2, 0.25)  # below and above 1
BETA = 0.1          # the preference loss's scale
IGNORE = -1


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def _masks(case, seed):
    """(positions, prefix): positions (B, T) restart at each document, prefix is the prompt's length, of each row (B,) or of
    each token's document (B, T).  Documents have lognormal lengths (mean 400), prompts 10 to 60% of theirs."""
    B, T, mask = case["B"], case["T"], case["mask"]
    rng = np.random.default_rng([int(seed), 77])
    if mask == "plain":
        return None, None
    if mask == "prefix":
        return None, rng.integers(0, T // 2 + 1, B).astype(np.int32)
    pos, pre = np.zeros((B, T), np.int32), np.zeros((B, T), np.int32)
    for b in range(B):
        t = 0
        while t < T:
            n = int(min(T - t, 4096, max(1, round(float(rng.lognormal(math.log(400.0) - 0.5, 1.0))))))
            pos[b, t:t + n] = np.arange(n)
            pre[b, t:t + n] = int(n * rng.uniform(0.1, 0.6))
            t += n
    return pos, (pre if mask == "prefix_documents" else None)


def _slopes(H):
    """Geometric slopes from 2^(-8/H) to 2^-8."""
    return [2.0 ** (-8.0 * (h + 1) / H) for h in range(H)]


def _attention_inputs(case, seed):
    g = _gen(seed)
    B, T, H, Hkv, D = (case[k] for k in ("B", "T", "H", "Hkv", "D"))
    # scores with a standard deviation of 3: some of them near the caps
    Q, K = (3.0 * _randn(g, B, T, H, D)).bfloat16(), _randn(g, B, T, Hkv, D).bfloat16()
    V, dO = _randn(g, B, T, Hkv, D).bfloat16(), (0.1 * _randn(g, B, T, H, D)).bfloat16()
    pos, pre = _masks(case, seed)
    return dict(Q=Q, K=K, V=V, dO=dO, window=(case["left"], 0), softcap=case["softcap"],
                positions=None if pos is None else torch.from_numpy(pos).to(DEV),
                prefix=None if pre is None else torch.from_numpy(pre).to(DEV),
                slopes=torch.tensor(_slopes(H), dtype=torch.float32, device=DEV) if case["bias"] else None)


def _logits(g, rows, T, V, dtype):
    """Logits, tokens drawn from their softmax, and those tokens' log-probabilities, a block of rows at a time."""
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    x = torch.empty(rows * T, V, dtype=dt, device=DEV)
    tok = torch.empty(rows * T, dtype=torch.int64, device=DEV)
    lp = torch.empty(rows * T, dtype=torch.float64, device=DEV)
    step = max(1, (1 << 25) // V)
    for i in range(0, rows * T, step):
        b = x[i:i + step]
        b.copy_(2.5 * torch.randn(b.shape, device=DEV, generator=g))
        f = b.float()
        u = torch.rand(b.shape, device=DEV, generator=g).clamp_(1e-10, 1.0 - 1e-7)
        tok[i:i + step] = (f - torch.log(-torch.log(u))).argmax(-1)
        d = f.double()
        lp[i:i + step] = d.gather(-1, tok[i:i + step, None])[:, 0] - torch.logsumexp(d, -1)
    return x.view(rows, T, V), tok.view(rows, T), lp.view(rows, T)


def _answers(seed, rows, T):
    """Which tokens belong to answers: a prompt in front and padding behind them are not trained on."""
    rng = np.random.default_rng([int(seed), 78])
    start = (T * rng.uniform(0.0, 0.3, rows)).astype(int)
    end = np.maximum(start + 1, T - (T * rng.uniform(0.0, 0.3, rows)).astype(int))
    t = np.arange(T)
    return torch.from_numpy((t >= start[:, None]) & (t < end[:, None])).to(DEV)


def _policy_inputs(case, seed):
    g = _gen(seed)
    B, T = case["B"], case["T"]
    x, tok, lp = _logits(g, B, T, case["V"], case["dtype"])
    # the policy has moved a little since the answers were drawn, and further from where training began
    old, ref = lp + 0.15 * _randn(g, B, T), lp + 0.3 * _randn(g, B, T)
    return dict(logits=x, tokens=torch.where(_answers(seed, B, T), tok, IGNORE), old=old.float(),
                ref=ref.float() if case["kl"] > 0 else None, advantages=_randn(g, B), kl=case["kl"])


def _preference_inputs(case, seed):
    g = _gen(seed)
    P, T = case["P"], case["T"]
    x, tok, lp = _logits(g, 2 * P, T, case["V"], case["dtype"])
    on = _answers(seed, 2 * P, T)
    ref = (lp * on).sum(-1) + 5.0 * _randn(g, 2 * P)  # the reference model's sums, within the spread that training reaches
    return dict(logits=x, tokens=torch.where(on, tok, IGNORE), ref=ref.float(), smoothing=case["smoothing"])


def prepare(case, seed):
    kind = case["kind"]
    s = {"attention": _attention_inputs, "policy": _policy_inputs, "preference": _preference_inputs}[kind](case, seed)
    s.update(kind=kind, entry=case.get("entry", "autograd"))
    if s["entry"] == "autograd":
        for k in ("Q", "K", "V") if kind == "attention" else ("logits",):
            s[k].requires_grad_()
    if s["entry"] == "buffers":  # a program with buffers of its own keeps the outputs and statistics too
        B, T, H = case["B"], case["T"], case["H"]
        s.update(O=torch.empty_like(s["Q"]), l=torch.empty(B, H, T, device=DEV), m=torch.empty(B, H, T, device=DEV),
                 dQ=torch.empty_like(s["Q"]), dK=torch.empty_like(s["K"]), dV=torch.empty_like(s["V"]))
    if s["entry"] == "fused":
        s.update(losses=torch.empty(case["B"], case["T"], device=DEV), delta=torch.empty_like(s["logits"]),
                 reduced=torch.empty(1, device=DEV))
    return s


# ---- the framework's calls ------------------------------------------------------------------------------------------


def _own_attention(s):
    import femtochat_amd as F

    how = dict(positions=s["positions"], softcap=s["softcap"], slopes=s["slopes"], prefix=s["prefix"])
    if s["entry"] == "forward":
        return F.attention(s["Q"], s["K"], s["V"], s["window"], **how)
    if s["entry"] == "buffers":
        A = F.MFMAFast()
        F.attention_(A, s["O"], s["l"], s["m"], s["Q"], s["K"], s["V"], s["window"], **how)
        F.delta_attention_(A, s["dQ"], s["dK"], s["dV"], s["dO"], s["Q"], s["K"], s["V"], s["O"], s["l"], s["m"], s["window"],
                           accumulate=False, **how)
        return s["O"], s["dQ"], s["dK"], s["dV"]
    O = F.AttentionFunction.apply(s["Q"], s["K"], s["V"], s["window"], None, s["positions"], s["softcap"], s["slopes"], s["prefix"])
    return (O.detach(),) + torch.autograd.grad(O, (s["Q"], s["K"], s["V"]), s["dO"])


def _own_policy(s):
    import femtochat_amd as F

    if s["entry"] == "fused":
        F.policy_loss_fused_(s["losses"], s["delta"], s["logits"], s["tokens"], s["old"], s["advantages"], ref_logprobs=s["ref"],
                             clip=CLIP, kl=s["kl"], ignore_index=IGNORE, reduction="mean", reduced=s["reduced"])
        return s["reduced"][0], s["delta"]
    loss = F.PolicyLossFunction.apply(s["logits"], s["tokens"], s["old"], s["advantages"], s["ref"], CLIP, s["kl"], IGNORE, "mean")
    return loss.detach(), torch.autograd.grad(loss, s["logits"])[0]


def _own_preference(s):
    import femtochat_amd as F

    loss, rewards = F.PreferenceLossFunction.apply(s["logits"], s["tokens"], s["ref"], BETA, s["smoothing"], IGNORE, "mean")
    return loss.detach(), rewards, torch.autograd.grad(loss, s["logits"])[0]


# ---- the plain forms ------------------------------------------------------------------------------------------------


def _visible(T, left, positions, prefix):
    """(B or 1, T, T): which keys (last) a query sees."""
    q, k = torch.arange(T, device=DEV)[:, None], torch.arange(T, device=DEV)[None, :]
    start = torch.zeros(1, T, 1, dtype=torch.int64, device=DEV) if positions is None else (q[:, 0] - positions.long()).clamp(min=0)[:, :, None]
    lo = start if left < 0 else torch.maximum(start, q - left)
    hi = q
    if prefix is not None:
        hi = torch.maximum(q, start + (prefix[:, None, None] if prefix.dim() == 1 else prefix[:, :, None]) - 1)
    return (k >= lo) & (k <= hi)


def _plain_attention(s):
    Q, K, V, dO = (s[n].detach().float().transpose(1, 2) for n in ("Q", "K", "V", "dO"))
    B, H, T, D = Q.shape
    Hkv = K.shape[1]
    G, scale = H // Hkv, 1.0 / math.sqrt(D)
    Q, dO = Q.reshape(B, Hkv, G, T, D), dO.reshape(B, Hkv, G, T, D)
    Kx, Vx = K[:, :, None].expand(B, Hkv, G, T, D).contiguous(), V[:, :, None].expand(B, Hkv, G, T, D).contiguous()
    S = torch.matmul(Q, Kx.transpose(-1, -2).contiguous()) * scale
    t = None
    if s["softcap"] > 0:
        t = torch.tanh(S / s["softcap"])
        S = s["softcap"] * t
    if s["slopes"] is not None:
        i = torch.arange(T, device=DEV, dtype=torch.float32)
        S = S - s["slopes"].view(1, Hkv, G, 1, 1) * (i[:, None] - i[None, :]).abs()
    seen = _visible(T, s["window"][0], s["positions"], s["prefix"])[:, None, None]
    S = S.masked_fill(~seen, -math.inf)
    m = S.amax(-1, keepdim=True)
    P = torch.exp(S - torch.where(torch.isinf(m), 0.0, m))
    l = P.sum(-1, keepdim=True)
    P = P / torch.where(l > 0, l, 1.0)
    O = torch.matmul(P, Vx)
    out = O.reshape(B, H, T, D).transpose(1, 2).to(s["Q"].dtype).contiguous()
    if s["entry"] == "forward":
        return out
    dV = torch.matmul(P.transpose(-1, -2).contiguous(), dO).sum(2)
    dS = P * (torch.matmul(dO, Vx.transpose(-1, -2).contiguous()) - (dO * O).sum(-1, keepdim=True))
    dS = dS.masked_fill(seen.sum(-1, keepdim=True) <= 1, 0.0)  # a row with one key has P = 1 whatever its score is
    if t is not None:
        dS = dS * (1.0 - t * t)
    dQ = torch.matmul(dS, Kx) * scale
    dK = torch.matmul(dS.transpose(-1, -2).contiguous(), Q).sum(2) * scale
    back = lambda x, like: x.reshape(B, -1, T, D).transpose(1, 2).to(like.dtype).contiguous()  # noqa: E731
    return out, back(dQ, s["Q"]), back(dK, s["K"]), back(dV, s["V"])


def _plain_logprobs(x, tokens):
    """(valid, index, log-sum-exp, log-probability); sums over the vocabulary and what follows in 64 bits: a ratio next to its
    clip and a difference of long sums need them."""
    valid = tokens != IGNORE
    idx = torch.where(valid, tokens, 0)[..., None]
    m = x.amax(-1, keepdim=True)
    lse = m.double() + torch.log(torch.exp((x - m).double()).sum(-1, keepdim=True))
    return valid, idx, lse, (x.gather(-1, idx).double() - lse)[..., 0]


def _plain_gradient(x, idx, lse, w, dtype):
    """w (onehot - softmax) for each token."""
    g = torch.exp(x - lse.float()) * -w.float()[..., None]
    g.scatter_add_(-1, idx, w.float()[..., None])
    return g.to(dtype)


def _plain_policy(s):
    x = s["logits"].detach().float()
    valid, idx, lse, lp = _plain_logprobs(x, s["tokens"])
    A = s["advantages"].double()[:, None]
    r = torch.exp(lp - s["old"])
    capped = r.clamp(1.0 - CLIP[0], 1.0 + CLIP[1]) * A
    loss = -torch.minimum(r * A, capped)
    w = torch.where(r * A <= capped, -r * A, 0.0)
    if s["ref"] is not None:
        d = s["ref"] - lp
        loss = loss + s["kl"] * (torch.exp(d) - d - 1.0)
        w = w + s["kl"] * (1.0 - torch.exp(d))
    n = valid.sum()
    loss = torch.where(valid, loss, 0.0).sum() / n
    return loss.float(), _plain_gradient(x, idx, lse, torch.where(valid, w, 0.0) / n, s["logits"].dtype)


def _plain_preference(s):
    x = s["logits"].detach().float()
    valid, idx, lse, lp = _plain_logprobs(x, s["tokens"])
    e, P = s["smoothing"], x.shape[0] // 2
    reward = BETA * (torch.where(valid, lp, 0.0).sum(-1) - s["ref"])
    h = reward[:P] - reward[P:]
    softplus = lambda z: torch.clamp(z, min=0.0) + torch.log1p(torch.exp(-z.abs()))  # noqa: E731
    loss = ((1.0 - e) * softplus(-h) + e * softplus(h)).mean()
    dh = (e / (1.0 + torch.exp(-h)) - (1.0 - e) / (1.0 + torch.exp(h))) * (BETA / P)
    w = torch.where(valid, torch.cat([dh, -dh])[:, None], 0.0)
    return loss.float(), reward.float(), _plain_gradient(x, idx, lse, w, s["logits"].dtype)


def run(s):
    if own:
        return {"attention": _own_attention, "policy": _own_policy, "preference": _own_preference}[s["kind"]](s)
    with torch.no_grad():
        return {"attention": _plain_attention, "policy": _plain_policy, "preference": _plain_preference}[s["kind"]](s)


# ---- what each path cannot do without -------------------------------------------------------------------------------


def work(case):
    if case["kind"] == "attention":
        B, T, H, Hkv, D = (case[k] for k in ("B", "T", "H", "Hkv", "D"))
        pos, pre = _masks(case, 0)  # the masks of one seed stand for all
        q = np.arange(T)[None, :]
        start = np.zeros((1, T), int) if pos is None else q - pos
        lo = start if case["left"] < 0 else np.maximum(start, q - case["left"])
        hi = q if pre is None else np.maximum(q, start + (pre[:, None] if pre.ndim == 1 else pre) - 1)
        pairs = H * int(np.broadcast_to(np.minimum(hi, T - 1) - lo + 1, (B, T)).sum())
        nq, nk = B * T * H * D, B * T * Hkv * D
        if case["entry"] == "forward":
            return dict(bytes=2 * (2 * nq + 2 * nk), flops=4 * D * pairs)
        return dict(bytes=2 * (4 * nq + 4 * nk), flops=14 * D * pairs)
    rows = (case["B"] if case["kind"] == "policy" else 2 * case["P"]) * case["T"]
    n = rows * case["V"]
    return dict(bytes=2 * n * (2 if case["dtype"] == "bf16" else 4) + 24 * rows, flops=8 * n)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------


def _exact_attention(case, seed):
    s = _attention_inputs(case, seed)
    Q, K, V, dO = (s[n].double() for n in ("Q", "K", "V", "dO"))
    B, T, H, D = Q.shape
    G, c = H // K.shape[2], s["softcap"]
    O, dQ, dK, dV = (torch.zeros_like(x) for x in (Q, Q, K, V))
    i = torch.arange(T, device=DEV)
    dist = (i[:, None] - i[None, :]).abs().double()
    hidden = None
    for b in range(B):
        if hidden is None or s["positions"] is not None or s["prefix"] is not None:
            row = lambda x: None if x is None else x[b:b + 1]  # noqa: E731
            hidden = ~_visible(T, case["left"], row(s["positions"]), row(s["prefix"]))[0]
            lone = (~hidden).sum(-1) <= 1
        for h in range(H):
            k, v = K[b, :, h // G], V[b, :, h // G]
            x = Q[b, :, h] @ k.T / math.sqrt(D)
            z = c * torch.tanh(x / c) if c > 0 else x
            if s["slopes"] is not None:
                z = z - float(s["slopes"][h]) * dist
            p = torch.softmax(z.masked_fill(hidden, -math.inf), -1)  # every query here sees itself
            O[b, :, h] = p @ v
            if case["entry"] == "forward":
                continue
            dp = dO[b, :, h] @ v.T
            ds = p * (dp - (p * dp).sum(-1, keepdim=True))
            ds[lone] = 0.0
            if c > 0:
                ds = ds / torch.cosh(x / c) ** 2
            dQ[b, :, h] = ds @ k / math.sqrt(D)
            dK[b, :, h // G] += ds.T @ Q[b, :, h] / math.sqrt(D)
            dV[b, :, h // G] += p.T @ dO[b, :, h]
    return O if case["entry"] == "forward" else (O, dQ, dK, dV)


def _exact_policy(case, seed):
    s = _policy_inputs(case, seed)
    x = s["logits"].double().requires_grad_()
    on = s["tokens"] >= 0
    lp = torch.log_softmax(x, -1).gather(-1, s["tokens"].clamp(min=0)[..., None])[..., 0]
    r, A = torch.exp(lp - s["old"].double()), s["advantages"].double()[:, None].expand_as(lp)
    loss = torch.where(A >= 0, -A * r.clamp(max=1.0 + CLIP[1]), -A * r.clamp(min=1.0 - CLIP[0]))
    if s["ref"] is not None:
        loss = loss + s["kl"] * (torch.expm1(s["ref"].double() - lp) - (s["ref"].double() - lp))
    loss = loss[on].mean()
    return loss.detach(), torch.autograd.grad(loss, x)[0]


def _exact_preference(case, seed):
    s = _preference_inputs(case, seed)
    x = s["logits"].double().requires_grad_()
    lp = torch.log_softmax(x, -1).gather(-1, s["tokens"].clamp(min=0)[..., None])[..., 0]
    reward = BETA * ((lp * (s["tokens"] >= 0)).sum(-1) - s["ref"].double())
    h = reward[:case["P"]] - reward[case["P"]:]
    logsigma = torch.nn.functional.logsigmoid
    loss = -((1.0 - case["smoothing"]) * logsigma(h) + case["smoothing"] * logsigma(-h)).mean()
    return loss.detach(), reward.detach(), torch.autograd.grad(loss, x)[0]


def exact(case, seed):
    return {"attention": _exact_attention, "policy": _exact_policy, "preference": _exact_preference}[case["kind"]](case, seed)
