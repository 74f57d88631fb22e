"""The operators for generating text with drafted tokens: what is measured, on which inputs, in plain form and by the framework.

Four groups: a cache of keys and values that is quantised as it is written, and read back; attention of new tokens (one, a run of
them, or a tree of drafted ones) over that cache; the drafted tokens' verification against the target's logits from given random
numbers; and the move of an accepted path's keys and values to the end of the sequence.
``run`` computes the plain form in elementary torch operations, or, with ``own``, makes the framework's calls.
"""
import math

import numpy as np
import torch

own = False
DEV = "cuda"


def listed():
    return [
        # One new token for each of eight running sequences, one layer: only launches and host work count.
        dict(name="append_token", kind="write", cache="int8", source="bf16", layers=0, B=8, T=1, Hkv=5, D=128, L=2000, page=0, ragged=False),
        # Prompts of ragged lengths into the pages of a pool, and back for the layers that attend to them whole.
        dict(name="append_prompts", kind="write", cache="fp8", source="bf16", layers=0, B=16, T=4096, Hkv=8, D=128, L=4096, page=64, ragged=True),
        # A toy layer's single token (2 heads of 16): latency.
        dict(name="toy_decode", kind="attention", cache="bf16", B=1, N=1, H=2, Hkv=1, D=16, L=60, page=0, tree=False, ragged=False, left=-1,
             softcap=0.0, bias=False),
        # A batch of single tokens, sequences of every length up to 4096, pages of 64, the headline layer's heads.
        dict(name="decode_batch", kind="attention", cache="int8", B=64, N=1, H=10, Hkv=5, D=128, L=4096, page=64, tree=False, ragged=False,
             left=-1, softcap=0.0, bias=False),
        # One long conversation.
        dict(name="decode_long", kind="attention", cache="fp8", B=1, N=1, H=16, Hkv=8, D=128, L=131072, page=0, tree=False, ragged=False,
             left=-1, softcap=0.0, bias=False),
        # Trees of up to 32 drafted tokens over long sequences in pages.
        dict(name="tree_batch", kind="attention", cache="int8", B=16, N=32, H=16, Hkv=8, D=128, L=8192, page=64, tree=True, ragged=True,
             left=-1, softcap=0.0, bias=False),
        # A layer with a 512-key window, capped and biased scores (the training script's 8 heads of 64), an odd tree.
        dict(name="tree_window", kind="attention", cache="bf16", B=4, N=13, H=8, Hkv=8, D=64, L=2048, page=16, tree=True, ragged=False,
             left=512, softcap=30.0, bias=True),
        # A toy model's accepted path, all layers at once.
        dict(name="keep_small", kind="keep", cache="bf16", layers=4, B=2, N=5, Hkv=1, D=16, L=60, page=0),
        # The same for a batch and a model of 20 layers.
        dict(name="keep_batch", kind="keep", cache="int8", layers=20, B=32, N=32, Hkv=5, D=128, L=1024, page=64),
        # Three drafted tokens over a byte vocabulary: latency.
        dict(name="verify_small", kind="verify", dtype="fp32", B=1, N=4, V=259, tree=False, temperature=1.0, ragged=False),
        # A batch of runs of five drafted tokens with the drafts' distributions.
        dict(name="verify_batch", kind="verify", dtype="bf16", B=64, N=6, V=32768, tree=False, temperature=0.8, ragged=True),
        # Trees of candidates, an odd vocabulary, fp32 logits.
        dict(name="verify_trees", kind="verify", dtype="fp32", B=16, N=32, V=50257, tree=True, temperature=1.0, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["write", "attention", "keep", "verify"], [2, 6, 1, 4])[0]
    if kind == "verify":
        V = rng.choice([259, 8192, 32768, _log(rng, 50, 50257), 50257, 50304])
        tree, dtype = rng.choice([True, False]), rng.choice(["bf16", "fp32"])
        N = rng.choice([1, 2, 5, 8, 13, 16, 32]) if tree else rng.randint(1, 9)
        return dict(kind=kind, dtype=dtype, B=_log(rng, 1, max(1, min(128, 25_000_000 // (V * N)))), N=N, V=V, tree=tree,
                    temperature=rng.choice([0.0, 0.7, 1.0, 1.0, round(rng.uniform(0.3, 1.5), 2)]), ragged=rng.choice([True, False]))
    cache, page = rng.choice(["bf16", "int8", "fp8"]), rng.choice([0, 16, 64, 256])
    Hkv, D = rng.choice([1, 2, 4, 5, 8, 16]), rng.choices([16, 32, 48, 64, 80, 96, 112, 128], [1, 1, 1, 4, 1, 1, 1, 6])[0]
    if kind == "write":
        B = _log(rng, 1, 64)
        T = _log(rng, 1, max(1, min(8192, 25_000_000 // (B * Hkv * D))))
        return dict(kind=kind, cache=cache, source=rng.choice(["bf16", "bf16", "fp32"]), layers=0, B=B, T=T, Hkv=Hkv, D=D,
                    L=_log(rng, 1, 4096), page=page, ragged=rng.choice([True, False]))
    if kind == "keep":
        return dict(kind=kind, cache=cache, layers=rng.randint(1, 12), B=_log(rng, 1, 32), N=rng.randint(2, 32), Hkv=Hkv, D=D,
                    L=_log(rng, 1, 1024), page=page)
    H, N = Hkv * rng.choice([1, 1, 2, 2, 3, 4, 8]), rng.choices([1, 2, 4, 8, 13, 16, 31, 64], [8, 1, 1, 2, 1, 2, 1, 1])[0]
    B, L = _log(rng, 1, 64), _log(rng, 1, 131072)
    # no draw costs more than the largest above, in keys or in products
    while B > 1 and (B * L * Hkv * D > 1.3e8 or B * L * H * N * D > 8.0e9):
        B -= 1
    while B * L * Hkv * D > 1.3e8 or B * L * H * N * D > 8.0e9:
        L = L * 3 // 4
    return dict(kind=kind, cache=cache, B=B, N=N, H=H, Hkv=Hkv, D=D, L=L, page=page, tree=N > 1 and rng.choice([True, True, False]),
                ragged=rng.choice([True, False]), left=rng.choice([-1, -1, 128, 512, rng.randint(0, L)]),
                softcap=rng.choice([0.0, 0.0, 30.0, 50.0]), bias=rng.choice([False, False, True]))


# ---- inputs ---------------------------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _rows(g, cache, *shape):
    """Keys or values as a layer makes them, 1.2 times their root mean square, as the cache's type holds them: (codes, scales)."""
    x = (1.2 * torch.randn(*shape, device=DEV, generator=g)).bfloat16()
    return _quantised(x, cache)


def _quantised(x, cache):
    """(values in the cache's type, scales or None): a token's values of one head share a scale, the largest magnitude over 127 (int8)
    or 448 (fp8)."""
    if cache == "bf16":
        return x.to(torch.bfloat16), None
    top = 127.0 if cache == "int8" else 448.0
    x = x.float()
    most = x.abs().amax(-1, keepdim=True)
    y = x * (torch.full_like(most, top) / most)
    y = torch.round(y).clamp(-127, 127).to(torch.int8) if cache == "int8" else y.to(torch.float8_e4m3fn)
    return y, most[..., 0] / torch.full_like(most[..., 0], top)


def _lengths(case, seed):
    """How many tokens each sequence holds: the longest all of L, the others anything from an eighth of it."""
    rng = np.random.default_rng([int(seed), 81])
    n = rng.integers(max(1, case["L"] // 8) if case["L"] > 0 else 0, case["L"] + 1, case["B"])
    n[0] = case["L"]
    return n.astype(np.int32)


def _counts(case, seed, n):
    """How many of n new tokens a ragged batch's sequences have."""
    rng = np.random.default_rng([int(seed), 82])
    c = rng.integers((n + 1) // 2, n + 1, case["B"])
    c[0] = n
    return c.astype(np.int32)


def _parents(case, seed):
    """Trees of drafted tokens: node 0 is the last token, each other node's parent is one of the nodes before it, mostly an early one."""
    rng = np.random.default_rng([int(seed), 83])
    B, N = case["B"], case["N"]
    p = np.full((B, N), -1, np.int32)
    for i in range(1, N):
        p[:, i] = (i * rng.random(B) ** 1.5).astype(np.int32)
    return p


def _dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEV)


def _cache_inputs(case, seed, more):
    """The cache as a program has it after L tokens with room for `more`: buffers, and the pages' table where it has one."""
    g, B, Hkv, D, page = _gen(seed), case["B"], case["Hkv"], case["D"], case["page"]
    room = -(-(case["L"] + more) // 16) * 16
    S, M = (page, -(-room // page)) if page else (room, 1)
    lead = (case["layers"],) if case.get("layers") else ()
    k, ks = _rows(g, case["cache"], *lead, B * M, Hkv, S, D)
    v, vs = _rows(g, case["cache"], *lead, B * M, Hkv, S, D)
    order = np.random.default_rng([int(seed), 84]).permutation(B * M).astype(np.int32)
    return dict(k=k, v=v, ks=ks, vs=vs, pages=_dev(order.reshape(B, M)) if page else None, lengths=_dev(_lengths(case, seed)))


def _write_inputs(case, seed):
    s = _cache_inputs(case, seed, case["T"])
    g = _gen(int(seed) + (1 << 40))
    lead = (case["layers"],) if case["layers"] else ()
    dt = torch.bfloat16 if case["source"] == "bf16" else torch.float32
    K, V = ((1.2 * torch.randn(*lead, case["B"], case["T"], case["Hkv"], case["D"], device=DEV, generator=g)).to(dt) for _ in range(2))
    return dict(s, K=K, V=V, T=case["T"], counts=_dev(_counts(case, seed, case["T"])) if case["ragged"] else None)


def _attention_inputs(case, seed):
    s = _cache_inputs(case, seed, case["N"])
    H = case["H"]
    Q = (2.0 * torch.randn(case["B"], case["N"], H, case["D"], device=DEV, generator=_gen(int(seed) + (1 << 40)))).bfloat16()
    slopes = [2.0 ** (-8.0 * (h + 1) / H) for h in range(H)]
    return dict(s, Q=Q, window=(case["left"], 0), softcap=case["softcap"], parents=_dev(_parents(case, seed)) if case["tree"] else None,
                counts=_dev(_counts(case, seed, case["N"])) if case["ragged"] else None,
                slopes=torch.tensor(slopes, dtype=torch.float32, device=DEV) if case["bias"] else None)


def _keep_inputs(case, seed):
    s = _cache_inputs(case, seed, case["N"])
    rng = np.random.default_rng([int(seed), 85])
    B, N = case["B"], case["N"]
    kept = np.minimum(N, 1 + rng.geometric(0.3, B)).astype(np.int32)
    path = np.full((B, N), -1, np.int32)
    for b in range(B):
        path[b, :kept[b]] = np.concatenate([[0], 1 + np.sort(rng.choice(N - 1, kept[b] - 1, replace=False))])
    return dict(s, path=_dev(path), kept=_dev(kept), N=N)


def _verify_inputs(case, seed):
    """Logits of a standard deviation of 2.5, the drafter's near them; drafted tokens drawn from the drafter's distribution (runs) or
    its best ones (trees)."""
    g, B, N, V = _gen(seed), case["B"], case["N"], case["V"]
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    x = (2.5 * torch.randn(B, N, V, device=DEV, generator=g)).to(dt)
    T, u = case["temperature"], torch.rand(B, N, device=DEV, generator=g)
    tokens = torch.randint(0, V, (B, N), device=DEV, generator=g)
    s = dict(logits=x, uniforms=u, temperature=T, counts=_dev(_counts(case, seed, N)) if case["ragged"] else None, draft=None, parents=None)
    if case["tree"]:
        p = _parents(case, seed)
        s["parents"] = _dev(p)
        best = torch.stack([(x[b].float() + 0.7 * torch.randn(N, V, device=DEV, generator=g)).topk(min(N, V), -1).indices for b in range(B)])
        rank = (p[:, :, None] == p[:, None, :]) & np.tri(N, N, -1, bool)  # how many siblings come first
        at = _dev(p.astype(np.int64)).clamp(min=0), _dev(rank.sum(-1)).clamp(max=min(N, V) - 1)
        tokens[:, 1:] = best[torch.arange(B, device=DEV)[:, None], at[0], at[1]][:, 1:]
    elif N > 1:
        d = (x[:, :-1].float() + 0.8 * torch.randn(B, N - 1, V, device=DEV, generator=g)).to(dt)
        s["draft"] = d
        if T > 0:
            noise = torch.rand(d.shape, device=DEV, generator=g).clamp_(1e-10, 1.0 - 1e-7)
            tokens[:, 1:] = (d.float() / T - torch.log(-torch.log(noise))).argmax(-1)
        else:
            tokens[:, 1:] = d.float().argmax(-1)
    return dict(s, tokens=tokens)


_INPUTS = {"write": _write_inputs, "attention": _attention_inputs, "keep": _keep_inputs, "verify": _verify_inputs}


def prepare(case, seed):
    return dict(_INPUTS[case["kind"]](case, seed), kind=case["kind"], cache=case.get("cache"))


# ---- the framework's calls ------------------------------------------------------------------------------------------


def _own(s):
    import femtochat_amd as F

    if s["kind"] == "verify":
        return F.verify_drafts(s["logits"], s["tokens"], s["uniforms"], draft_logits=s["draft"], parents=s["parents"], counts=s["counts"],
                               temperature=s["temperature"])
    cache = F.KVCache(s["k"], s["v"], s["ks"], s["vs"], s["pages"])
    if s["kind"] == "write":
        F.cache_write_(cache, s["K"], s["V"], s["lengths"], s["counts"])
        return F.cache_read(cache, s["lengths"], s["T"], s["counts"])
    if s["kind"] == "keep":
        F.cache_keep_(cache, s["lengths"], s["path"], s["kept"])
        return F.cache_read(cache, s["lengths"], s["N"], s["kept"])
    return F.cached_attention(s["Q"], cache, s["lengths"], s["window"], counts=s["counts"], parents=s["parents"], softcap=s["softcap"],
                              slopes=s["slopes"])


# ---- the plain forms ------------------------------------------------------------------------------------------------


def _slots(s, positions):
    """(page, place in it) of positions (B, T)."""
    S = s["k"].shape[-2]
    if s["pages"] is None:
        return torch.arange(positions.shape[0], device=DEV)[:, None].expand_as(positions), positions
    return s["pages"].gather(1, positions // S).long(), positions % S


def _bits(x):
    """What indexing takes of any type."""
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


def _plain_read(s, positions, valid, dtype=torch.bfloat16):
    """The values at positions (B, T) as (..., B, T, Hkv, D), zeros where not valid."""
    page, at = _slots(s, torch.where(valid, positions, 0))
    pick = lambda x: x[page, :, at] if s["k"].dim() == 4 else x.transpose(0, 1)[page, :, :, at].movedim(2, 0)  # noqa: E731
    out = []
    for x, scale in ((s["k"], s["ks"]), (s["v"], s["vs"])):
        y = pick(_bits(x)).contiguous().view(x.dtype).float()
        if scale is not None:
            y = y * pick(scale)[..., None]
        out.append(torch.where(valid[..., None, None], y, 0.0).to(dtype))
    return tuple(out)


def _plain_write(s):
    lengths, T = s["lengths"].long(), s["T"]
    t = torch.arange(T, device=DEV)
    n = torch.full_like(lengths, T) if s["counts"] is None else s["counts"].long()
    valid, positions = t < n[:, None], lengths[:, None] + t
    page, at = _slots(s, positions)
    b, i = torch.nonzero(valid, as_tuple=True)
    for into, scale, x in ((s["k"], s["ks"], s["K"]), (s["v"], s["vs"], s["V"])):
        y, ys = _quantised(x, s["cache"])
        _bits(into)[page[b, i], :, at[b, i]] = _bits(y)[b, i]
        if scale is not None:
            scale[page[b, i], :, at[b, i]] = ys[b, i]
    return _plain_read(s, positions, valid)


def _plain_keep(s):
    lengths, kept, N = s["lengths"].long(), s["kept"].long(), s["N"]
    t = torch.arange(N, device=DEV)
    valid = t < kept[:, None]
    b, i = torch.nonzero(valid, as_tuple=True)
    src, dst = lengths[:, None] + torch.where(valid, s["path"].long(), 0), lengths[:, None] + t
    (sp, sa), (dp, da) = _slots(s, src), _slots(s, dst)
    for x in (s["k"], s["v"], s["ks"], s["vs"]):
        if x is not None:
            y = _bits(x).transpose(0, 1)  # pages first
            y[dp[b, i], :, :, da[b, i]] = y[sp[b, i], :, :, sa[b, i]]
    return _plain_read(s, dst, valid)


def _ancestors(parents, counts, B, N):
    """(B, N, N): whether node j is node i or one of its ancestors; (B, N): depths; (B, N): whether there is a node i."""
    i = torch.arange(N, device=DEV)
    there = (i < (N if counts is None else counts[:, None])).expand(B, N)
    if parents is None:
        return (i[:, None] >= i[None, :]).expand(B, N, N), i.expand(B, N), there
    A = (parents[:, :, None] == i).float() + torch.eye(N, device=DEV)
    for _ in range(max(1, (N - 1).bit_length())):
        A = torch.matmul(A, A).clamp(max=1.0)
    return A > 0, (A > 0).sum(-1) - 1, there


def _plain_attention(s):
    Q, lengths = s["Q"], s["lengths"].long()
    B, N, H, D = Q.shape
    room = s["k"].shape[-2] * (1 if s["pages"] is None else s["pages"].shape[1])
    key = torch.arange(room, device=DEV)
    anc, depth, there = _ancestors(s["parents"], s["counts"], B, N)
    K, V = _plain_read(s, key.expand(B, room), key < lengths[:, None] + N, torch.float32)
    K, V = K.transpose(1, 2).contiguous(), V.transpose(1, 2).contiguous()  # (B, Hkv, room, D)
    Hkv, G = K.shape[1], H // K.shape[1]
    q = Q.float().view(B, N, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * N, D)
    S = torch.matmul(q, K.transpose(-1, -2).contiguous()).view(B, Hkv, G, N, room) * (1.0 / math.sqrt(D))
    if s["softcap"] > 0:
        S = s["softcap"] * torch.tanh(S / s["softcap"])
    node = key - lengths[:, None]  # (B, room): the node in a place, if one is there
    new = (node >= 0) & (node < N)
    at = node.clamp(0, N - 1)
    place = torch.where(new, lengths[:, None] + depth.gather(1, at), key)  # positions of the keys in the text
    distance = lengths[:, None, None] + depth[:, :, None] - place[:, None, :]  # (B, N, room)
    seen = torch.where(new[:, None, :], anc.gather(2, at[:, None, :].expand(B, N, room)), (node < 0)[:, None, :])
    seen = seen & there[:, :, None]
    if s["window"][0] >= 0:
        seen = seen & (distance <= s["window"][0])
    if s["slopes"] is not None:
        S = S - s["slopes"].view(1, Hkv, G, 1, 1) * distance[:, None, None].float()
    S = S.masked_fill(~seen[:, None, None], -math.inf)
    m = S.amax(-1, keepdim=True)
    P = torch.exp(S - torch.where(torch.isinf(m), 0.0, m))
    l = P.sum(-1, keepdim=True)
    O = torch.matmul((P / torch.where(l > 0, l, 1.0)).view(B, Hkv, G * N, room), V)
    return O.view(B, Hkv, G, N, D).permute(0, 3, 1, 2, 4).reshape(B, N, H, D).to(Q.dtype)


def _plain_verify(s):
    """In 64 bits: a random number next to an acceptance's border, or to one of a vocabulary's many, needs them."""
    x, tokens, u, T = s["logits"].double(), s["tokens"], s["uniforms"].double(), s["temperature"]
    B, N, V = x.shape
    b, i = torch.arange(B, device=DEV), torch.arange(N, device=DEV)
    n = torch.full_like(b, N) if s["counts"] is None else s["counts"].long()
    there = i < n[:, None]
    anc, depth, _ = _ancestors(s["parents"], None, B, N)
    parents = (i - 1).expand(B, N) if s["parents"] is None else s["parents"].long()
    up = parents.clamp(min=0)
    sibling = (parents[:, :, None] == parents[:, None, :]) & (i[:, None] > i[None, :]) & (i[None, :] > 0)  # j comes before i
    best = torch.where(x == x.amax(-1, keepdim=True), torch.arange(V, device=DEV), V).amin(-1)  # the lowest of the largest
    if T > 0:
        p = torch.softmax(x / T, -1)
        own_p = p[b[:, None], up, tokens]
        if s["draft"] is not None:
            q = torch.softmax(s["draft"].double() / T, -1)
            own_q = torch.cat([torch.ones_like(u[:, :1]), q.gather(-1, tokens[:, 1:, None])[..., 0]], 1)
            test = u * own_q < own_p
        else:
            again = (sibling & (tokens[:, :, None] == tokens[:, None, :])).any(-1)
            left = 1.0 - (sibling & ~again[:, None, :]).double().matmul(own_p[..., None])[..., 0]
            test = (u * left < own_p) & ~again
    else:
        test = tokens == best.gather(1, up)
    chosen = test & there & ~(sibling & (test & there)[:, None, :]).any(-1)
    chosen[:, 0] = True
    reached = (chosen[:, None, :] | ~anc).all(-1) & anc[:, :, 0] & there
    kept = reached.sum(-1)
    path = torch.where(i < kept[:, None], torch.where(reached, i, N).sort(-1).values, -1)
    last = torch.where(reached, i, 0).amax(-1)
    if T > 0:
        w = p[b, last]
        if s["draft"] is not None:
            w = torch.where((last + 1 < n)[:, None], (w - q[b, last.clamp(max=N - 2)]).clamp(min=0.0), w)
        elif N > 1:
            tried = (parents == last[:, None]) & there & (i > 0)
            w = w * (1.0 - torch.zeros_like(w).scatter_reduce(1, tokens, tried.double(), "amax"))
        w = torch.where(w.sum(-1, keepdim=True) > 0, w, p[b, last])
        c = w.cumsum(-1)
        token = (c <= u[:, :1] * c[:, -1:]).sum(-1)
    else:
        token = best[b, last]
    return path.int(), kept.int(), torch.where(n > 0, token, -1).int()


def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return {"write": _plain_write, "attention": _plain_attention, "keep": _plain_keep, "verify": _plain_verify}[s["kind"]](s)


# ---- what each path cannot do without -------------------------------------------------------------------------------


def work(case):
    """Lengths and trees of one seed stand for all."""
    kind = case["kind"]
    if kind == "verify":
        size = 2 if case["dtype"] == "bf16" else 4
        rows = case["B"] * (case["N"] + (0 if case["tree"] else case["N"] - 1))
        return dict(bytes=rows * case["V"] * size, flops=4 * rows * case["V"])
    D, size = case["D"], 2 if case["cache"] == "bf16" else 1
    token = 2 * case["Hkv"] * (D * size + (0 if case["cache"] == "bf16" else 4))  # bytes of a token's keys and values
    values = 4 * case["Hkv"] * D  # the same in bf16
    given = values * (2 if case.get("source") == "fp32" else 1)
    if kind == "write":  # read and written; read again and written out
        tokens = int(_counts(case, 0, case["T"]).sum()) if case["ragged"] else case["B"] * case["T"]
        return dict(bytes=tokens * (given + 2 * token) + case["B"] * case["T"] * values, flops=4 * tokens * case["Hkv"] * D)
    if kind == "keep":
        kept = int(_keep_counts(case).sum())
        return dict(bytes=case["layers"] * (kept * 3 * token + case["B"] * case["N"] * values), flops=case["layers"] * kept * case["Hkv"] * D)
    n, new = _lengths(case, 0).astype(np.int64), _counts(case, 0, case["N"]) if case["ragged"] else np.full(case["B"], case["N"])
    keys = n if case["left"] < 0 else np.minimum(n, case["left"])
    pairs = int((keys * new).sum())
    return dict(bytes=int((keys + new).sum()) * token + 4 * case["B"] * case["N"] * case["H"] * D, flops=4 * D * case["H"] * pairs)


def _keep_counts(case):
    rng = np.random.default_rng([0, 85])
    return np.minimum(case["N"], 1 + rng.geometric(0.3, case["B"]))


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------


def _held(s, layer=None):
    """The cache's values as (pages, Hkv, page, D) in 64 bits."""
    out = []
    for x, scale in ((s["k"], s["ks"]), (s["v"], s["vs"])):
        x = (x if layer is None else x[layer]).double()
        out.append(x if scale is None else x * (scale if layer is None else scale[layer]).double()[..., None])
    return out


def _places(s, b, lo, hi):
    """Row numbers of sequence b's tokens lo to hi in the cache's (page, place) order."""
    S, t = s["k"].shape[-2], torch.arange(lo, hi, device=DEV)
    return (b * S + t) if s["pages"] is None else s["pages"][b].long()[t // S] * S + t % S


def _exact_write(case, seed):
    s = _write_inputs(case, seed)
    top = {"int8": 127.0, "fp8": 448.0}.get(case["cache"])
    out = []
    for x in (s["K"], s["V"]):
        x = x.double()
        if top is None:
            y = x.bfloat16().double()
        else:
            step = x.abs().amax(-1, keepdim=True) / top
            y = x / step
            y = (y.round() if case["cache"] == "int8" else y.float().to(torch.float8_e4m3fn).double()) * step
        if s["counts"] is not None:
            y = y * (torch.arange(s["T"], device=DEV) < s["counts"][:, None]).double()[..., None, None]
        out.append(y)
    return tuple(out)


def _exact_keep(case, seed):
    s = _keep_inputs(case, seed)
    B, N, path, kept = case["B"], case["N"], s["path"].tolist(), s["kept"].tolist()
    n = s["lengths"].tolist()
    out = [torch.zeros(case["layers"], B, N, case["Hkv"], case["D"], dtype=torch.float64, device=DEV) for _ in range(2)]
    for layer in range(case["layers"]):
        for x, to in zip(_held(s, layer), out):
            rows = x.transpose(1, 2).reshape(-1, case["Hkv"], case["D"])
            for b in range(B):
                at = _places(s, b, n[b], n[b] + N)
                to[layer, b, :kept[b]] = rows[at[torch.tensor(path[b][:kept[b]], device=DEV)]]
    return tuple(out)


def _exact_attention(case, seed):
    s = _attention_inputs(case, seed)
    B, N, H, D, Hkv = (case[k] for k in ("B", "N", "H", "D", "Hkv"))
    G, c, n = H // Hkv, case["softcap"], s["lengths"].tolist()
    new = [N] * B if s["counts"] is None else s["counts"].tolist()
    O = torch.zeros(B, N, H, D, dtype=torch.float64, device=DEV)
    Kd, Vd = _held(s)
    for b in range(B):
        at = _places(s, b, 0, n[b] + new[b])
        page, place = at // Kd.shape[2], at % Kd.shape[2]
        up = list(range(-1, N - 1)) if s["parents"] is None else s["parents"][b].tolist()
        text = torch.arange(n[b] + new[b], device=DEV)  # where in the text each key is
        hidden = torch.ones(new[b], n[b] + new[b], dtype=torch.bool, device=DEV)
        depths = []
        for i in range(new[b]):
            line, j = [], i
            while j >= 0:
                line.append(n[b] + j)
                j = up[j]
            depths.append(n[b] + len(line) - 1)
            hidden[i, :n[b]] = False
            hidden[i, torch.tensor(line, device=DEV)] = False
        text[n[b]:] = torch.tensor(depths, device=DEV)
        far = (torch.tensor(depths, device=DEV)[:, None] - text).double()
        if case["left"] >= 0:
            hidden |= far > case["left"]
        for h in range(H):
            k, v = Kd[page, h // G, place], Vd[page, h // G, place]
            z = s["Q"][b, :new[b], h].double() @ k.T / math.sqrt(D)
            if c > 0:
                z = c * torch.tanh(z / c)
            if s["slopes"] is not None:
                z = z - float(s["slopes"][h]) * far
            O[b, :new[b], h] = torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ v
    return O


def _exact_verify(case, seed):
    """A walk from node to node: the children of a node in order, each against what the ones before it have left of the target."""
    s = _verify_inputs(case, seed)
    B, N, T = case["B"], case["N"], case["temperature"]
    tokens, u = s["tokens"].tolist(), s["uniforms"].double().tolist()
    path, kept, token = torch.full((B, N), -1, dtype=torch.int32), torch.zeros(B, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        n = N if s["counts"] is None else int(s["counts"][b])
        up = list(range(-1, N - 1)) if s["parents"] is None else s["parents"][b].tolist()
        at, walk, moved = 0, [0], True
        while moved:
            moved, x = False, s["logits"][b, at].double()
            if T == 0:
                w = (torch.arange(case["V"], device=DEV) == torch.nonzero(x == x.max())[0]).double()
            else:
                w = torch.exp(torch.log_softmax(x / T, -1))
            for i in range(1, n):
                if up[i] != at:
                    continue
                y = tokens[b][i]
                if s["draft"] is not None and T > 0:
                    d = torch.exp(torch.log_softmax(s["draft"][b, i - 1].double() / T, -1))
                    moved = u[b][i] * float(d[y]) < float(w[y])
                    rest = (w - d).clamp(min=0.0)
                else:
                    moved = float(w[y]) > (u[b][i] * float(w.sum()) if T > 0 else 0.5)
                    rest = w.clone()
                    rest[y] = 0.0 if T > 0 else rest[y]
                if moved:
                    at = i
                    walk.append(i)
                    break
                w = rest if float(rest.sum()) > 0 else w
        c = w.cumsum(0)
        path[b, :len(walk)], kept[b] = torch.tensor(walk, dtype=torch.int32), len(walk)
        token[b] = int(torch.nonzero(c > u[b][0] * c[-1])[0])
    return path, kept, token


def exact(case, seed):
    return {"write": _exact_write, "keep": _exact_keep, "attention": _exact_attention, "verify": _exact_verify}[case["kind"]](case, seed)
