"""Timed cases: the operators that serve drafted tokens over a key/value cache.

Every case is a dict of plain values with a ``kind``; the kinds and what they stand for:

    cache     rows of new tokens written into a layer's cache, and the whole prefix read back as dense bf16 rows
              (``ops.cache.KVCache.append`` and ``.read``): one layer of a prompt that is processed in chunks
    attend    attention of T drafted tokens per sequence over the cache (``ops.draft.draft_attention``): one layer of a
              step; T = 1 is plain decoding
    keep      the rows of the accepted branch moved to their places in every layer (``ops.cache.CacheGroup.keep``)
    logits    penalties, biases and a grammar mask on logits, and the token chosen from them
              (``ops.logits.constrain_logits``): the end of a step

``draw`` gives further cases of the same ranges, ragged and odd sizes among them.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
BF16 = torch.bfloat16


def listed():
    return [
        # A short chunk of one sequence in a layer of the decoder (2 KV heads of 256): launches count.
        dict(name="cache_chunk_short", kind="cache", B=1, T=64, Hkv=2, hd=256, max_seq=1024, pos_lo=512, pos_hi=512, bits=8),
        # The second half of the decoder's prompts, a batch of 8 with ragged lengths.
        dict(name="cache_chunk_batch", kind="cache", B=8, T=511, Hkv=2, hd=256, max_seq=1024, pos_lo=200, pos_hi=513, bits=8),
        # A long context's last chunk in a layer with 8 KV heads of 128.
        dict(name="cache_chunk_long", kind="cache", B=4, T=4096, Hkv=8, hd=128, max_seq=32768, pos_lo=20000, pos_hi=28672, bits=8),
        # One token per sequence in a global layer of the decoder: a batch of 8, latency.
        dict(name="attend_step_short", kind="attend", B=8, T=1, H=8, Hkv=2, hd=256, max_seq=1024, pos_lo=512, pos_hi=767, window=0, bits=8, tree="chain"),
        # One token per sequence over long ragged contexts, 4 query heads per KV head: the cache's bytes count.
        dict(name="attend_step_long", kind="attend", B=16, T=1, H=32, Hkv=8, hd=128, max_seq=32768, pos_lo=4000, pos_hi=32767, window=0, bits=8, tree="chain"),
        # A tree of 16 drafts in a sliding-window layer of the decoder, bf16 cache.
        dict(name="attend_tree_window", kind="attend", B=8, T=16, H=8, Hkv=2, hd=256, max_seq=1024, pos_lo=500, pos_hi=1008, window=512, bits=16, tree="random"),
        # Odd everything: 33 drafts, heads of 64, 3 query heads per KV head, three sequences.
        dict(name="attend_tree_odd", kind="attend", B=3, T=33, H=12, Hkv=4, hd=64, max_seq=1300, pos_lo=1, pos_hi=1111, window=0, bits=16, tree="random"),
        # The widest tree over long contexts: 256 query rows per KV head share every key.
        dict(name="attend_tree_long", kind="attend", B=4, T=64, H=8, Hkv=2, hd=256, max_seq=32768, pos_lo=20001, pos_hi=32704, window=0, bits=8, tree="random"),
        # The accepted branch in all 30 layers of the decoder, a batch of 8 with 16 drafts each, bf16 caches.
        dict(name="keep_decoder", kind="keep", layers=30, B=8, T=16, most=6, Hkv=2, hd=256, max_seq=1024, pos_lo=300, pos_hi=1000, bits=16),
        # Wide trees in one layer of a large batch, 8-bit rows, and the kept rows read back.
        dict(name="keep_wide", kind="keep", layers=1, B=64, T=64, most=20, Hkv=8, hd=128, max_seq=2048, pos_lo=1, pos_hi=1984, bits=8),
        # One sequence over the trainer's vocabulary: penalties and the chosen token only.
        dict(name="logits_one", kind="logits", rows=1, vocab=50304, hist=1000, prompt=512, nbias=5, mask=False, out=False, half=False),
        # Eight sequences with 16 drafted positions each over the decoder's vocabulary, with a grammar, processed logits kept.
        dict(name="logits_drafts", kind="logits", rows=128, vocab=262144, hist=2048, prompt=512, nbias=300, mask=True, out=True, half=False),
    ]


def _log_int(rng, lo, hi, step=1):
    """An integer of lo..hi, a multiple of ``step``, spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["cache", "attend", "attend", "attend", "keep", "logits"])
    hd = rng.choice([64, 128, 256])
    Hkv = rng.choice([1, 2, 4, 8])
    bits = rng.choice([8, 8, 16])
    if kind == "cache":
        B, T = _log_int(rng, 1, 16), _log_int(rng, 1, 2048)
        max_seq = _log_int(rng, T + 1, 8192)
        hi = rng.randint(0, max_seq - T)
        return dict(kind=kind, B=B, T=T, Hkv=Hkv, hd=hd, max_seq=max_seq, pos_lo=rng.randint(0, hi), pos_hi=hi, bits=bits)
    if kind == "attend":
        B, T = _log_int(rng, 1, 16), rng.choice([1, 1, _log_int(rng, 2, 64)])
        G = rng.choice([1, 2, 3, 4, 5, 8])
        max_seq = _log_int(rng, T + 1, 16384)
        hi = rng.randint(0, max_seq - T)
        return dict(kind=kind, B=B, T=T, H=G * Hkv, Hkv=Hkv, hd=hd, max_seq=max_seq, pos_lo=rng.randint(0, hi), pos_hi=hi,
                    window=rng.choice([0, 0, max(T, _log_int(rng, 64, 2048))]), bits=bits, tree=rng.choice(["chain", "random", "random"]))
    if kind == "keep":
        B, T = _log_int(rng, 1, 32), rng.randint(2, 64)
        max_seq = _log_int(rng, T + 1, 2048)
        hi = rng.randint(0, max_seq - T)
        return dict(kind=kind, layers=rng.randint(1, 30) if bits == 16 else 1, B=B, T=T, most=rng.randint(1, min(T, 20)), Hkv=Hkv, hd=hd,
                    max_seq=max_seq, pos_lo=rng.randint(0, hi), pos_hi=hi, bits=bits)
    hist = rng.choice([0, _log_int(rng, 1, 8192)])
    out = rng.random() < 0.5
    return dict(kind=kind, rows=_log_int(rng, 1, 128), vocab=_log_int(rng, 1000, 262144), hist=hist, prompt=rng.randint(0, hist),
                nbias=rng.choice([0, _log_int(rng, 1, 300)]), mask=rng.random() < 0.6, out=out, half=rng.random() < 0.4)


# ------------------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _spread(B, lo, hi, g=None):
    """B lengths spread evenly over lo..hi, in an order of their own."""
    v = [lo + (hi - lo) * i // max(1, B - 1) for i in range(B)] if B > 1 else [hi]
    t = torch.tensor(v, dtype=torch.int32, device=DEV)
    return t if g is None else t[torch.randperm(B, generator=g, device=DEV)].contiguous()


def _counts(B, T, g=None):
    """How many of T new tokens each sequence has: all, or down to three quarters."""
    return _spread(B, T - T // 4, T, g)


def _rows(shape, g, spread=True):
    """Keys or values as a model has them: normal, with a few channels that are larger."""
    x = torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)
    if spread:
        x *= 1 + 3 * (torch.rand(shape[-1], generator=g, device=DEV) < 0.03).float()
    return x.to(BF16)


def _quantise(x):
    """Codes and scales of rows."""
    f = x.float()
    a = f.abs().amax(-1, keepdim=True)
    c = torch.round(f * 127 / torch.where(a > 0, a, 1)).to(torch.int8)
    return c, (a / 127)[..., 0]


def _cache(B, Hkv, max_seq, hd, bits, g):
    """A layer's cache, full of rows: key, value, and their scales."""
    got = []
    for _ in range(2):
        if bits == 16:
            got.append((_rows((B, Hkv, max_seq, hd), g), None))
        else:
            c = torch.empty((B, Hkv, max_seq, hd), dtype=torch.int8, device=DEV)
            s = torch.empty((B, Hkv, max_seq), dtype=torch.float32, device=DEV)
            for b in range(B):
                c[b], s[b] = _quantise(_rows((Hkv, max_seq, hd), g))
            got.append((c, s))
    (k, ks), (v, vs) = got
    return dict(k=k, v=v, k_scale=ks, v_scale=vs)


def _tree(B, T, how, g):
    """visible [B, T]: bit j of a node's word says that it sees node j: itself and its ancestors."""
    r = torch.rand((B, T), generator=g, device=DEV).cpu().tolist()
    rows = []
    for b in range(B):
        bits = []
        for t in range(T):
            parent = t - 1 if how == "chain" else int(r[b][t] * t)      # every node before it is as likely
            bits.append((bits[parent] if t else 0) | (1 << t))
        rows.append([x - (1 << 64) if x >> 63 else x for x in bits])
    return torch.tensor(rows, dtype=torch.int64, device=DEV)


def _handle(st):
    from mesh_b200.ops.cache import KVCache
    return KVCache(st["k"], st["v"], st["k_scale"], st["v_scale"])


def prepare(case, seed):
    g = _gen(seed)
    c = case
    st = dict(c)
    if c["kind"] in ("cache", "attend", "keep"):
        B, T, Hkv, hd = c["B"], c["T"], c["Hkv"], c["hd"]
        st["pos"] = _spread(B, c["pos_lo"], c["pos_hi"], g)
    if c["kind"] == "cache":
        st |= _cache(B, Hkv, c["max_seq"], hd, c["bits"], g)
        # keys and values are columns of one fused projection, as a layer has them
        kv = torch.cat([_rows((B, T, Hkv * hd), g), _rows((B, T, Hkv * hd), g)], -1)
        st["new_k"], st["new_v"] = kv[..., :Hkv * hd].view(B, T, Hkv, hd), kv[..., Hkv * hd:].view(B, T, Hkv, hd)
        st["counts"] = _counts(B, T, g)
        st["start"] = torch.zeros_like(st["pos"])
        st["ends"] = st["pos"] + st["counts"]
        st["most"] = c["pos_hi"] + T
    elif c["kind"] == "attend":
        st |= _cache(B, Hkv, c["max_seq"], hd, c["bits"], g)
        st["q"] = (torch.randn((B, T, c["H"], hd), generator=g, device=DEV) * 1.5).to(BF16)
        st["counts"] = _counts(B, T, g)
        st["visible"] = _tree(B, T, c["tree"], g) if T > 1 else None
        st["out"] = torch.zeros((B, T, c["H"], hd), dtype=BF16, device=DEV)
    elif c["kind"] == "keep":
        st["layers_"] = [_cache(B, Hkv, c["max_seq"], hd, c["bits"], g) for _ in range(c["layers"])]
        # the root and its first children may lie where they are kept; the others come from behind the kept ones, so that
        # a second pass finds the rows as the first one left them
        n, T = c["most"], c["T"]
        stay = torch.randint(0, n + 1, (B,), generator=g, device=DEV).tolist()
        rows = []
        for b in range(B):
            order = (torch.randperm(T - n, generator=g, device=DEV) + n).tolist() if T > n else []
            k = max(stay[b], n - len(order))
            rows.append(list(range(k)) + sorted(order[:n - k]))
        st["path"] = torch.tensor(rows, dtype=torch.int32, device=DEV)
        st["counts"] = _spread(B, 1, n, g)
    else:
        R, V, Hn = c["rows"], c["vocab"], c["hist"]
        st["logits"] = (torch.randn((R, V), generator=g, device=DEV) * 3).to(BF16 if c["half"] else torch.float32)
        # a text repeats itself: half of the history is drawn from few tokens
        few = torch.randint(0, V, (R, max(1, Hn // 8)), generator=g, device=DEV)
        near = few.gather(1, torch.randint(0, few.shape[1], (R, Hn), generator=g, device=DEV))
        far = torch.randint(0, V, (R, Hn), generator=g, device=DEV)
        st["history"] = torch.where(torch.rand((R, Hn), generator=g, device=DEV) < 0.5, near, far).to(torch.int32)
        st["history_len"] = _spread(R, Hn - Hn // 3, Hn, g)
        st["prompt_len"] = torch.minimum(_spread(R, c["prompt"] // 2, c["prompt"], g), st["history_len"])
        st["repetition"] = 1 + 0.3 * torch.rand(R, generator=g, device=DEV)
        st["presence"] = 0.5 * torch.rand(R, generator=g, device=DEV)
        st["frequency"] = 0.5 * torch.rand(R, generator=g, device=DEV)
        st["bias_ids"] = torch.stack([torch.randperm(V, generator=g, device=DEV)[:c["nbias"]] for _ in range(R)]).to(torch.int32)
        st["bias"] = torch.randn((R, c["nbias"]), generator=g, device=DEV) * 5
        st["allowed"] = None
        if c["mask"]:       # a grammar allows one token in eight, in runs of neighbours
            w = torch.randint(-2**31, 2**31, (R, (V + 31) // 32, 2), generator=g, device=DEV).to(torch.int32)
            st["allowed"] = (w[..., 0] & w[..., 1] & (torch.rand(w.shape[:2], generator=g, device=DEV) < 0.5).to(torch.int32).neg()).contiguous()
        st["out"] = torch.empty_like(st["logits"]) if c["out"] else None
        st["tokens"] = torch.zeros(R, dtype=torch.int32, device=DEV)
    if own:                 # the handles that a serving program keeps beside its caches
        if c["kind"] in ("cache", "attend"):
            st["handle"] = _handle(st)
        elif c["kind"] == "keep":
            from mesh_b200.ops.cache import CacheGroup
            st["handles"] = [_handle(x) for x in st["layers_"]]
            st["group"] = CacheGroup(st["handles"])
    return st


# ------------------------------------------------------------------------------------------------------- one pass
def run(st):
    kind = st["kind"]
    if own:
        if kind == "cache":
            c = st["handle"]
            c.append(st["new_k"], st["new_v"], st["pos"], st["counts"])
            return c.read(st["start"], st["most"], st["ends"])
        if kind == "attend":
            from mesh_b200.ops.draft import draft_attention
            return draft_attention(st["q"], st["handle"], st["pos"], counts=st["counts"], visible=st["visible"], window=st["window"], out=st["out"])
        if kind == "keep":
            st["group"].keep(st["pos"], st["path"], st["counts"])
            if st["bits"] == 16:
                return [(x["k"], x["v"]) for x in st["layers_"]]
            return [h.read(st["pos"], st["most"], st["counts"]) for h in st["handles"]]
        from mesh_b200.ops.logits import constrain_logits
        constrain_logits(st["logits"], history=st["history"], history_len=st["history_len"], prompt_len=st["prompt_len"],
                         repetition=st["repetition"], presence=st["presence"], frequency=st["frequency"], bias_ids=st["bias_ids"],
                         bias=st["bias"], allowed=st["allowed"], out=st["out"], tokens=st["tokens"])
        return st["out"], st["tokens"]
    if kind == "cache":
        _plain_append(st, st["new_k"], st["new_v"], st["pos"], st["counts"])
        return _plain_read(st, st["start"], st["most"], st["ends"])
    if kind == "attend":
        return _plain_attend(st)
    if kind == "keep":
        for x in st["layers_"]:
            _plain_keep(x, st["pos"], st["path"], st["counts"])
        if st["bits"] == 16:
            return [(x["k"], x["v"]) for x in st["layers_"]]
        return [_plain_read(x, st["pos"], st["most"], st["counts"]) for x in st["layers_"]]
    return _plain_logits(st)


def _plain_append(st, k, v, pos, counts):
    """Row t of sequence b to slot pos[b] + t, for t < counts[b]."""
    T = k.shape[1]
    t = torch.arange(T, device=DEV)
    b, t = torch.nonzero(t < counts[:, None], as_tuple=True)
    slot = pos.long()[b] + t
    for name, x in (("k", k), ("v", v)):
        x = x[b, t]
        if st["bits"] == 16:
            st[name][b, :, slot] = x
        else:
            f = x.float()
            a = f.abs().amax(-1, keepdim=True)
            st[name][b, :, slot] = torch.round(f * 127 / torch.where(a > 0, a, 1)).to(torch.int8)
            st[name + "_scale"][b, :, slot] = (a / 127)[..., 0]


def _plain_read(st, start, T, counts):
    """Rows start[b] .. start[b] + T of every sequence, zero behind counts[b]: [B, T, kv heads, hd]."""
    B, max_seq = st["k"].shape[0], st["k"].shape[2]
    t = torch.arange(T, device=DEV)
    slot = (start.long()[:, None] + t).clamp(max=max_seq - 1)
    b = torch.arange(B, device=DEV)[:, None]
    there = (t < counts[:, None])[..., None, None]
    got = []
    for name in ("k", "v"):
        x = st[name][b, :, slot].float()
        if st[name + "_scale"] is not None:
            x = x * st[name + "_scale"][b, :, slot][..., None]
        got.append(torch.where(there, x, 0).to(BF16))
    return tuple(got)


def _plain_attend(st):
    B, T, H, hd = st["q"].shape
    Hkv, S = st["k"].shape[1], st["k"].shape[2]
    k, v = st["k"].float(), st["v"].float()
    if st["k_scale"] is not None:
        k, v = k * st["k_scale"][..., None], v * st["v_scale"][..., None]
    q = st["q"].float().view(B, T, Hkv, H // Hkv, hd).permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, hd)
    s = (q @ k.transpose(-1, -2)).view(B, Hkv, T, H // Hkv, S) * hd ** -0.5
    slot, t = torch.arange(S, device=DEV), torch.arange(T, device=DEV)
    pos = st["pos"].long()[:, None, None]
    vis = st["visible"] if st["visible"] is not None else torch.ones((B, T), dtype=torch.int64, device=DEV)
    node = (vis[..., None] >> torch.arange(64, device=DEV)) & 1                      # [B, T, 64]
    sees = node.gather(2, (slot - pos).clamp(0, 63).expand(B, T, S)).bool()
    sees = sees & (slot >= pos) & (slot < pos + st["counts"].long()[:, None, None])
    past = slot < pos
    if st["window"] > 0:
        past = past & (slot > pos + node.sum(-1, keepdim=True).clamp(min=1) - 1 - st["window"])
    s = torch.where((sees | past)[:, None, :, None], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m > -math.inf, m, 0))
    l = p.sum(-1, keepdim=True)
    o = (p.reshape(B, Hkv, -1, S) @ v).view(B, Hkv, T, H // Hkv, hd) / torch.where(l > 0, l, 1)
    o = o.permute(0, 2, 1, 3, 4).reshape(B, T, H, hd).to(BF16)
    st["out"].copy_(torch.where((t < st["counts"][:, None])[..., None, None], o, st["out"]))
    return st["out"]


def _plain_keep(st, pos, path, counts):
    i = torch.arange(path.shape[1], device=DEV)
    b, i = torch.nonzero(i < counts[:, None], as_tuple=True)
    to = pos.long()[b] + i
    src = pos.long()[b] + path.long()[b, i]
    for name in ("k", "v", "k_scale", "v_scale"):
        if st[name] is not None:
            st[name][b, :, to] = st[name][b, :, src]


def _plain_logits(st):
    x = st["logits"].float()
    R, V = x.shape
    h = st["history"].long()
    i = torch.arange(h.shape[1], device=DEV)
    inside = i < st["history_len"][:, None]
    n_all = torch.zeros((R, V), device=DEV).scatter_add_(1, h, inside.float())
    n = torch.zeros((R, V), device=DEV).scatter_add_(1, h, (inside & (i >= st["prompt_len"][:, None])).float())
    r = st["repetition"][:, None]
    x = torch.where(n_all > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - st["frequency"][:, None] * n - torch.where(n > 0, st["presence"][:, None], 0)
    x = x.scatter_add(1, st["bias_ids"].long(), st["bias"])
    if st["allowed"] is not None:
        v = torch.arange(V, device=DEV)
        x = torch.where(((st["allowed"][:, v // 32] >> (v % 32)) & 1).bool(), x, -math.inf)
    top = x.argmax(-1)                                  # the lowest index of equal ones
    st["tokens"].copy_(torch.where(x.amax(-1) > -math.inf, top, -1))
    if st["out"] is not None:
        st["out"].copy_(x)
    return st["out"], st["tokens"]


# ------------------------------------------------------------------------------------------- what a pass cannot do without
def _ends(c, B, T, lo, hi):
    """Mean of pos and of counts over a batch, whatever the order."""
    pos = [lo + (hi - lo) * i // max(1, B - 1) for i in range(B)] if B > 1 else [hi]
    cnt = [T - T // 4 + (T // 4) * i // max(1, B - 1) for i in range(B)] if B > 1 else [T]
    return pos, cnt


def work(case):
    c = case
    if c["kind"] in ("cache", "attend", "keep"):
        row = c["hd"] + 4 if c["bits"] == 8 else 2 * c["hd"]            # bytes of one key or value in the cache
    if c["kind"] == "cache":
        pos, cnt = _ends(c, c["B"], c["T"], c["pos_lo"], c["pos_hi"])
        new, old = sum(cnt), sum(pos)
        dense = c["B"] * (c["pos_hi"] + c["T"])         # all rows of the result are written, zeros too
        return dict(bytes=2 * c["Hkv"] * (new * (2 * c["hd"] + row) + old * row + dense * 2 * c["hd"]), flops=6 * c["Hkv"] * c["hd"] * new)
    if c["kind"] == "attend":
        pos, cnt = _ends(c, c["B"], c["T"], c["pos_lo"], c["pos_hi"])
        seen = [min(p, c["window"]) if c["window"] else p for p in pos]
        n_q = sum(cnt) * c["H"]
        per = [(s + (n + 1) / 2) * n for s, n in zip(seen, cnt)]
        return dict(bytes=2 * c["Hkv"] * row * (sum(seen) + sum(cnt)) + n_q * c["hd"] * 4, flops=4 * c["H"] * c["hd"] * sum(per))
    if c["kind"] == "keep":
        moved = sum([1 + (c["most"] - 1) * i // max(1, c["B"] - 1) for i in range(c["B"])] if c["B"] > 1 else [c["most"]])
        n = 2 * c["layers"] * c["Hkv"] * moved * row * 2
        return dict(bytes=n + (2 * c["Hkv"] * c["B"] * c["most"] * c["hd"] * 2 if c["bits"] == 8 else 0), flops=0)
    size = 2 if c["half"] else 4
    n = c["rows"] * c["vocab"]
    return dict(bytes=n * size * (2 if c["out"] else 1) + (n // 8 if c["mask"] else 0) + c["rows"] * (4 * c["hist"] + 8 * c["nbias"]), flops=2 * n)


# ------------------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if st["kind"] == "cache":
        return _exact_cache(st)
    if st["kind"] == "attend":
        return _exact_attend(st)
    if st["kind"] == "keep":
        return _exact_keep(st)
    return _exact_logits(st)


def _stored(codes, scale):
    x = codes.double()
    return x if scale is None else x * scale.double().unsqueeze(-1)


def _exact_cache(st):
    B = st["B"]
    got = []
    for name, new in (("k", st["new_k"]), ("v", st["new_v"])):
        dense = torch.zeros((B, st["most"], st["Hkv"], st["hd"]), dtype=torch.float64, device=DEV)
        for b in range(B):
            p, n = int(st["pos"][b]), int(st["counts"][b])
            old = _stored(st[name][b, :, :p], None if st[name + "_scale"] is None else st[name + "_scale"][b, :, :p])
            x = new[b, :n].double()
            if st["bits"] == 8:
                a = x.abs().max(-1, keepdim=True).values
                x = torch.where(a > 0, torch.round(127 * x / a) * (a / 127), torch.zeros_like(x))
            dense[b, :p] = old.transpose(0, 1)
            dense[b, p:p + n] = x
        got.append(dense)
    return tuple(got)


def _exact_attend(st):
    q, out = st["q"].double(), st["out"].double().clone()
    B, T, H, hd = q.shape
    G = H // st["Hkv"]
    for b in range(B):
        p, n = int(st["pos"][b]), int(st["counts"][b])
        mask = torch.zeros((n, p + n), dtype=torch.bool)
        for t in range(n):
            word = int(st["visible"][b, t]) & ((1 << 64) - 1) if st["visible"] is not None else 1
            at = p + max(1, bin(word).count("1")) - 1
            lo = max(0, at - st["window"] + 1) if st["window"] else 0
            mask[t, min(lo, p):p] = True
            for j in range(n):
                mask[t, p + j] = bool(word >> j & 1)
        mask = mask.to(DEV)
        for h in range(H):
            kv = h // G
            k = _stored(st["k"][b, kv, :p + n], None if st["k_scale"] is None else st["k_scale"][b, kv, :p + n])
            v = _stored(st["v"][b, kv, :p + n], None if st["v_scale"] is None else st["v_scale"][b, kv, :p + n])
            s = (q[b, :n, h] @ k.t()) / math.sqrt(hd)
            s = s.masked_fill(~mask, -math.inf)
            out[b, :n, h] = torch.softmax(s, -1) @ v
    return out


def _exact_keep(st):
    got = []
    for x in st["layers_"]:
        one = []
        for name in ("k", "v"):
            now = _stored(x[name], x[name + "_scale"])
            new = now.clone()
            for b in range(st["B"]):
                p, n = int(st["pos"][b]), int(st["counts"][b])
                new[b, :, p:p + n] = now[b][:, p + st["path"][b, :n].long()]
            if st["bits"] == 8:
                back = torch.zeros((st["B"], st["most"], st["Hkv"], st["hd"]), dtype=torch.float64, device=DEV)
                for b in range(st["B"]):
                    p, n = int(st["pos"][b]), int(st["counts"][b])
                    back[b, :n] = new[b, :, p:p + n].transpose(0, 1)
                new = back
            one.append(new if st["bits"] == 8 else new.to(BF16))       # moved rows are what they were, to the bit
        got.append(tuple(one))
    return got


def _exact_logits(st):
    rows, tokens = [], []
    for r in range(st["rows"]):
        x = st["logits"][r].double()
        h = st["history"][r, :int(st["history_len"][r])].long()
        rep = st["repetition"][r].double()
        seen = torch.unique(h)
        x[seen] = torch.where(x[seen] > 0, x[seen] / rep, x[seen] * rep)
        made, times = torch.unique(h[int(st["prompt_len"][r]):], return_counts=True)
        x[made] -= st["frequency"][r].double() * times + st["presence"][r].double()
        x[st["bias_ids"][r].long()] += st["bias"][r].double()
        if st["allowed"] is not None:
            bits = (st["allowed"][r].unsqueeze(-1) >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
            x[bits.flatten()[:st["vocab"]] == 0] = -math.inf
        tokens.append(int(x.argmax()) if float(x.max()) > -math.inf else -1)
        rows.append(x)
    out = torch.stack(rows)
    return (out if st["out"] is not None else None), torch.tensor(tokens, dtype=torch.int32, device=DEV)
