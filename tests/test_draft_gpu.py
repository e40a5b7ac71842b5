"""Operators for drafted tokens against plain statements in 64 bits: cache rows, attention of a tree, the kept branch, constraints
on logits, and a run of them together."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F64 = torch.bfloat16, torch.float64
DEV = "cuda"


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _same(a, b):
    return torch.equal(a, b)


def _randn(*shape, g, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(BF16)


def _encode(x):
    """Codes and scales of rows from the definition, in 64 bits."""
    f = x.double()
    a = f.abs().amax(-1, keepdim=True)
    code = torch.where(a > 0, torch.round(127 * f / torch.where(a > 0, a, 1)), 0)
    bad = ~torch.isfinite(a)
    return torch.where(bad, 0, code).to(torch.int8), torch.where(bad, math.nan, a / 127).float()[..., 0]


def _cache(B, H, S, hd, bits, g, scale=1.0):
    from mesh_b200.ops.cache import KVCache
    rows = [_randn(B, H, S, hd, g=g, scale=scale) for _ in range(2)]
    if bits == 16:
        return KVCache(*rows)
    (k, ks), (v, vs) = map(_encode, rows)
    return KVCache(k, v, ks, vs)


# ------------------------------------------------------------------------------------------------------------ rows
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("B,T,H", [(1, 1, 1), (3, 7, 3), (2, 33, 8)])
def test_append_and_read(hd, bits, B, T, H):
    g = _gen(B * T + hd)
    S = 50
    c = _cache(B, H, S, hd, bits, g)
    was = [x.clone() for x in (c.k, c.v) + ((c.k_scale, c.v_scale) if bits == 8 else ())]
    fused = _randn(B, T, 3 * H * hd, g=g)                      # keys and values are columns of a wider matrix
    k, v = fused[..., H * hd:2 * H * hd].view(B, T, H, hd), fused[..., 2 * H * hd:].view(B, T, H, hd)
    pos = _i32([5, 30, 17][:B])                                # the second sequence's rows run past the end when T = 33
    counts = _i32([T, max(0, T - 2), 0][:B])
    c.append(k, v, pos, counts)
    for name, x, old in zip("kv", (k, v), was):
        new = getattr(c, name)
        ref, ref_scale = old.clone(), None if bits == 16 else was[2 + "kv".index(name)].clone()
        for b in range(B):
            p, n = int(pos[b]), min(int(counts[b]), S - int(pos[b]))
            rows = x[b, :n].transpose(0, 1)
            if bits == 16:
                ref[b, :, p:p + n] = rows
            else:
                ref[b, :, p:p + n], ref_scale[b, :, p:p + n] = _encode(rows)
        assert _same(new, ref)
        if bits == 8:
            assert _same(getattr(c, name + "_scale"), ref_scale)
    n = _i32([12, 0, 51][:B])
    start = _i32([0, 3, 2][:B])
    got = c.read(start, 48, n)
    for x, full in zip(got, c.dequantize()):
        for b in range(B):
            s, m = int(start[b]), min(int(n[b]), 48)
            assert _same(x[b, :m], full[b, :, s:s + m].transpose(0, 1).to(BF16))
            assert not x[b, m:].any()


def test_every_code_is_the_definitions():
    """All pairs of a row's largest value and another one, at both ends of the exponents and between: ties and borders among them."""
    from mesh_b200.ops.cache import KVCache
    for e in (-133, -126, -100, -60, -58, 0, 100, 120):
        rows = []
        for m in range(128):
            a = (1 + m / 128) * 2.0 ** e if e > -126 else max(1, m) * 2.0 ** -133
            top = torch.tensor(a, dtype=F64).to(BF16)
            bits = int(top.view(torch.int16))
            others = torch.arange(max(0, bits - 9 * 128), bits + 1, dtype=torch.int32).to(torch.int16).view(BF16)
            for i in range(0, others.numel(), 255):
                row = torch.cat([top[None], others[i:i + 255]])
                rows.append(torch.cat([row, row.new_zeros(256 - row.numel())]))
        x = torch.stack(rows).to(DEV)
        x = x * torch.where(torch.arange(256, device=DEV) % 3 == 1, -1, 1).to(BF16)
        c = KVCache.empty(1, 1, len(rows), 256)
        c.append(x[None, :, None], x.flip(0)[None, :, None], _i32([0]))
        code, scale = _encode(x)
        assert _same(c.k[0, 0], code) and _same(c.k_scale[0, 0], scale)
        assert _same(c.v[0, 0], code.flip(0)) and _same(c.v_scale[0, 0], scale.flip(0))


def test_rows_that_are_not_finite_or_zero():
    from mesh_b200.ops.cache import KVCache
    x = torch.randn(1, 6, 1, 128, device=DEV).to(BF16)
    x[0, 1, 0, 77], x[0, 2, 0, 3], x[0, 3, 0, 127] = math.nan, math.inf, -math.inf
    x[0, 4] = 0
    c = KVCache.empty(1, 1, 8, 128)
    c.append(x, x.flip(1), _i32([0]))
    k, v = c.read(_i32([0]), 6)
    assert k[0, 1:4].isnan().all() and v[0, 2:5].isnan().all()
    assert k[0, 0].isfinite().all() and not k[0, 4].any() and k[0, 5].isfinite().all()


def test_rows_at_any_address():
    """Keys that do not start on 16 bytes, values with a stride that is no multiple of 8: read one by one."""
    g = _gen(3)
    wide = _randn(2, 5, 3 * 64 + 3, g=g)
    k, v = wide[..., 1:129].unflatten(-1, (2, 64)), wide[..., 67:195].unflatten(-1, (2, 64))
    for bits in (8, 16):
        a, b = _cache(2, 2, 9, 64, bits, _gen(0)), _cache(2, 2, 9, 64, bits, _gen(0))
        a.append(k, v, _i32([1, 4]))
        b.append(k.contiguous(), v.contiguous(), _i32([1, 4]))
        assert _same(a.k, b.k) and _same(a.v, b.v)


def test_rows_outside_the_cache_are_not_written():
    g = _gen(4)
    c = _cache(2, 1, 8, 64, 8, g)
    was = c.k.clone()
    x = _randn(2, 3, 1, 64, g=g)
    c.append(x, x, _i32([-5, 8]))
    c.append(x, x, _i32([2**31 - 1, -2**31]))
    c.append(x, x, _i32([0, 0]), _i32([-1, -2**31]))
    assert _same(c.k, was)
    c.append(x, x, _i32([-1, 7]))                              # two rows of the first land, one of the second
    assert _same(c.k[0, 0, :2], _encode(x[0, 1:, 0])[0]) and _same(c.k[1, 0, 7], _encode(x[1, 0, 0])[0])
    assert _same(c.k[0, 0, 2:], was[0, 0, 2:]) and _same(c.k[1, 0, :7], was[1, 0, :7])
    assert not c.read(_i32([8, -3]), 3)[0].any()


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes: the last sequence's rows are written, read and seen where they are."""
    from mesh_b200.ops.draft import draft_attention
    B, H, S, hd = 9, 8, 240000, 256
    c = _empty_big(B, H, S, hd)
    g = _gen(5)
    x, q = _randn(B, 2, H, hd, g=g), _randn(B, 2, H, hd, g=g)
    pos = _i32([S - 2] * B)
    c.append(x, x, pos)
    k, _ = c.read(pos, 2)
    code, scale = _encode(x)
    assert _same(k, (code.float() * scale[..., None]).to(BF16))
    o = draft_attention(q, c, pos, window=2)                   # the root sees slot S - 3 (zeros), the second node the two new rows
    s = ((q[:, 1] * hd ** -0.5).double()[:, None] * k.double()).sum(-1)
    want = (torch.softmax(s, 1)[..., None] * k.double()).sum(1)
    assert (o[:, 1].double() - want).abs().max() < 2e-2


def _empty_big(B, H, S, hd):
    from mesh_b200.ops.cache import KVCache
    k = torch.zeros((B, H, S, hd), dtype=torch.int8, device=DEV)
    return KVCache(k, torch.zeros_like(k), torch.zeros((B, H, S), device=DEV), torch.zeros((B, H, S), device=DEV))


# ------------------------------------------------------------------------------------------------------- kept rows
@pytest.mark.parametrize("bits,hd", [(8, 64), (8, 128), (8, 256), (16, 64), (16, 128), (16, 256)])
def test_keep(bits, hd):
    from mesh_b200.ops.cache import CacheGroup
    g = _gen(hd + bits)
    caches = [_cache(4, 3, 70, hd, bits, g) for _ in range(3)]
    pos = _i32([0, 5, 6, 60])
    path = torch.stack([torch.arange(64, device=DEV).flip(0),                     # every row of 64 changes places
                        torch.randint(0, 64, (64,), generator=g, device=DEV),     # some twice
                        torch.arange(64, device=DEV) // 2 * 2 + 1,
                        torch.arange(64, device=DEV) - 3]).to(torch.int32)        # before the first, behind the last slot
    counts = _i32([64, 64, 7, 64])
    want = []
    for c in caches:
        for x in (c.k, c.v) + ((c.k_scale, c.v_scale) if bits == 8 else ()):
            new = x.clone()
            for b in range(4):
                for i in range(int(counts[b])):
                    f, p = int(path[b, i]), int(pos[b])
                    if f >= 0 and p + f < 70 and p + i < 70:
                        new[b, :, p + i] = x[b, :, p + f]
            want.append(new)
    CacheGroup(caches).keep(pos, path, counts)
    got = [x for c in caches for x in (c.k, c.v) + ((c.k_scale, c.v_scale) if bits == 8 else ())]
    for a, b in zip(got, want):
        assert _same(a.view(torch.int8) if bits == 16 else a, b.view(torch.int8) if bits == 16 else b)


def test_keep_of_many_layers_and_odd_entries():
    from mesh_b200.ops.cache import CacheGroup
    g = _gen(9)
    caches = [_cache(1, 1, 16, 64, 16, g) for _ in range(130)]                    # three launches
    was = [c.k.clone() for c in caches]
    group = CacheGroup(caches)
    group.keep(_i32([2]), _i32([[5, 1, -1, 2**31 - 1]]))
    for c, w in zip(caches, was):
        w[0, 0, 2] = w[0, 0, 7]
        assert _same(c.k, w)
    group.keep(_i32([-3]), _i32([[5, 4]]))                                        # no slot
    group.keep(_i32([2**31 - 1]), _i32([[5, 4]]))
    group.keep(_i32([2]), _i32([[5, 4]]), _i32([-7]))
    for c, w in zip(caches, was):
        assert _same(c.k, w)


# ------------------------------------------------------------------------------------------------------- attention
def _words(B, T, how, g):
    from mesh_b200.ops.draft import tree_visible
    r = torch.rand((B, T), generator=g, device=DEV).tolist()
    if how == "chain":
        return None
    return tree_visible([[int(r[b][t] * t) if t else -1 for t in range(T)] for b in range(B)]).to(DEV)


def _attend64(q, cache, pos, counts, visible, window, scale):
    """(result, the same with |v|, a bound of |scores|), in 64 bits, of the rows behind counts nothing."""
    B, T, qh, hd = q.shape
    H = cache.k.shape[1]
    k, v = (x.double() for x in cache.dequantize())
    if cache.bits == 8:
        k, v = cache.k.double() * cache.k_scale.double()[..., None], cache.v.double() * cache.v_scale.double()[..., None]
    out = torch.zeros(B, T, qh, hd, dtype=F64, device=DEV)
    mag = torch.zeros_like(out)
    most = 0.0
    S = k.shape[2]
    for b in range(B):
        p, n = int(pos[b]), T if counts is None else int(counts[b])
        for t in range(min(n, T)):
            word = (1 << (t + 1)) - 1 if visible is None else int(visible[b, t]) & (1 << 64) - 1
            lo = max(0, p + max(1, bin(word).count("1")) - window) if window else 0
            slots = list(range(min(lo, p), p)) + [p + j for j in range(min(n, T)) if word >> j & 1 and p + j < S]
            if not slots:
                continue
            kk, vv = k[b][:, slots].repeat_interleave(qh // H, 0), v[b][:, slots].repeat_interleave(qh // H, 0)
            s = torch.einsum("hd,hsd->hs", q[b, t].double(), kk) * scale
            w = torch.softmax(s, -1)
            out[b, t] = torch.einsum("hs,hsd->hd", w, vv)
            mag[b, t] = torch.einsum("hs,hsd->hd", w, vv.abs())
            most = max(most, float((torch.einsum("hd,hsd->hs", q[b, t].double().abs(), kk.abs()) * scale).nan_to_num(0).max()))
    return out, mag, most


def _check(got, want, bits, keys, hd):
    """The result is rounded once (bf16, 2^-8).  A weight is rounded once (2^-11 in fp16, 2^-8 in bf16); its exponent is off by what the
    score is (a sum of hd products in fp32, at most (hd + 4) 2^-24 of the sum of their magnitudes), and ex2 and the
    factors around it by 2^-20; sums of `keys` terms in fp32 by keys 2^-24, in the numerator and in the denominator.  All
    of that is relative to the weighted sum of |v|."""
    out, mag, most = want
    rel = (2.0 ** -11 if bits == 8 else 2.0 ** -8) + 2 * ((hd + 4) * 2.0 ** -24 * most + 2.0 ** -20 + keys * 2.0 ** -24)
    far = (got.double() - out).abs() - (2.0 ** -8 * out.abs() + rel * (1 + 2.0 ** -8) * mag + 1e-30)
    assert not torch.isnan(got).any()
    assert far.max() <= 0, f"{far.max().item()} beyond the bound at {(far == far.max()).nonzero()[0].tolist()}"


CASES = [
    # B, T, G, H, S, positions, counts, tree, window, splits
    (1, 1, 1, 1, 16, [0], None, "chain", 0, 0),                       # the first token: one key
    (1, 1, 4, 2, 300, [17], None, "chain", 0, 1),
    (3, 1, 4, 2, 700, [0, 129, 699], None, "chain", 0, 0),            # the last slot
    (2, 1, 8, 1, 513, [512, 16], [1, 0], "chain", 0, 0),              # a sequence without tokens
    (2, 2, 3, 2, 64, [0, 15], None, "tree", 0, 1),
    (2, 5, 5, 1, 200, [31, 100], [5, 3], "tree", 0, 3),
    (2, 16, 4, 2, 1024, [500, 1008], [16, 12], "tree", 512, 0),       # the decoder's local layer
    (2, 33, 3, 2, 1300, [1, 1111], [33, 25], "tree", 0, 0),
    (1, 64, 8, 1, 400, [300], None, "tree", 64, 5),                   # a window as short as it may be
    (1, 64, 1, 3, 130, [66], None, "chain", 0, 64),                   # more slices than keys to share
    (4, 7, 2, 4, 260, [3, 250, 255, 259], [7, 7, 5, 1], "tree", 40, 2),   # drafts that run past the cache
    (1, 17, 16, 1, 2000, [1800], None, "chain", 0, 0),
]


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_attention(case, bits, hd):
    from mesh_b200.ops.draft import draft_attention
    B, T, G, H, S, positions, counts, how, window, splits = case
    g = _gen(hash((case[:5], hd)) % 2**31)
    cache = _cache(B, H, S, hd, bits, g)
    q = _randn(B, T, G * H, hd, g=g, scale=1.5)
    pos, counts = _i32(positions), None if counts is None else _i32(counts)
    visible = _words(B, T, how, g)
    out = torch.full_like(q, 7.0)
    got = draft_attention(q, cache, pos, counts=counts, visible=visible, window=window, out=out, splits=splits)
    assert got is out
    want = _attend64(q, cache, pos, counts, visible, window, hd ** -0.5)
    for b in range(B):
        n = T if counts is None else int(counts[b])
        assert (out[b, n:] == 7.0).all()                              # rows behind the last node are left alone
        out[b, n:] = 0
    _check(out, want, bits, S, hd)
    again = draft_attention(q, cache, pos, counts=counts, visible=visible, window=window, splits=splits)
    for b in range(B):
        n = T if counts is None else int(counts[b])
        assert _same(again[b, :n], out[b, :n]) and not again[b, n:].any()


CUTS = [
    # B, T, G, H, S, positions, counts: short caches, where a cluster has an item and its CTAs join their parts, and more items than SMs
    (1, 2, 4, 2, 1500, [1400], None),                                 # few items: clusters of 8
    (3, 1, 4, 8, 2000, [0, 60, 1999], None),                          # 24 items; the first two lie in one CTA
    (8, 3, 2, 8, 900, [0, 100, 897, 300, 890, 500, 2, 899], [3, 0, 1, 2, 3, 3, 3, 3]),      # 64 items; one sequence has none
    (16, 1, 2, 8, 400, [25 * i for i in range(16)], None),            # 128 items, a CTA each
    (40, 1, 1, 8, 300, [7 * i for i in range(40)], None),             # 320 items
    (2, 40, 4, 1, 900, [850, 3], [40, 10]),                           # tiles of 128 rows; the second sequence has one tile of two
    (5, 33, 4, 3, 500, [0, 31, 64, 400, 467], [33, 32, 1, 0, 33]),
    (2, 9, 16, 12, 700, [690, 63], None),                             # 48 items of 128 rows, the last 16 in tiles of their own
    (4, 40, 4, 8, 600, [0, 100, 300, 560], [40, 33, 3, 0]),           # 64 items of 128 rows, some sequences with one tile of two
    (1, 64, 8, 2, 2500, [2436], None),                                # 8 items of 128 rows
]


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("case", CUTS, ids=str)
def test_attention_of_short_caches(case, bits, hd):
    from mesh_b200.ops.draft import draft_attention
    B, T, G, H, S, positions, counts = case
    g = _gen(B * T + hd)
    cache = _cache(B, H, S, hd, bits, g)
    q = _randn(B, T, G * H, hd, g=g, scale=1.5)
    pos, counts, visible = _i32(positions), None if counts is None else _i32(counts), _words(B, T, "tree", g)
    want = _attend64(q, cache, pos, counts, visible, 0, hd ** -0.5)
    for splits in (0, 148):                                           # shares of all keys, joined by the second kernel
        _check(draft_attention(q, cache, pos, counts=counts, visible=visible, splits=splits), want, bits, S, hd)


@pytest.mark.parametrize("bits,hd,T", [(8, 128, 16), (16, 128, 16), (8, 256, 64), (16, 256, 12), (8, 64, 33)])
def test_attention_of_many_rows_repeats(bits, hd, T):
    """Many passes over long contexts give the same bits: no group of threads runs ahead of what another has still to read."""
    from mesh_b200.ops.draft import draft_attention
    from mesh_b200.utils.status import check_status
    B, G, H, S = 4, 4, 8, 12000
    g = _gen(hd + T)
    cache = _cache(B, H, S, hd, bits, g)
    q = _randn(B, T, G * H, hd, g=g, scale=3.0)                       # large scores: the reference points move
    pos, visible = _i32([11000, 6001, 9000, 11900]), _words(B, T, "tree", g)
    first = draft_attention(q, cache, pos, visible=visible)
    for _ in range(100):
        assert _same(draft_attention(q, cache, pos, visible=visible), first)
    check_status()


@pytest.mark.parametrize("T", [2, 12])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("positions", [[1500] * 6, [0, 40, 6000, 90, 3, 20990], [1], [700] * 33 + [20990, 8]], ids=["alike", "ragged", "one", "many"])
def test_attention_in_a_long_cache(positions, bits, T):
    """Contexts much shorter than the cache: items in equal pieces, or shares that end within items, by the lengths found on the device."""
    from mesh_b200.ops.draft import draft_attention
    B, G, H, S, hd = len(positions), 4, 2, 21000, 64
    g = _gen(B + T)
    cache = _cache(B, H, S, hd, bits, g)
    q = _randn(B, T, G * H, hd, g=g, scale=1.5)
    pos, visible = _i32(positions), _words(B, T, "tree", g)
    _check(draft_attention(q, cache, pos, visible=visible), _attend64(q, cache, pos, None, visible, 0, hd ** -0.5), bits, S, hd)


@pytest.mark.parametrize("bits", [8, 16])
def test_attention_rows_that_see_nothing(bits):
    from mesh_b200.ops.draft import draft_attention
    g = _gen(1)
    cache = _cache(2, 2, 40, 64, bits, g)
    q = _randn(2, 4, 4, 64, g=g)
    visible = torch.tensor([[0, 2, 0, 15], [0, 0, 0, 0]], dtype=torch.int64, device=DEV)
    pos = _i32([0, 9])
    got = draft_attention(q, cache, pos, visible=visible)
    assert not got[0, 0].any() and not got[0, 2].any()
    assert _same(got[0, 1].view(2, 2, 64), cache.dequantize()[1][0, :, 1].to(BF16)[:, None].expand(2, 2, 64)) or bits == 8
    _check(got, _attend64(q, cache, pos, None, visible, 0, 0.125), bits, 40, 64)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_does_not_see_what_is_hidden(bits, hd, bad):
    """NaN and infinities behind the drafts, in other branches, before the window and in other sequences reach nobody else."""
    from mesh_b200.ops.draft import draft_attention, tree_visible
    g = _gen(2)
    B, T, H, S = 3, 6, 2, 200
    cache = _cache(B, H, S, hd, bits, g)
    q = _randn(B, T, 2 * H, hd, g=g)
    pos = _i32([100, 60, 100])
    visible = tree_visible([[-1, 0, 0, 2, 1, 3]] * B).to(DEV)
    window = 30
    want = _attend64(q, cache, pos, None, visible, window, hd ** -0.5)

    def spoil(b, slot):
        if bits == 16:
            cache.k[b, :, slot, ::3] = bad
            cache.v[b, :, slot, 1::5] = bad
        else:
            cache.k_scale[b, :, slot] = cache.v_scale[b, :, slot] = math.nan if math.isnan(bad) else bad
    spoil(0, 101)                          # node 1: seen by nodes 1 and 4 only
    for slot in (0, 70, 106, 199):         # before every window and behind the drafts
        spoil(0, slot)
    spoil(2, 71)                           # the root's window begins here; its descendants' later
    got = draft_attention(q, cache, pos, visible=visible, window=window)
    hit = torch.zeros(B, T, dtype=torch.bool)
    hit[0, [1, 4]] = True
    hit[2, 0] = True
    for b in range(B):
        for t in range(T):
            if hit[b, t]:
                assert not got[b, t].isfinite().all()
                got[b, t] = 0
                want[0][b, t] = 0
                want[1][b, t] = 0
    _check(got, want, bits, S, hd)


def test_attention_scales_far_apart():
    """8-bit rows whose scales span 2^100: values of large rows are not lost beside small ones and the other way round."""
    from mesh_b200.ops.draft import draft_attention
    g = _gen(6)
    cache = _cache(1, 1, 64, 128, 8, g)
    cache.v_scale[0, 0, :32] *= 2.0 ** 60
    cache.v_scale[0, 0, 32:40] *= 2.0 ** -40
    q = _randn(1, 2, 2, 128, g=g)
    for pos in (40, 30, 62):
        visible = torch.tensor([[1, 3]], device=DEV)
        p = _i32([pos])
        _check(draft_attention(q, cache, p, visible=visible), _attend64(q, cache, p, None, visible, 0, 128 ** -0.5), 8, 64, 128)
    small = _cache(1, 1, 64, 128, 8, g)
    small.v_scale *= 2.0 ** -70
    small.k_scale *= 2.0 ** -30
    p = _i32([50])
    _check(draft_attention(q * 2.0 ** 30, small, p), _attend64(q * 2.0 ** 30, small, p, None, None, 0, 128 ** -0.5), 8, 64, 128)
    zero = _cache(1, 1, 64, 128, 8, g)
    zero.v_scale.zero_()
    assert not draft_attention(q, zero, p).any()


def test_attention_strides_and_scale():
    """Queries that are columns of a fused projection, an output that is part of a wider one, a scale of one's own."""
    from mesh_b200.ops.draft import draft_attention
    g = _gen(7)
    for bits in (8, 16):
        cache = _cache(2, 2, 90, 128, bits, g)
        fused = _randn(2, 5, 4 * 128 + 3 * 128 + 1, g=g)
        q = fused[..., 1:513].unflatten(-1, (4, 128))                     # 2-byte aligned
        wide = torch.full((2, 5, 700), 5.0, dtype=BF16, device=DEV)
        out = wide[..., 2:514].unflatten(-1, (4, 128))
        pos = _i32([80, 3])
        draft_attention(q, cache, pos, out=out, scale=0.3)
        _check(out, _attend64(q, cache, pos, None, None, 0, 0.3), bits, 90, 128)
        assert (wide[..., :2] == 5).all() and (wide[..., 514:] == 5).all()


def test_attention_positions_outside_the_cache_read_nothing_there():
    from mesh_b200.ops.draft import draft_attention
    g = _gen(8)
    cache = _cache(3, 1, 20, 64, 8, g)
    q = _randn(3, 2, 1, 64, g=g)
    got = draft_attention(q, cache, _i32([2**31 - 1, -2**31, 20]))
    full = draft_attention(q, cache, _i32([20, 0, 20]))
    assert _same(got, full)


@pytest.mark.parametrize("bits", [8, 16])
def test_attention_long_cache_in_slices(bits):
    """A long sequence beside short ones; slices of every number give the same rows to rounding."""
    from mesh_b200.ops.draft import draft_attention
    g = _gen(11)
    B, T, H, S, hd = 3, 4, 2, 20011, 128
    cache = _cache(B, H, S, hd, bits, g)
    q = _randn(B, T, 4 * H, hd, g=g, scale=2.0)
    pos, visible = _i32([20007, 5, 9000]), _words(B, T, "tree", g)
    want = _attend64(q, cache, pos, None, visible, 0, hd ** -0.5)
    for splits in (0, 1, 2, 7, 63, 64, 1000):
        _check(draft_attention(q, cache, pos, visible=visible, splits=splits), want, bits, S, hd)


# ---------------------------------------------------------------------------------------------------------- logits
def _constrain64(x, history, hlen, plen, rep, pres, freq, ids, bias, blen, allowed, offset):
    R, V = x.shape
    out = x.double().clone()
    for r in range(R):
        h = [int(i) - offset for i in history[r, :int(hlen[r])]] if history is not None else []
        made = h[max(0, int(plen[r])) if plen is not None else 0:]
        for i in set(h):
            if 0 <= i < V:
                if rep is not None:
                    out[r, i] = out[r, i] / rep[r].double() if out[r, i] > 0 else out[r, i] * rep[r].double()
                n = made.count(i)
                if n:
                    out[r, i] -= (freq[r].double() * n if freq is not None else 0) + (pres[r].double() if pres is not None else 0)
        if ids is not None:
            last = {int(ids[r, j]) - offset: float(bias[r, j]) for j in range(int(blen[r]) if blen is not None else ids.shape[1])}
            for i, b in last.items():
                if 0 <= i < V:
                    out[r, i] += b
        if allowed is not None:
            for w in range((V + 31) // 32):
                word = int(allowed[r, w]) & 0xFFFFFFFF
                for i in range(32):
                    if w * 32 + i < V and not word >> i & 1:
                        out[r, w * 32 + i] = -math.inf
    return out


def _check_logits(got, want, half):
    """fp32: at most five steps (quotient, product, two differences, sum), each half a step of a value not above the largest one
    met, 64 here; bf16: rounded once more."""
    inf = torch.isinf(want)
    assert _same(got.double()[inf], want[inf])
    far = (got.double() - want)[~inf].abs() - (5 * 64 * 2.0 ** -24 + (2.0 ** -8 * want[~inf].abs() if half else 0))
    assert far.numel() == 0 or far.max() <= 0


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("R,V,hist,nbias,mask", [(1, 1, 3, 1, False), (3, 1000, 40, 7, True), (2, 16384, 300, 0, False), (2, 16385, 1500, 33, True),
                                                 (5, 40001, 0, 5, True), (2, 131072, 64, 0, True)])
def test_constrain(R, V, hist, nbias, mask, half):
    from mesh_b200.ops.logits import constrain_logits
    g = _gen(V + half)
    off = 100
    logits = (torch.randn((R, V), generator=g, device=DEV) * 3).to(BF16 if half else torch.float32)
    few = torch.randint(off - 5, off + V + 5, (R, max(1, hist // 4)), generator=g, device=DEV)
    history = few.gather(1, torch.randint(0, few.shape[1], (R, hist), generator=g, device=DEV)).to(torch.int32)
    hlen = torch.randint(0, hist + 1, (R,), generator=g, device=DEV).to(torch.int32)
    hlen[0] = hist
    plen = hlen // 3
    rep, pres, freq = (0.5 + torch.rand(R, generator=g, device=DEV) for _ in range(3))
    ids = torch.randint(off - 2, off + V + 2, (R, nbias), generator=g, device=DEV).to(torch.int32)
    if nbias > 2:
        ids[:, 2] = ids[:, 0]                                             # an id twice: the later one counts
    bias = torch.randn((R, nbias), generator=g, device=DEV) * 5
    blen = _i32([nbias - (r % 2) for r in range(R)]).clamp(min=0)
    allowed = torch.randint(-2**31, 2**31, (R, (V + 31) // 32), generator=g, device=DEV).to(torch.int32) if mask else None
    want = _constrain64(logits.cpu(), history.cpu(), hlen, plen, rep.cpu(), pres.cpu(), freq.cpu(), ids.cpu(), bias.cpu(), blen, None if allowed is None else allowed.cpu(), off)
    kw = dict(history=history, history_len=hlen, prompt_len=plen, repetition=rep, presence=pres, frequency=freq, bias_ids=ids, bias=bias,
              bias_len=blen, allowed=allowed, vocab_offset=off)
    tokens = torch.full((R,), -7, dtype=torch.int32, device=DEV)
    out = constrain_logits(logits, out=torch.empty_like(logits), tokens=tokens, **kw)
    _check_logits(out.cpu(), want, half)
    for r in range(R):
        top = float(want[r].max())
        t = int(tokens[r])
        if top == -math.inf:
            assert t == -1
        else:                                                             # within rounding of the largest, and the only one if it leads
            assert want[r, t - off] >= top - 2 * 5 * 64 * 2.0 ** -24
    # the choice alone, and the result written over the logits
    alone = torch.full((R,), -7, dtype=torch.int32, device=DEV)
    assert constrain_logits(logits, tokens=alone, **kw) is alone and _same(alone, tokens)
    own = logits.clone()
    assert constrain_logits(own, out=own, **kw) is own and _same(own, out)


def test_constrain_ties_nan_and_nothing_allowed():
    from mesh_b200.ops.logits import constrain_logits
    V = 50000
    x = torch.full((5, V), 1.5, device=DEV)
    x[1, 17], x[1, 30000] = math.nan, 2.0
    x[2] = -math.inf
    x[3] = math.nan
    x[4, 49999] = math.inf
    tokens = torch.zeros(5, dtype=torch.int32, device=DEV)
    constrain_logits(x, tokens=tokens)
    assert tokens.tolist() == [0, 30000, -1, -1, 49999]
    none = torch.zeros((1, (V + 31) // 32), dtype=torch.int32, device=DEV).expand(5, -1)     # one mask for all rows
    out = torch.empty_like(x)
    constrain_logits(x, allowed=none, out=out, tokens=tokens)
    assert tokens.tolist() == [-1] * 5 and (out == -math.inf).all()
    one = none.clone()
    one[:, 40000 // 32] = 1 << 40000 % 32
    constrain_logits(x, allowed=one, out=out, tokens=tokens)
    assert tokens.tolist() == [40000, 40000, -1, -1, 40000]


def test_constrain_long_history_of_one_token():
    """65535 times the same token: the count does not run over; and the largest bias list."""
    from mesh_b200.ops.logits import constrain_logits
    V = 20000
    x = torch.zeros((1, V), device=DEV)
    h = torch.full((1, 65535), 7, dtype=torch.int32, device=DEV)
    ids = torch.arange(32767, device=DEV).remainder(V)[None].to(torch.int32)
    bias = torch.arange(32767, device=DEV).float()[None]
    one = torch.ones(1, device=DEV)
    out = constrain_logits(x, history=h, frequency=one, bias_ids=ids, bias=bias, out=torch.empty_like(x))
    want = torch.arange(V, device=DEV).float()
    want[:32767 - V] += V                                                 # the second entry of an id
    want[7] -= 65535
    assert _same(out[0], want)


def test_constrain_strides():
    from mesh_b200.ops.logits import constrain_logits
    for dtype in (torch.float32, BF16):
        wide = torch.randn(3, 5003, device=DEV).to(dtype)
        x = wide[:, 1:5001]                                               # neither aligned nor a stride of whole vectors
        room = torch.zeros(3, 6001, device=DEV, dtype=dtype)
        out = room[:, 3:5003]
        h = torch.arange(9, device=DEV, dtype=torch.int32)[None].expand(3, -1)
        rep = torch.tensor([1.3, 2.0, 0.7], device=DEV)
        constrain_logits(x, history=h, repetition=rep, out=out)
        want = x.float().clone()
        want[:, :9] = torch.where(want[:, :9] > 0, want[:, :9] / rep[:, None], want[:, :9] * rep[:, None])
        assert _same(out, want.to(dtype)) and not room[:, :3].any() and not room[:, 5003:].any()


def test_constrain_refusals():
    from mesh_b200.ops.logits import constrain_logits
    x = torch.zeros(2, 64, device=DEV)
    tok = torch.zeros(2, dtype=torch.int32, device=DEV)
    h = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    f = torch.ones(2, device=DEV)
    for kw in (dict(), dict(out=x.double()), dict(out=x[:1]), dict(tokens=tok.long()), dict(tokens=tok[:1]), dict(tokens=tok, repetition=f),
               dict(tokens=tok, history_len=tok), dict(tokens=tok, history=h.long()), dict(tokens=tok, history=h[:1]), dict(tokens=tok, history=h.cpu()),
               dict(tokens=tok, history=h, presence=f.double()), dict(tokens=tok, history=h, frequency=f[:1]), dict(tokens=tok, bias=torch.zeros(2, 3, device=DEV)),
               dict(tokens=tok, bias_ids=h), dict(tokens=tok, bias_ids=h, bias=torch.zeros(2, 4, device=DEV)), dict(tokens=tok, bias_len=tok),
               dict(tokens=tok, allowed=torch.zeros(2, 3, dtype=torch.int32, device=DEV)), dict(tokens=tok, history=torch.zeros(2, 65536, dtype=torch.int32, device=DEV)),
               dict(tokens=tok, bias_ids=torch.zeros(2, 32768, dtype=torch.int32, device=DEV), bias=torch.zeros(2, 32768, device=DEV)),
               dict(out=x[:1].expand(2, -1))):
        with pytest.raises(ValueError):
            constrain_logits(x, **kw)
    for bad in (x.half(), x[0], x[:, :0], x.t(), x[:1].expand(2, -1)):
        with pytest.raises(ValueError):
            constrain_logits(bad, tokens=tok)
    assert constrain_logits(x[:0], tokens=tok[:0]).numel() == 0


# ---------------------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("bits", [8, 16])
def test_a_step_of_drafts(bits):
    """Rows appended, a tree attends, its accepted branch is kept, and the next token sees the same sequence that a cache written without
    a tree holds; the whole step captured in a graph and replayed on other inputs."""
    from mesh_b200.ops.cache import CacheGroup
    from mesh_b200.ops.draft import draft_attention, tree_visible
    g = _gen(12)
    B, T, H, G, S, hd = 2, 7, 2, 2, 64, 128
    parents = [[-1, 0, 0, 1, 1, 2, 4]] * B
    branch = _i32([[0, 1, 4, 6], [0, 2, 5, 0]])
    kept = _i32([4, 3])
    visible = tree_visible(parents).to(DEV)
    layers = [_cache(B, H, S, hd, bits, g) for _ in range(2)]
    group = CacheGroup(layers)
    pos = _i32([20, 33])
    rows = [_randn(B, T, 2 * H * hd, g=g) for _ in layers]
    q = _randn(B, T, G * H, hd, g=g)
    out = [torch.zeros_like(q) for _ in layers]

    def step():
        for c, x, o in zip(layers, rows, out):
            c.append(x[..., :H * hd].view(B, T, H, hd), x[..., H * hd:].view(B, T, H, hd), pos)
            draft_attention(q, c, pos, visible=visible, out=o)
        group.keep(pos, branch, kept)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        step()
    for c in layers:                                                      # new inputs, in place
        fresh = _cache(B, H, S, hd, bits, g)
        c.k.copy_(fresh.k); c.v.copy_(fresh.v)
        if bits == 8:
            c.k_scale.copy_(fresh.k_scale); c.v_scale.copy_(fresh.v_scale)
    for x in rows:
        x.copy_(_randn(B, T, 2 * H * hd, g=g))
    q.copy_(_randn(B, T, G * H, hd, g=g))
    pos.copy_(_i32([11, 40]))
    # the same by hand: every node by itself, along its path
    plain = [[x.clone() for x in (c.k, c.v) + ((c.k_scale, c.v_scale) if bits == 8 else ())] for c in layers]
    graph.replay()
    torch.cuda.synchronize()
    from mesh_b200.ops.cache import KVCache
    for c, tensors, x, o in zip(layers, plain, rows, out):
        ref = KVCache(*tensors)
        ref.append(x[..., :H * hd].view(B, T, H, hd), x[..., H * hd:].view(B, T, H, hd), pos)
        _check(o, _attend64(q, ref, pos, None, visible, 0, hd ** -0.5), bits, S, hd)
        for b in range(B):
            p, path = int(pos[b]), branch[b, :int(kept[b])].long()
            line = KVCache(*[t[b:b + 1].clone() for t in tensors])        # a sequence that was never drafted
            xs = x[b:b + 1, path]
            line.append(xs[..., :H * hd].view(1, -1, H, hd), xs[..., H * hd:].view(1, -1, H, hd), pos[b:b + 1])
            n = p + len(path)
            assert _same(c.k[b, :, :n], line.k[0, :, :n]) and _same(c.v[b, :, :n], line.v[0, :, :n])
            if bits == 8:
                assert _same(c.k_scale[b, :, :n], line.k_scale[0, :, :n]) and _same(c.v_scale[b, :, :n], line.v_scale[0, :, :n])
            # node 6 (or 5) saw exactly what the last token of that line sees
            last = q[b:b + 1, path[-1:]].contiguous()
            one = draft_attention(last, line, pos[b:b + 1] + len(path) - 1)
            far = (one.double() - o[b:b + 1, path[-1:]].double()).abs().max()
            assert far <= 4 * 2.0 ** -8 * one.abs().max().double()


def test_two_streams_at_once():
    """Two streams attend over one cache, in slices: neither touches the other's partial sums."""
    from mesh_b200.ops.draft import draft_attention
    g = _gen(13)
    cache = _cache(2, 2, 3000, 128, 8, g)
    qs = [_randn(2, 1, 8, 128, g=g) for _ in range(2)]
    pos = _i32([2999, 1500])
    want = [draft_attention(q, cache, pos, splits=16) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(draft_attention(qs[i], cache, pos, splits=16))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(_same(x, want[i]) for x in got[i])
