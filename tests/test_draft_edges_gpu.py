"""Operators for drafted tokens at the edges of what their documentation allows, beside ``test_draft_gpu``: the kernel for many query
rows with everything that is hidden, absent or unaligned, a cancelled pass, large lists."""
import math

import pytest
import torch

from test_draft_gpu import BF16, DEV, _attend64, _cache, _check, _check_logits, _gen, _i32, _randn, _same, _words

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits,hd", [(8, 128), (16, 256)])
def test_a_cancelled_pass_ends_and_is_reported_as_cancelled(bits, hd):
    """The host's abort flag is up while passes over long contexts run: waits may give up, and then say so; none is reported as one that
    ran out.  With the flag down again the next pass is right."""
    from mesh_b200.ops.draft import draft_attention
    from mesh_b200.utils.status import clear_abort, decode, raise_abort, status_block
    B, T, G, H, S = 4, 16, 4, 2, 12000
    g = _gen(hd)
    cache = _cache(B, H, S, hd, bits, g)
    q = _randn(B, T, G * H, hd, g=g)
    pos, visible = _i32([11000, 6001, 9000, 11900]), _words(B, T, "tree", g)
    want = draft_attention(q, cache, pos, visible=visible)
    torch.cuda.synchronize()
    try:
        raise_abort()
        for _ in range(20):
            draft_attention(q, cache, pos, visible=visible)
        torch.cuda.synchronize()
        code = decode(status_block())["code"]
    finally:
        clear_abort()
        status_block()[:11].zero_()
    assert code in ("OK", "CANCELED")
    assert _same(draft_attention(q, cache, pos, visible=visible), want)
    assert decode(status_block())["code"] == "OK"


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hist,nbias", [(65535, 32767), (16384, 0), (16001, 382), (5000, 300)])
def test_large_lists_over_a_large_vocabulary(hist, nbias, half):
    """As many listed ids as a CTA's memory takes, and more, where sixteen CTAs share a row, or eight if sixteen do not fit."""
    from mesh_b200.ops.logits import constrain_logits
    g = _gen(hist + half)
    R, V = 3, 262144
    logits = (torch.randn((R, V), generator=g, device=DEV) * 3).to(BF16 if half else torch.float32)
    history = torch.randint(0, V, (R, hist), generator=g, device=DEV).to(torch.int32)
    history[1] %= 16384                                                   # all in the first CTA's share
    history[2, ::2] = 200000
    plen = _i32([hist // 3, 0, hist // 2])
    rep, pres, freq = (0.5 + torch.rand(R, generator=g, device=DEV) for _ in range(3))
    freq *= 2.0 ** -12                                                    # 65535 times that is below 25
    ids = torch.randint(0, V, (R, nbias), generator=g, device=DEV).to(torch.int32)
    bias = torch.randn((R, nbias), generator=g, device=DEV) * 5
    want = logits.double()
    for r in range(R):
        seen = torch.bincount(history[r].long(), minlength=V) > 0
        times = torch.bincount(history[r, int(plen[r]):].long(), minlength=V).double()
        x = torch.where(seen, torch.where(want[r] > 0, want[r] / rep[r].double(), want[r] * rep[r].double()), want[r])
        x -= freq[r].double() * times + pres[r].double() * (times > 0)
        last = {int(i): float(b) for i, b in zip(ids[r].tolist(), bias[r].tolist())}          # of an id listed twice the last entry counts
        x[torch.tensor(list(last), dtype=torch.int64, device=DEV)] += torch.tensor(list(last.values()), dtype=torch.float64, device=DEV)
        want[r] = x
    want = want.cpu()
    tokens = torch.zeros(R, dtype=torch.int32, device=DEV)
    out = constrain_logits(logits, history=history, prompt_len=plen, repetition=rep, presence=pres, frequency=freq, bias_ids=ids, bias=bias,
                           out=torch.empty_like(logits), tokens=tokens)
    _check_logits(out.cpu(), want, half)
    for r in range(R):
        assert want[r, int(tokens[r])] >= want[r].max() - 2 * 5 * 64 * 2.0 ** -24


# ------------------------------------------------------- the kernel for many query rows: more than 32 of a (sequence, KV head), `splits` given
def _spoil(cache, b, slot, bad):
    if cache.bits == 16:
        cache.k[b, :, slot, ::3] = bad
        cache.v[b, :, slot, 1::5] = bad
    else:
        cache.k_scale[b, :, slot] = cache.v_scale[b, :, slot] = bad


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("T,G,window,splits", [(12, 4, 100, 3), (33, 4, 90, 40), (9, 4, 0, 1)])
def test_many_rows_do_not_see_what_is_hidden(bits, hd, bad, T, G, window, splits):
    """NaN and infinities behind the drafts, in other branches, before the window and in other sequences reach nobody else."""
    from mesh_b200.ops.draft import draft_attention
    g = _gen(2)
    B, H, S = 3, 2, 700
    cache = _cache(B, H, S, hd, bits, g)
    q = _randn(B, T, G * H, hd, g=g)
    pos = _i32([400, 60, 401])
    visible = _words(B, T, "tree", g)
    want = _attend64(q, cache, pos, None, visible, window, hd ** -0.5)
    words, p = visible.cpu(), pos.tolist()
    spoilt = [(0, 400 + 1), (0, 400 + T), (0, S - 1), (2, 401 + T - 1), (2, S - 1)]     # nodes 1 and T - 1, and what lies behind
    if window:
        spoilt += [(0, 0), (0, 400 - window), (2, 401 - window + 1), (1, 60 + T)]       # before every window; where the root's window begins
    for b, slot in spoilt:
        _spoil(cache, b, slot, bad)
    got = draft_attention(q, cache, pos, visible=visible, window=window, splits=splits)
    for b in range(B):
        for t in range(T):
            word = int(words[b, t]) & (1 << 64) - 1
            lo = max(0, p[b] + bin(word).count("1") - window) if window else 0
            if any(sb == b and (lo <= s < p[b] or (p[b] <= s < p[b] + T and word >> (s - p[b]) & 1)) for sb, s in spoilt):
                assert not got[b, t].isfinite().all(), (b, t)
                got[b, t] = 0
                want[0][b, t] = 0
                want[1][b, t] = 0
    assert want[0].any(-1).any(-1).any(-1).all()                          # in every sequence some node saw none of it
    _check(got, want, bits, S, hd)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("T,G,splits", [(12, 4, 1), (12, 4, 7), (64, 4, 30), (40, 1, 2)])
def test_many_rows_see_infinite_values_where_they_are(hd, T, G, splits):
    """An infinite value that a node sees makes its column infinite, of its sign, and no other; opposite ones make a NaN."""
    from mesh_b200.ops.draft import draft_attention
    g = _gen(hd + T)
    B, H, S = 2, 2, 500
    cache = _cache(B, H, S, hd, 16, g)
    q = _randn(B, T, G * H, hd, g=g)
    pos = _i32([S - T, 70])
    visible = _words(B, T, "tree", g)
    for b, node, column, bad in ((0, 1, 3, math.inf), (0, 2, hd - 1, -math.inf), (0, 0, 9, math.inf), (0, 3, 9, -math.inf), (1, 1, 0, math.nan)):
        cache.v[b, :, int(pos[b]) + node, column] = bad
    cache.v[1, 0, 69, 5] = math.inf                                       # the last slot before the drafts: every node of one head sees it
    out, mag, most = _attend64(q, cache, pos, None, visible, 0, hd ** -0.5)
    got = draft_attention(q, cache, pos, visible=visible, splits=splits)
    odd = ~out.isfinite()
    assert odd.any() and odd.float().mean() < 0.2
    assert _same(got.double()[odd].nan_to_num(0), out[odd].nan_to_num(0)) and _same(got[odd].isnan(), out[odd].isnan())
    _check(got.masked_fill(odd, 0), (out.masked_fill(odd, 0), mag.masked_fill(odd, 0), most), 16, S, hd)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("splits", [1, 5])
def test_many_rows_that_see_nothing(bits, splits):
    from mesh_b200.ops.draft import draft_attention
    g = _gen(1)
    B, T, G, H, S, hd = 2, 12, 4, 2, 300, 128
    cache = _cache(B, H, S, hd, bits, g)
    q = _randn(B, T, G * H, hd, g=g)
    visible = torch.tensor([[0, 2, 0, 15] * 3, [0] * 12], dtype=torch.int64, device=DEV)
    pos = _i32([0, 200])
    got = draft_attention(q, cache, pos, visible=visible, splits=splits)
    assert not got[0, ::4].any() and not got[0, 2::4].any()
    _check(got, _attend64(q, cache, pos, None, visible, 0, hd ** -0.5), bits, S, hd)
    window = draft_attention(q, cache, pos, visible=visible, window=12, splits=splits)
    _check(window, _attend64(q, cache, pos, None, visible, 12, hd ** -0.5), bits, S, hd)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_many_rows_scales_far_apart(hd):
    """8-bit rows whose scales span 2^100, and queries of the inverse size."""
    from mesh_b200.ops.draft import draft_attention
    g = _gen(6)
    T, G, S = 10, 4, 200
    q = _randn(1, T, G, hd, g=g)
    visible = _words(1, T, "tree", g)
    cache = _cache(1, 1, S, hd, 8, g)
    cache.v_scale[0, 0, :100] *= 2.0 ** 60
    cache.v_scale[0, 0, 100:140] *= 2.0 ** -40
    for pos in (150, 70, 190):
        p = _i32([pos])
        _check(draft_attention(q, cache, p, visible=visible, splits=2), _attend64(q, cache, p, None, visible, 0, hd ** -0.5), 8, S, hd)
    small = _cache(1, 1, S, hd, 8, g)
    small.v_scale *= 2.0 ** -70
    small.k_scale *= 2.0 ** -30
    p = _i32([130])
    _check(draft_attention(q * 2.0 ** 30, small, p, splits=1), _attend64(q * 2.0 ** 30, small, p, None, None, 0, hd ** -0.5), 8, S, hd)
    zero = _cache(1, 1, S, hd, 8, g)
    zero.v_scale.zero_()
    assert not draft_attention(q, zero, p, splits=2).any()


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("splits", [0, 1, 3])
def test_many_rows_strides_and_scale(bits, splits):
    """Queries that are columns of a fused projection, an output that is part of a wider one, a scale of one's own."""
    from mesh_b200.ops.draft import draft_attention
    g = _gen(7)
    S = 6000                                                              # long enough for this kernel with splits of 0 too
    cache = _cache(2, 2, S, 128, bits, g)
    fused = _randn(2, 20, 4 * 128 + 3 * 128 + 1, g=g)
    q = fused[..., 1:513].unflatten(-1, (4, 128))                         # 2-byte aligned
    wide = torch.full((2, 20, 700), 5.0, dtype=BF16, device=DEV)
    out = wide[..., 2:514].unflatten(-1, (4, 128))
    pos = _i32([500, 3])
    draft_attention(q, cache, pos, out=out, scale=0.3, splits=splits)
    _check(out, _attend64(q, cache, pos, None, None, 0, 0.3), bits, S, 128)
    assert (wide[..., :2] == 5).all() and (wide[..., 514:] == 5).all()


def test_many_rows_outside_the_cache_read_nothing_there():
    from mesh_b200.ops.draft import draft_attention
    g = _gen(8)
    cache = _cache(3, 1, 150, 64, 8, g)
    q = _randn(3, 40, 1, 64, g=g)
    for splits in (1, 4):
        got = draft_attention(q, cache, _i32([2**31 - 1, -2**31, 150]), splits=splits)
        full = draft_attention(q, cache, _i32([150, 0, 150]), splits=splits)
        assert _same(got, full)
        _check(got, _attend64(q, cache, _i32([150, 0, 150]), None, None, 0, 0.125), 8, 150, 64)


@pytest.mark.parametrize("bits", [8, 16])
def test_many_rows_past_32_bits(bits):
    """A cache of more than 2^32 bytes a side: the last sequence's rows are seen where they are."""
    from mesh_b200.ops.cache import KVCache
    from mesh_b200.ops.draft import draft_attention
    B, H, S, hd, T, G = 5, 8, 240000 // (bits // 8) , 256, 10, 4
    g = _gen(5)
    k = torch.zeros((B, H, S, hd), dtype=torch.int8 if bits == 8 else BF16, device=DEV)
    scales = [torch.zeros((B, H, S), device=DEV) for _ in range(2)] if bits == 8 else []
    c = KVCache(k, torch.zeros_like(k), *scales)
    x, y, q = _randn(B, T, H, hd, g=g), _randn(B, T, H, hd, g=g), _randn(B, T, G * H, hd, g=g)
    pos = _i32([S - T] * B)
    c.append(x, y, pos)
    near = KVCache(*(t[:, :, S - 2 * T:].contiguous() for t in (c.k, c.v, *scales)))
    got = draft_attention(q, c, pos, window=T, splits=64)
    want = _attend64(q, near, _i32([T] * B), None, None, T, hd ** -0.5)
    _check(got, want, bits, 2 * T, hd)


def test_a_sequence_without_keys_between_others_with_infinite_values():
    """Contexts that fill the cache and a window of one: nothing to see.  Eight of them between two sequences whose values are not finite."""
    from mesh_b200.ops.draft import draft_attention
    g = _gen(14)
    B, H, S, hd, G = 9, 1, 128, 64, 40
    cache = _cache(B, H, S, hd, 16, g)
    pos = _i32([100] + [S] * 7 + [100])
    cache.v[0, 0, 100, 7], cache.v[8, 0, 100, 9] = math.inf, -math.inf
    q = _randn(B, 1, G, hd, g=g)
    for _ in range(20):
        got = draft_attention(q, cache, pos, window=1, splits=1)
        assert not got[1:8].any()
        for b in (0, 8):                                                  # a node that sees itself alone
            assert _same(got[b, 0], cache.v[b, 0, 100].expand(G, hd)), b


def test_many_rows_on_two_streams_and_in_a_graph():
    """Calls with scratch memory of their own: two streams at once, and a captured call beside eager ones."""
    from mesh_b200.ops.draft import draft_attention
    g = _gen(13)
    cache = _cache(2, 2, 9000, 128, 8, g)
    qs = [_randn(2, 16, 8, 128, g=g) for _ in range(2)]
    pos = _i32([8900, 5000])
    want = [draft_attention(q, cache, pos) for q in qs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = draft_attention(qs[0], cache, pos)
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        graph.replay()
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(draft_attention(qs[i], cache, pos))
    torch.cuda.synchronize()
    assert _same(kept, want[0])
    for i in range(2):
        assert all(_same(x, want[i]) for x in got[i])


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("bits", [8, 16])
def test_strides_of_dimensions_of_one_do_not_matter(bits, T):
    from mesh_b200.ops.draft import draft_attention
    g = _gen(15)
    B, S, hd = (1, 90, 64) if T == 1 else (2, 90, 64)
    cache = _cache(B, 1, S, hd, bits, g)
    pos = _i32([40, 13][:B])
    room, want = torch.zeros(16384, dtype=BF16, device=DEV), _randn(B, T, 1, hd, g=g)
    q = room.as_strided((B, T, 1, hd), (7001, 71, 5, 1))
    q.copy_(want)
    out = torch.zeros(16384, dtype=BF16, device=DEV).as_strided((B, T, 1, hd), (7001 if B == 1 else 7002, 71 if T == 1 else 72, 5, 1))
    draft_attention(q, cache, pos, out=out, splits=1)
    _check(out, _attend64(want, cache, pos, None, None, 0, hd ** -0.5), bits, S, hd)


@pytest.mark.parametrize("T,splits", [(3, 0), (3, 5), (40, 0), (40, 7)])
def test_attention_over_its_own_queries(T, splits):
    """``out`` may be ``q``; sequences and tokens may lie in either order."""
    from mesh_b200.ops.draft import draft_attention
    g = _gen(16)
    cache = _cache(3, 2, 700, 128, 8, g)
    q = _randn(T, 3, 8, 128, g=g).transpose(0, 1)
    pos = _i32([640, 100, 3])
    want = draft_attention(q.contiguous(), cache, pos, splits=splits)
    assert draft_attention(q, cache, pos, out=q, splits=splits) is q and _same(q, want)


# ------------------------------------------------------------------------------------------------------------ rows of the cache
@pytest.mark.parametrize("hd,T", [(128, 9001), (64, 17011), (256, 4099)])
def test_reading_many_rows(hd, T):
    """Enough 8-bit rows for two of them a thread, an odd number of CTAs of one, counts that end anywhere."""
    from mesh_b200.ops.cache import KVCache
    g = _gen(hd)
    B, H, S = 3, 5, T + 100
    k, v = (torch.randint(-127, 128, (B, H, S, hd), generator=g, device=DEV).to(torch.int8) for _ in range(2))
    ks, vs = (torch.rand((B, H, S), generator=g, device=DEV) for _ in range(2))
    c = KVCache(k, v, ks, vs)
    start, counts = _i32([0, 37, 101]), _i32([T, T - 1234, T])
    assert B * T * H >= 4096 * (256 // (hd // 8))                         # rows of 4096 CTAs, one a thread
    for n in (counts, None):
        for got, full in zip(c.read(start, T, n), c.dequantize()):
            for b in range(B):
                s, m = int(start[b]), T if n is None else int(n[b])
                there = min(m, S - s)
                assert _same(got[b, :there], full[b, :, s:s + there].transpose(0, 1).to(BF16))
                assert not got[b, there:].any()


# ------------------------------------------------------------------------------------------------------------ logits
def test_logits_refuse_an_output_that_meets_them():
    from mesh_b200.ops.logits import constrain_logits
    room = torch.randn(4, 300, device=DEV)
    x = room[:, :128]
    for out in (room[:, 1:129], room[:, 127:255], room.view(-1)[64:64 + 512].view(4, 128), room.view(-1)[:512].view(4, 128)):
        with pytest.raises(ValueError, match="apart"):
            constrain_logits(x, out=out)
    with pytest.raises(ValueError, match="apart"):
        constrain_logits(x[:1], out=room[:1, 8:136])
    was = room.clone()
    assert _same(constrain_logits(x, out=room[:, 128:256]), was[:, :128]) and _same(constrain_logits(x, out=x), was[:, :128])
    assert _same(constrain_logits(x[:1], out=x[:1].as_strided((1, 128), (999, 1))), was[:1, :128])
    assert _same(room[:, :128], was[:, :128]) and _same(room[:, 256:], was[:, 256:])
    tok = torch.zeros(4, dtype=torch.int32, device=DEV)
    for offset in (-1, 2**31 - 128, 2**31, 2**40):
        with pytest.raises(ValueError, match="ids"):
            constrain_logits(x, tokens=tok, vocab_offset=offset)
    last = 2**31 - 1 - 128
    h = torch.full((4, 1), last + 127, dtype=torch.int32, device=DEV)
    constrain_logits(x, tokens=tok, vocab_offset=last, history=h, presence=torch.full((4,), -100.0, device=DEV))
    assert tok.tolist() == [last + 127] * 4


# ------------------------------------------------------------------------------------------------------------ graphs
_FIRST = """
import torch
from mesh_b200.ops.cache import CacheGroup, KVCache
from mesh_b200.ops.draft import draft_attention
from mesh_b200.ops.logits import constrain_logits
def make(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").bfloat16()
    return r(2, 40, 8, 128), r(2, 40, 2, 128), r(2, 40, 2, 128), torch.randn((2, 262144), generator=g, device="cuda")
caches = [KVCache.empty(2, 2, 900, 128), KVCache.empty(2, 2, 20000, 128, bits=16)]
pos, tok = torch.tensor([700, 30], dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
path, h = torch.tensor([[0, 3, 2]] * 2, dtype=torch.int32, device="cuda"), torch.arange(5000, dtype=torch.int32, device="cuda")[None].expand(2, -1)
one = torch.ones(2, device="cuda")
def step(q, k, v, x):
    out = []
    for c in caches:
        c.append(k, v, pos)
        out += [draft_attention(q, c, pos), draft_attention(q[:, :2], c, pos), *c.read(pos, 40)]
        CacheGroup([c]).keep(pos, path)
    return out + [constrain_logits(x, history=h, presence=one, out=torch.empty_like(x), tokens=tok)]
x = make(1)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step(*x)
for a, b in zip(x, make(2)):
    a.copy_(b)
graph.replay()
kept = [t.clone() for t in got] + [tok.clone()]
want = step(*make(2)) + [tok]
assert all(torch.equal(a, b) for a, b in zip(kept, want))
print("the same")
"""


def test_the_first_calls_of_a_process_are_captured():
    """Kernels are loaded and configured, and the device is asked what it can run, while a stream is being captured."""
    import subprocess
    import sys
    from pathlib import Path
    r = subprocess.run([sys.executable, "-c", _FIRST], capture_output=True, text=True, timeout=300, cwd=Path(__file__).resolve().parent.parent)
    assert r.returncode == 0 and "the same" in r.stdout, r.stderr[-2000:]
