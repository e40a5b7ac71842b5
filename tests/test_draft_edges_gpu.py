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
