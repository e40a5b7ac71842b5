"""Operators for drafted tokens at the edges of what their documentation allows, beside ``test_draft_gpu``: the kernel for many query
rows with everything that is hidden, absent or unaligned, a cancelled pass, large lists."""
import math

import pytest
import torch

from test_draft_gpu import BF16, DEV, _attend64, _cache, _check, _gen, _i32, _randn, _same, _words

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
