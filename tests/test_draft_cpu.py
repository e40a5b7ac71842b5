"""What the operators for drafted tokens refuse, and the helpers that run on the host."""
import pytest
import torch

from mesh_b200.ops.cache import CacheGroup, KVCache
from mesh_b200.ops.draft import draft_attention, tree_depth, tree_visible
from mesh_b200.ops.logits import constrain_logits

BF16 = torch.bfloat16


def _cache(B=2, H=2, S=32, hd=64, bits=8):
    return KVCache.empty(B, H, S, hd, bits=bits, device="cpu")


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def test_tree_words_and_depths():
    #   0 - 1 - 3 - 4      2 is 0's second child, 5 stands alone
    #     \ 2
    vis = tree_visible([[-1, 0, 0, 1, 3, -1], [-1, 0, 1, 2, 3, 4]])
    assert vis[0].tolist() == [0b1, 0b11, 0b101, 0b1011, 0b11011, 0b100000]
    assert vis[1].tolist() == [1, 3, 7, 15, 31, 63]
    assert tree_depth(vis).tolist() == [[0, 1, 1, 2, 3, 0], [0, 1, 2, 3, 4, 5]]
    chain = tree_visible([list(range(-1, 63))])                # bit 63 is the sign
    assert chain.shape == (1, 64) and chain[0, 63].item() == -1 and tree_depth(chain)[0, 63].item() == 63
    assert tree_depth(torch.zeros(1, 3, dtype=torch.int64)).tolist() == [[0, 0, 0]]
    assert tree_visible(torch.tensor([[-1, 0]])).tolist() == [[1, 3]]
    assert tree_visible([]).shape[0] == 0


@pytest.mark.parametrize("parents", [[[0]], [[-1, 1]], [[-1] * 65]])
def test_tree_refusals(parents):
    with pytest.raises(ValueError):
        tree_visible(parents)


def test_cache_refusals():
    k = torch.zeros(2, 2, 32, 64, dtype=torch.int8)
    s = torch.zeros(2, 2, 32)
    KVCache(k, k.clone(), s, s.clone())
    for bad in ((k, k[:1], s, s), (k, k.float(), s, s), (k, k, None, s), (k, k, s[:, :1], s), (k, k, s.double(), s), (k.transpose(0, 1), k, s, s),
                (k.float(), k.float()), (k.to(BF16), k.to(BF16), s, s), (k[..., :48].contiguous(), k[..., :48].contiguous(), s, s),
                (k[:, :0], k[:, :0], s[:, :0], s[:, :0]), (k[0], k[0], s, s)):
        with pytest.raises(ValueError):
            KVCache(*bad)
    with pytest.raises(ValueError):
        KVCache.empty(1, 1, 8, 64, bits=4, device="cpu")


def test_append_and_read_refusals():
    c = _cache()
    x, pos = torch.zeros(2, 3, 2, 64, dtype=BF16), _i32(0, 1)
    for k, v in ((x.float(), x), (x, x[:, :2]), (x[:1], x[:1]), (x[..., :32], x[..., :32]), (x.transpose(2, 3).contiguous().transpose(2, 3), x), (x[0], x[0])):
        with pytest.raises(ValueError):
            c.append(k, v, pos)
    for p, n in ((pos.long(), None), (_i32(0), None), (pos, _i32(1)), (pos, pos.float()), (torch.zeros(4, dtype=torch.int32)[::2], None)):
        with pytest.raises(ValueError):
            c.append(x, x, p, n)
        with pytest.raises(ValueError):
            c.read(p, 3, n)
    with pytest.raises(ValueError):
        c.read(pos, -1)
    with pytest.raises(ValueError, match="GPU"):
        c.append(x, x, pos)
    c.append(x[:, :0], x[:, :0], pos)                           # nothing to do
    assert c.read(pos, 0)[0].shape == (2, 0, 2, 64)


def test_keep_refusals():
    with pytest.raises(ValueError):
        CacheGroup([])
    with pytest.raises(ValueError):
        CacheGroup([_cache(), _cache(S=33)])
    with pytest.raises(ValueError):
        CacheGroup([_cache(), _cache(bits=16)])
    g = CacheGroup([_cache(), _cache()])
    pos = _i32(0, 1)
    for path, n in ((torch.zeros(2, 65, dtype=torch.int32), None), (torch.zeros(2, 3), None), (torch.zeros(1, 3, dtype=torch.int32), None),
                    (torch.zeros(2, 3, dtype=torch.int32), _i32(1)), (torch.zeros(3, dtype=torch.int32), None)):
        with pytest.raises(ValueError):
            g.keep(pos, path, n)
    with pytest.raises(ValueError, match="GPU"):
        g.keep(pos, torch.zeros(2, 3, dtype=torch.int32))


def test_attention_refusals():
    c, pos = _cache(), _i32(0, 1)
    q = torch.zeros(2, 3, 4, 64, dtype=BF16)
    ok = dict(counts=None, visible=None)
    for args in (dict(q=q.float()), dict(q=q[:1]), dict(q=q[..., :32]), dict(q=q[:, :, :3]), dict(q=q[:, :, :0]), dict(q=torch.zeros(2, 65, 4, 64, dtype=BF16)),
                 dict(q=q[0]), dict(q=torch.zeros(2, 3, 8, 64, dtype=BF16)[:, :, ::2]), dict(pos=pos.long()), dict(pos=_i32(0)),
                 dict(counts=_i32(1)), dict(visible=torch.zeros(2, 3, dtype=torch.int32)), dict(visible=torch.zeros(2, 4, dtype=torch.int64)),
                 dict(visible=torch.zeros(3, 2, dtype=torch.int64).t()), dict(window=2), dict(window=-1), dict(scale=0.0), dict(scale=float("nan")),
                 dict(out=q.float()), dict(out=q[:, :2])):
        call = {**dict(q=q, pos=pos), **ok, **args}
        with pytest.raises(ValueError):
            draft_attention(call.pop("q"), c, call.pop("pos"), **call)
    with pytest.raises(ValueError, match="GPU"):
        draft_attention(q, c, pos, window=3)
    assert draft_attention(q[:, :0], c, pos).shape == (2, 0, 4, 64)


def test_logits_refuse_the_host():
    with pytest.raises(ValueError, match="GPU"):
        constrain_logits(torch.zeros(1, 8), tokens=torch.zeros(1, dtype=torch.int32))
