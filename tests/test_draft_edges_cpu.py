"""What the operators for drafted tokens take and refuse, beside ``test_draft_cpu``."""
import random

import pytest
import torch

from test_draft_cpu import BF16, _cache, _i32

from mesh_b200.ops.cache import CacheGroup, KVCache
from mesh_b200.ops.draft import draft_attention


def test_strides_of_dimensions_of_one_do_not_matter():
    """A single head, token or sequence has no neighbour for its stride to lead to: refused for want of a GPU alone."""
    c = _cache(B=1, H=1)
    x = torch.zeros(4096, dtype=BF16)
    for strides in ((777, 333, 111, 1), (64, 64, 64, 1), (0, 0, 0, 1)):
        q = x.as_strided((1, 1, 1, 64), strides)
        with pytest.raises(ValueError, match="GPU"):
            draft_attention(q, c, _i32(3), out=q)
    two = _cache(B=2, H=1)
    q = x.as_strided((2, 3, 1, 64), (1000, 200, 7, 1))
    with pytest.raises(ValueError, match="GPU"):
        draft_attention(q, two, _i32(3, 4), out=q.clone(memory_format=torch.preserve_format))
    with pytest.raises(ValueError, match="dense"):
        draft_attention(x.as_strided((2, 3, 2, 64), (1000, 200, 100, 1)), two, _i32(3, 4))


def test_a_group_moves_every_row_once():
    """The same cache twice, one tensor for keys and values, scales of two caches in one: their rows would be moved by two CTAs at once."""
    a, b = _cache(), _cache()
    CacheGroup([a, b])
    parts = torch.zeros(3, 2, 2, 32, 64, dtype=torch.int8)
    scales = torch.zeros(4, 2, 2, 32)
    CacheGroup([KVCache(parts[0], parts[1], scales[0], scales[1])])                     # neighbours in one tensor
    for group in ([a, b, a], [a, KVCache(a.k, a.v, a.k_scale, a.v_scale)], [KVCache(parts[0], parts[0], scales[0], scales[1])],
                  [KVCache(parts[0], parts[1], scales[0], scales[0])], [a, KVCache(b.k, b.v, a.v_scale, b.v_scale)],
                  [KVCache(parts[0], parts[1], scales[0], scales[1]), KVCache(parts[1], parts[2], scales[2], scales[3])]):
        with pytest.raises(ValueError, match="share memory"):
            CacheGroup(group)
    x = torch.zeros(2 * 2 * 32 * 64 + 64, dtype=BF16)
    with pytest.raises(ValueError, match="share memory"):
        CacheGroup([KVCache(x[:-64].view(2, 2, 32, 64), x[64:].view(2, 2, 32, 64))])
    CacheGroup([_cache(B=0), _cache(B=0)])


def test_a_cache_of_one_tensor_is_not_written():
    """Keys and values in the same memory may be attended to and read; appended, one would overwrite the other."""
    k, s = torch.zeros(2, 2, 32, 64, dtype=torch.int8), torch.zeros(2, 2, 2, 32)
    x, pos = torch.zeros(2, 3, 2, 64, dtype=BF16), _i32(0, 1)
    for c in (KVCache(k, k, s[0], s[1]), KVCache(k, k.clone(), s[0], s[0]), KVCache(k.to(BF16), k.to(BF16)[:]), KVCache(*[k.to(BF16)] * 2)):
        with pytest.raises(ValueError, match="share memory|GPU") as e:
            c.append(x, x, pos)
        assert ("share" in str(e.value)) == (c.k.data_ptr() == c.v.data_ptr() or c.bits == 8)
        with pytest.raises(ValueError, match="GPU"):
            draft_attention(x, c, pos)


def test_attention_refuses_an_output_whose_rows_overlap():
    c, pos, row = _cache(), _i32(0, 1), 4 * 64
    q, x = torch.zeros(2, 3, 4, 64, dtype=BF16), torch.zeros(4096, dtype=BF16)
    for sb, st in ((0, row), (3 * row, 0), (row, row), (2 * row, row), (row, row - 64), (3 * row - 2, row), (row, 2 * row - 2), (0, 0)):
        with pytest.raises(ValueError, match="overlap"):
            draft_attention(q, c, pos, out=x.as_strided(q.shape, (sb, st, 64, 1)))
    for sb, st in ((3 * row, row), (row, 2 * row), (5 * row, row + 8), (row + 2, 2 * row + 4)):
        out = x.as_strided(q.shape, (sb, st, 64, 1))
        with pytest.raises(ValueError, match="GPU"):
            draft_attention(q, c, pos, out=out)
        with pytest.raises(ValueError, match="GPU"):
            draft_attention(out, c, pos, out=out)
    with pytest.raises(ValueError, match="GPU"):
        draft_attention(x.as_strided(q.shape, (0, 0, 64, 1)), c, pos)                  # queries may be shared


def test_rows_of_two_matrices_that_meet():
    """Against the addresses themselves; matrices of unequal strides whose spans meet count as meeting."""
    from mesh_b200.ops.logits import _rows_meet
    x, rng, both = torch.zeros(400), random.Random(1), set()
    for _ in range(3000):
        R, V = rng.randint(0, 4), rng.randint(1, 20)
        lda, ldb = (rng.randint(V, 60) for _ in range(2))
        if rng.random() < 0.7:
            ldb = lda
        a, b = (x.as_strided((R, V), (ld, 1), rng.randint(0, 100)) for ld in (lda, ldb))
        if a.data_ptr() == b.data_ptr() and (lda == ldb or R <= 1):
            continue                                                                    # in place
        cells = [{(t.data_ptr() + 4 * (r * t.stride(0) + c)) for r in range(R) for c in range(V)} for t in (a, b)]
        meet = bool(cells[0] & cells[1])
        got = _rows_meet(a, b)
        assert got or not meet
        if R <= 1 or lda == ldb:
            assert got == meet
        both.add((got, meet))
    assert both >= {(True, True), (False, False)}
