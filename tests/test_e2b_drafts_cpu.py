"""The decoder's bookkeeping of drafts without a GPU: which branch is accepted, and where the caches end."""
import pytest
import torch

from mesh_b200.models.e2b import E2BConfig, E2BDecoder


class _Kept:
    def __init__(self):
        self.calls = []

    def keep(self, pos, path, counts):
        self.calls.append((pos.tolist(), path.tolist(), counts.tolist()))


def _decoder(pos, max_seq=96):
    """A decoder with its counters alone; the caches note what is kept."""
    m = E2BDecoder.__new__(E2BDecoder)
    m.cfg, m.dev, m._group = E2BConfig(max_seq=max_seq), torch.device("cpu"), _Kept()
    m.pos = torch.tensor(pos, dtype=torch.int32)
    m.tok = torch.full((len(pos),), 3, dtype=torch.int32)
    m.filled = 0
    return m


def _i32(v):
    return torch.tensor(v, dtype=torch.int32)


def _matching(B, T):
    """Drafts that the model all chooses: token t + 10 after node t."""
    return _i32([[9 + t for t in range(T)]] * B), _i32([[10 + t for t in range(T)]] * B)


@pytest.mark.parametrize("pos,taken", [(80, 16), (81, 15), (90, 6), (95, 1)])
def test_a_branch_ends_with_the_caches(pos, taken):
    m = _decoder([pos, 10])
    new = m.accept(*_matching(2, 16))
    assert [len(t) for t in new] == [taken, 16] and m.pos.tolist() == [pos + taken, 26]
    assert new[0] == [10 + t for t in range(taken)] and m.tok.tolist() == [9 + taken, 25]
    (before, path, counts), = m._group.calls
    assert counts == [taken, 16] and path[0] == list(range(taken)) + [-1] * (16 - taken)
    assert m.filled == max(pos + taken, 26)


def test_full_caches_are_refused_before_anything_moves():
    m = _decoder([5, 96])
    with pytest.raises(ValueError, match="full"):
        m.accept(*_matching(2, 4))
    assert m.pos.tolist() == [5, 96] and m.tok.tolist() == [3, 3] and not m._group.calls
    new = m.accept(*_matching(2, 4), counts=_i32([4, 0]))           # the full sequence rests
    assert new == [[10, 11, 12, 13], []] and m.pos.tolist() == [9, 96] and m.tok.tolist() == [13, 3]


def test_decoding_past_the_caches_is_refused():
    m = _decoder([90, 70])
    m.filled = 90
    m._need(6, "decode")
    assert m.filled == 96
    with pytest.raises(ValueError, match="decode: 7 more tokens do not fit"):
        m._need(7, "decode")
    assert m.filled == 90                                           # as the positions say
    m.pos.fill_(20)                                                 # set back by hand
    m.filled = 96
    m._need(3, "decode")
    assert m.filled == 23
    m.graph = object()
    with pytest.raises(ValueError, match="do not fit"):
        m.decode(77)


def test_a_draft_that_is_no_token_is_not_accepted():
    """-1 pads a tree and says that no token was allowed: the two are not the same token."""
    m = _decoder([4])
    with pytest.raises(ValueError, match="no token was allowed"):
        m.accept(_i32([[5, -1]]), _i32([[-1, 7]]))
    assert m.pos.tolist() == [4] and not m._group.calls
    assert m.accept(_i32([[5, -1, 6]]), _i32([[6, 7, 8]]), [[-1, 0, 0]]) == [[6, 8]]


def test_choices_of_other_drafts_are_refused():
    m = _decoder([4, 5])
    drafts, chosen = _matching(2, 6)
    for bad in (chosen[:, :5], chosen[:1], chosen.reshape(-1), torch.cat([chosen, chosen])):
        with pytest.raises(ValueError, match="chosen"):
            m.accept(drafts, bad)
    assert m.pos.tolist() == [4, 5] and not m._group.calls
