"""E2B-class decoder with a cache of 8-bit codes, and with trees of drafts, against a plain fp32 model with the same weights."""
import pytest
import torch

from test_e2b_gpu import _ref_logits, _rel, _small_cfg, _solo_ctx

pytestmark = pytest.mark.gpu

# Of the largest logit: 0.06 with bf16 rows, as in the tests of the decoder.  In 8 bits an element of a row is off by a / 440 (root of the
# mean square of a step of a / 127 evenly filled), where the largest a of 128 normal values is 2.8 of their deviations: 0.0064 of
# the row's size for keys and as much for values, in each of 5 layers: 0.0064 sqrt(2 * 5) = 0.02, and half as much again.
TOL = {16: 0.06, 8: 0.09}
PARENTS = [-1, 0, 0, 1, 2, 2, 4, 5, 6, 3, 6, 10]                # the branch that is taken below: 0 2 4 6 10 11
BRANCH = [0, 2, 4, 6, 10, 11]


def _model(B, quant, bits, T, seed=3):
    from mesh_b200.models.e2b import E2BDecoder
    m = E2BDecoder(_small_cfg(), _solo_ctx(), B, quant, cache_bits=bits)
    g = torch.Generator().manual_seed(seed)
    prompt = torch.randint(0, m.cfg.vocab, (B, T), generator=g, dtype=torch.int32).cuda()
    m.prefill(prompt)
    return m, prompt, g


@pytest.mark.parametrize("quant,B", [("bf16", 2), ("w4", 3), ("w8", 1)])
def test_coded_cache_matches_reference(quant, B):
    from mesh_b200.utils.status import check_status
    T, steps = 24, 6
    m, prompt, _ = _model(B, quant, 8, T)
    assert _rel(m.logits, _ref_logits(m, prompt)) < 0.05            # the prompt attends to its rows before they are coded
    seq = torch.cat([prompt, m.tok[:, None]], 1)
    m.capture("graph")
    m.pos.fill_(T)
    m.tok.copy_(seq[:, -1])
    for _ in range(steps):
        m.decode(1)
        assert _rel(m.logits, _ref_logits(m, seq)) < TOL[8]
        seq = torch.cat([seq, m.tok[:, None]], 1)
    check_status()
    assert m.pos.tolist() == [T + steps] * B
    with pytest.raises(ValueError, match="step kernel"):
        m.capture("step")


def _paths(parents):
    out = []
    for t, p in enumerate(parents):
        out.append((out[p] if p >= 0 else []) + [t])
    return out


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("quant", ["bf16", "w4"])
@pytest.mark.parametrize("n", [1, 3, 12])                           # drafts: 2 * 3 rows of fp32 logits, 2 * 12 rows from the product
def test_tree_of_drafts_matches_reference(bits, quant, n):
    """The token chosen after every node is one whose logit in the plain model lies within the logits' own error of the best."""
    from mesh_b200.ops.draft import tree_visible
    from mesh_b200.utils.status import check_status
    B, T = 2, 24
    m, prompt, g = _model(B, quant, bits, T)
    drafts = torch.randint(0, m.cfg.vocab, (B, n), generator=g, dtype=torch.int32).cuda()
    drafts[:, 0] = m.tok
    pos = m.pos.clone()
    chosen = m.draft_step(drafts, tree_visible([PARENTS[:n]] * B).cuda())
    check_status()
    assert torch.equal(m.pos, pos) and torch.equal(m.tok, drafts[:, 0])
    for t, path in enumerate(_paths(PARENTS[:n])):
        ref = _ref_logits(m, torch.cat([prompt, drafts[:, path]], 1))
        best, got = ref.amax(-1), ref.gather(1, chosen[:, t:t + 1].long())[:, 0]
        assert ((best - got) <= 2 * TOL[bits] * ref.abs().amax(-1)).all(), t


@pytest.mark.parametrize("bits", [8, 16])
def test_accepted_branch_continues_as_if_decoded(bits):
    """A bias per row says which token is chosen, so the branch is known; after it has been accepted, with two sequences that accept
    different numbers, the decoder goes on as after the accepted tokens."""
    from mesh_b200.ops.draft import tree_visible
    from mesh_b200.utils.status import check_status
    B, T, n = 3, 24, len(PARENTS)
    m, prompt, g = _model(B, "bf16", bits, T)
    m.capture("graph")
    m.pos.fill_(T)
    drafts = torch.randint(1, m.cfg.vocab, (B, n), generator=g, dtype=torch.int32).cuda()
    drafts[:, 0] = m.tok
    drafts[:, 1] = drafts[:, 2]                                     # two children with one token: the first is taken
    want = torch.zeros((B, n), dtype=torch.int32, device="cuda")    # token 0 follows, which no draft is
    branches = [[0, 1, 3], BRANCH, [0]]
    drafts[1, 1] = 0                                                # ... but not here
    for b, br in enumerate(branches):
        for t, child in zip(br, br[1:]):
            want[b, t] = drafts[b, child]
    want[1, 0] = drafts[1, 2]
    counts = torch.tensor([n, n, 1], dtype=torch.int32, device="cuda")
    chosen = m.draft_step(drafts, tree_visible([PARENTS] * B).cuda(), counts,
                          dict(bias_ids=want.reshape(-1, 1), bias=torch.full((B * n, 1), 1e6, device="cuda")))
    for b, br in enumerate(branches):
        assert chosen[b, br].tolist() == want[b, br].tolist()
    new = m.accept(drafts, chosen, [PARENTS] * B, counts)
    assert new == [drafts[b, br[1:]].tolist() + [0] for b, br in enumerate(branches)]
    assert m.pos.tolist() == [T + len(br) for br in branches] and m.tok.tolist() == [0] * B
    seqs = [torch.cat([prompt[b], drafts[b, br], m.tok[b:b + 1]]) for b, br in enumerate(branches)]
    for _ in range(2):
        m.decode(1)
        for b in range(B):
            assert _rel(m.logits[b:b + 1], _ref_logits(m, seqs[b][None])) < TOL[bits]
            seqs[b] = torch.cat([seqs[b], m.tok[b:b + 1]])
    check_status()


def test_drafts_under_a_grammar_and_a_chain():
    from mesh_b200.utils.status import check_status
    B, T, n = 2, 20, 7
    m, _, g = _model(B, "bf16", 8, T)
    drafts = torch.randint(0, m.cfg.vocab, (B, n), generator=g, dtype=torch.int32).cuda()
    words = torch.zeros((B * n, m.cfg.vocab // 32), dtype=torch.int32, device="cuda")
    words[:, 5] = 1 << 9
    assert (m.draft_step(drafts, constraints=dict(allowed=words)) == 5 * 32 + 9).all()
    none = m.draft_step(drafts, constraints=dict(allowed=torch.zeros_like(words)))
    assert (none == -1).all()
    with pytest.raises(ValueError, match="no token was allowed"):
        m.accept(drafts, none)
    assert m.pos.tolist() == [T] * B
    some = m.draft_step(drafts, counts=torch.tensor([2, 0], dtype=torch.int32, device="cuda"))
    padded = drafts.clone()
    padded[0, 2:], padded[1] = -1, 2**31 - 1                        # what lies behind the counts may be anything
    again = m.draft_step(padded, counts=torch.tensor([2, 0], dtype=torch.int32, device="cuda"))
    assert torch.equal(some[0, :2], again[0, :2])
    chosen = m.draft_step(drafts)
    drafts[:, 1] = chosen[:, 0]
    new = m.accept(drafts, m.draft_step(drafts))
    assert all(len(t) >= 1 for t in new) and m.pos.tolist() == [T + len(t) for t in new] and m.tok.tolist() == [t[-1] for t in new]
    check_status()


def test_captured_step_of_drafts_follows_its_inputs():
    from mesh_b200.ops.draft import tree_visible
    from mesh_b200.utils.status import check_status
    B, T, n = 2, 24, len(PARENTS)
    m, _, g = _model(B, "w4", 8, T)
    drafts = torch.zeros((B, n), dtype=torch.int32, device="cuda")
    visible = tree_visible([PARENTS] * B).cuda()
    m.draft_step(drafts, visible)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chosen = m.draft_step(drafts, visible)
    for at in (T, T + 9, 1):
        drafts.copy_(torch.randint(0, m.cfg.vocab, (B, n), generator=g, dtype=torch.int32))
        m.pos.fill_(at)
        graph.replay()
        assert torch.equal(chosen, m.draft_step(drafts, visible))
    check_status()


def test_refusals():
    from mesh_b200.models.e2b import E2BDecoder
    with pytest.raises(ValueError, match="does not fit"):
        _model(1, "bf16", 8, 97)
    with pytest.raises(ValueError, match="cache_bits"):
        E2BDecoder(_small_cfg(), _solo_ctx(), 1, cache_bits=4)
    m, _, _ = _model(1, "bf16", 16, 8)
    for bad in (torch.zeros((1, 65), dtype=torch.int32, device="cuda"), torch.zeros((1, 0), dtype=torch.int32, device="cuda"),
                torch.zeros((2, 3), dtype=torch.int32, device="cuda"), torch.zeros((1, 3), device="cuda"), torch.zeros((1, 3), dtype=torch.int32)):
        with pytest.raises(ValueError, match="drafts"):
            m.draft_step(bad)
