"""The decoder's drafts where its caches end."""
import pytest
import torch

from test_e2b_drafts_gpu import PARENTS, TOL, _model
from test_e2b_gpu import _ref_logits, _rel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("n", [3, 12])                              # the decode step's kernels; the products of the prompt
def test_drafts_at_the_end_of_the_caches(bits, n):
    """The last slots, a tree that does not fit, a full cache: what fits is computed as with as many drafts by ``counts``, -1 is chosen after
    the others, and no row of the caches but the ones that are there changes."""
    from mesh_b200.ops.draft import tree_visible
    from mesh_b200.utils.status import check_status
    B, S = 2, 96
    m, _, g = _model(B, "bf16", bits, 20)
    drafts = torch.randint(0, m.cfg.vocab, (B, n), generator=g, dtype=torch.int32).cuda()
    visible = tree_visible([PARENTS[:n]] * B).cuda()
    for pos in ((S - n, S - n - 1), (S - n + 1, 40), (S - 1, S), (S, S)):
        m.pos.copy_(torch.tensor(pos, dtype=torch.int32))
        room = [min(n, S - p) for p in pos]
        chosen = m.draft_step(drafts, visible)
        rows = [[c.clone() for c in (L["cache"].k, L["cache"].v)] for L in m.layers]
        fewer = m.draft_step(drafts, visible, torch.tensor(room, dtype=torch.int32, device="cuda"))
        for b in range(B):
            assert torch.equal(chosen[b, :room[b]], fewer[b, :room[b]]) and (chosen[b, :room[b]] >= 0).all()
            assert (chosen[b, room[b]:] == -1).all()
        assert all(torch.equal(a, b) for L, was in zip(m.layers, rows) for a, b in zip((L["cache"].k, L["cache"].v), was))
        assert m.pos.tolist() == list(pos)
    with pytest.raises(ValueError, match="full"):
        m.accept(drafts, chosen)
    for bad in (torch.zeros(B, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32)):
        with pytest.raises(ValueError, match="counts"):
            m.draft_step(drafts, visible, bad)
    check_status()


@pytest.mark.parametrize("bits", [8, 16])
def test_a_decoder_runs_to_the_end_of_its_caches_and_no_further(bits):
    """Greedy drafts up to the last slot: the accepted branch ends there, what follows is refused, and the logits of the last token are the
    plain model's."""
    from mesh_b200.utils.status import check_status
    B, T, S, n = 1, 88, 96, 6
    m, prompt, _ = _model(B, "bf16", bits, T)
    m.capture("graph")
    m.pos.fill_(T)
    line = torch.cat([prompt, m.tok[:, None]], 1)
    while int(m.pos[0]) < S:
        drafts = torch.zeros((B, n), dtype=torch.int32, device="cuda")
        drafts[:, 0] = m.tok
        for t in range(1, n):                                       # what the model chooses, node by node
            drafts[:, t] = m.draft_step(drafts)[:, t - 1]
        pos = int(m.pos[0])
        new = m.accept(drafts, m.draft_step(drafts))
        assert len(new[0]) == min(n, S - pos) and int(m.pos[0]) == pos + len(new[0])
        line = torch.cat([line, torch.tensor(new, dtype=torch.int32, device="cuda")], 1)
    assert line.shape[1] == S + 1                                   # the last token has no slot
    ref = _ref_logits(m, line[:, :S])
    assert (ref.amax(-1) - ref.gather(1, line[:, S:].long())[:, 0] <= 2 * TOL[bits] * ref.abs().amax(-1)).all()
    for call in (lambda: m.decode(1), lambda: m.capture("graph"), lambda: m.accept(drafts, drafts)):
        with pytest.raises(ValueError, match="do not fit|full"):
            call()
    m.pos.fill_(S - 2)                                              # set back: the two last tokens again
    m.tok.copy_(line[:, S - 2])
    m.decode(2)
    assert _rel(m.logits, ref) < TOL[bits] and m.pos.tolist() == [S]
    with pytest.raises(ValueError, match="do not fit"):
        m.decode(1)
    check_status()


@pytest.mark.parametrize("quant", ["bf16", "w4", "w8"])
def test_more_than_eight_rows_choose_from_fp32_logits(quant):
    """Two tokens are raised above all others, the one of the higher id by 2^-11 of its logit more, less than half a step of bf16 (2^-9 to 2^-8): it is
    chosen in every row."""
    B, n = 2, 12
    m, _, g = _model(B, quant, 16, 20)
    drafts = torch.randint(0, m.cfg.vocab, (B, n), generator=g, dtype=torch.int32).cuda()
    logits = torch.empty((B * n, m.cfg.vocab), device="cuda")
    plain = m.draft_step(drafts, constraints=dict(out=logits))
    assert torch.equal(plain.view(-1).long(), logits.argmax(-1))
    assert not torch.equal(logits, logits.bfloat16().float())
    low, high = 7, 300
    l = logits[:, [low, high]].double()
    up = 2.0 ** -11 * l.abs().amax(-1)
    # sums of magnitudes below 256 are off by at most 2^-17 in fp32, and so are the biases
    assert l.abs().max() + 128 < 256 and up.min() > 4 * 2.0 ** -17
    bias = torch.stack([128 - l[:, 0], 128 - l[:, 1] + up], 1).float()
    ids = torch.tensor([[low, high]], dtype=torch.int32, device="cuda").expand(B * n, -1)
    chosen = m.draft_step(drafts, constraints=dict(bias_ids=ids.contiguous(), bias=bias))
    assert (chosen == high).all()


def test_more_drafts_than_the_window_are_refused_before_a_row_is_written():
    m, _, g = _model(1, "bf16", 8, 20)
    rows = [L["cache"].k.clone() for L in m.layers]
    with pytest.raises(ValueError, match="window of 16"):
        m.draft_step(torch.zeros((1, 17), dtype=torch.int32, device="cuda"))
    assert all(torch.equal(L["cache"].k, was) for L, was in zip(m.layers, rows))
    m.draft_step(torch.zeros((1, 16), dtype=torch.int32, device="cuda"))
