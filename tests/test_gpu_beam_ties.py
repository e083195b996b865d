"""GPU: equal scores go to the lower (beam, token), however the logits are divided among blocks.

The scores stand at -3,000, as after a long answer, where one fp32 step is 2^-12: logits closer than that share a score.  The
logits' upper part lies in clusters whose scores are whole steps, to within a few hundredths of one, so that the rounded scores
are known whatever the last bits of a logsumexp are."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -12


def _center(x, at, off):
    """Sets x[at] = base + off (x: 64-bit logits of one beam) with a base that makes base's log-softmax a whole number of steps;
    returns the log-softmax of the tokens at `at`, in steps."""
    base = 1.2
    for _ in range(200):
        x[at] = (base + off).float().double()
        score = (base - float(torch.logsumexp(x, 0))) / STEP
        base -= (score - round(score)) * STEP * 0.7
    exact = (x[at] - torch.logsumexp(x, 0)) / STEP
    assert float((exact - exact.round()).abs().max()) < 0.1
    return exact.round().long()


def _clusters(groups, beams, vocab, per, gen):
    """Logits and scores, and each candidate's score in steps (64-bit whole numbers, lowest: below every cluster)."""
    logits = torch.empty(groups, beams, vocab, dtype=torch.float32)
    steps = torch.full((groups, beams, vocab), -10 ** 9, dtype=torch.int64)
    for g in range(groups):
        for k in range(beams):
            x = (2 * torch.rand(vocab, generator=gen, dtype=torch.float64) - 1).float().double()
            at = torch.randperm(vocab, generator=gen)[:per]
            level = torch.randint(0, 3, (per,), generator=gen)
            off = -4 * level * STEP + 0.02 * STEP * (2 * torch.rand(per, generator=gen, dtype=torch.float64) - 1)
            steps[g, k, at] = _center(x, at, off) + round(-3000 / STEP)
            logits[g, k] = x.float()
    return logits, torch.full((groups, beams), -3000.0), steps


def _want(steps, beams):
    """(tokens, parents) in the order of falling score, then rising flat index."""
    g, k, v = steps.shape
    flat = steps.view(g, k * v)
    key = flat * (1 << 24) - torch.arange(k * v)
    best = key.topk(beams, 1).indices
    return best % v, best // v


@pytest.mark.parametrize("groups,beams,vocab,per", [(3, 1, 5000, 40), (2, 4, 20001, 300), (1, 8, 70001, 3000), (2, 32, 9000, 400),
                                                    (40, 8, 20001, 500), (1, 3, 151936, 20), (4, 16, 8192, 2000)])
def test_scores_that_round_together(groups, beams, vocab, per):
    from vault_b200 import beam_select
    gen = torch.Generator().manual_seed(vocab + beams)
    logits, run, steps = _clusters(groups, beams, vocab, per, gen)
    tokens, parents, best, _ = (t.cpu() for t in beam_select(logits.cuda(), run.cuda()))
    want_t, want_p = _want(steps, beams)
    assert torch.equal(tokens.long(), want_t) and torch.equal(parents.long(), want_p)
    flat = steps.view(groups, -1).gather(1, want_p * vocab + want_t)
    assert torch.equal(best.double(), flat.double() * STEP)


@pytest.mark.parametrize("gap", [1, 5000, 100000])
def test_the_lower_token_has_the_smaller_logit(gap):
    """Two tokens of one beam, the later one larger by a hundredth of a step of the score."""
    from vault_b200 import beam_select
    x = (2 * torch.rand(151936, generator=torch.Generator().manual_seed(gap), dtype=torch.float64) - 1).float().double()
    _center(x, torch.tensor([700, 700 + gap]), torch.tensor([0.0, 0.01 * STEP], dtype=torch.float64))
    assert float(x[700]) < float(x[700 + gap])
    tokens, _, _, _ = beam_select(x.float().view(1, 1, -1).cuda(), torch.full((1, 1), -3000.0, device="cuda"))
    assert int(tokens) == 700


def test_a_finished_beam_among_ties():
    """A finished beam's only continuation takes its place by its flat index, between the ties of lower and higher beams."""
    from vault_b200 import beam_select
    gen = torch.Generator().manual_seed(9)
    logits, run, steps = _clusters(1, 4, 9000, 2, gen)
    finished = torch.zeros(1, 4, dtype=torch.uint8)
    finished[0, 2] = 1
    steps[0, 2] = -10 ** 9
    level = int(steps[0, [0, 1, 3]].flatten().topk(4).values[3])   # the score that the last place is worth
    run[0, 2] = level * STEP
    steps[0, 2, 5] = level
    tokens, parents, best, done = (t.cpu() for t in beam_select(logits.cuda(), run.cuda(), finished.cuda(), eos_id=5))
    want_t, want_p = _want(steps, 4)
    assert torch.equal(tokens.long(), want_t) and torch.equal(parents.long(), want_p)
    assert torch.equal(done.bool(), (parents == 2) | (tokens == 5))


def test_a_group_decides_alone():
    """The same group by itself and among others, where its logits are divided into other slices."""
    from vault_b200 import beam_select
    gen = torch.Generator().manual_seed(11)
    logits, run, _ = _clusters(1, 8, 70001, 2000, gen)
    alone = beam_select(logits.cuda(), run.cuda())
    many = beam_select(logits.expand(30, -1, -1).contiguous().cuda(), run.expand(30, -1).contiguous().cuda())
    for a, m in zip(alone, many):
        assert torch.equal(a.expand(30, -1), m)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_16_bit_logits(dtype):
    """Equal 16-bit logits, and different ones that share a score, over strided rows."""
    from vault_b200 import beam_select
    gen = torch.Generator().manual_seed(13)
    wide = torch.randint(0, 3, (2, 5, 30100), generator=gen).to(dtype)
    x = wide[:, :, 3:30001]
    run = torch.full((2, 5), -3.0e8)                 # a step is 32: every logit of a beam shares a score
    tokens, parents, best, _ = (t.cpu() for t in beam_select(x.cuda(), run.cuda()))
    assert tokens.tolist() == [[0, 1, 2, 3, 4]] * 2 and not bool(parents.any()) and bool((best == -3.0e8).all())
    hidden = x.clone()
    hidden[:, :, :20000] = -math.inf
    hidden[0, 0] = math.nan
    tokens, parents, _, _ = (t.cpu() for t in beam_select(hidden.cuda(), run.cuda()))
    assert tokens.tolist() == [list(range(20000, 20005))] * 2 and parents.tolist() == [[1] * 5, [0] * 5]
