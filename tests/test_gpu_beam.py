"""GPU: beam_select against log-softmax and a full sort in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

# fp32 log-softmax and sum: the running score, the logit and the logsumexp are each rounded near their size
TOL = 2.0 ** -20


def _candidates(logits, scores, finished, eos):
    """64-bit scores [groups, beams * vocab], -inf where there is no continuation."""
    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x)
    c = x - torch.logsumexp(x, -1, keepdim=True) + scores.double()[..., None]
    for g, k in finished.nonzero().tolist():
        c[g, k] = -math.inf
        if eos >= 0:
            c[g, k, eos] = scores[g, k].double()
    return torch.where(c.isnan() | c.isinf(), -math.inf, c).flatten(1)


def _check(logits, scores, finished, eos):
    from vault_b200 import beam_select
    tokens, parents, best, done = (t.cpu() for t in beam_select(logits.cuda(), scores.cuda(), finished.cuda(), eos))
    b, k, v = logits.shape
    cand = _candidates(logits, scores, finished, eos)
    want = cand.sort(1, descending=True).values
    tol = TOL * (logits.double().nan_to_num(0, 0, 0).abs().max() + scores.double().nan_to_num(0, 0, 0).abs().max() + 16)
    for g in range(b):
        chosen = set()
        for j in range(k):
            if j >= v * k or want[g, j] == -math.inf:
                assert (int(tokens[g, j]), int(parents[g, j]), float(best[g, j]), int(done[g, j])) == (max(eos, 0), j, -math.inf, 1)
                continue
            flat = int(parents[g, j]) * v + int(tokens[g, j])
            assert flat not in chosen
            chosen.add(flat)
            assert abs(float(cand[g, flat]) - float(want[g, j])) <= tol and abs(float(best[g, j]) - float(want[g, j])) <= tol
            assert int(done[g, j]) == int(bool(finished[g, int(parents[g, j])]) or int(tokens[g, j]) == eos)
            if j:
                assert best[g, j] <= best[g, j - 1]
                if best[g, j] == best[g, j - 1] and parents[g, j] == parents[g, j - 1] and \
                        logits[g, parents[g, j], tokens[g, j]] == logits[g, parents[g, j], tokens[g, j - 1]]:
                    assert tokens[g, j] > tokens[g, j - 1]


@pytest.mark.parametrize("groups,beams,vocab", [(1, 1, 1), (1, 4, 3), (2, 3, 7), (3, 2, 4096), (1, 8, 4097), (2, 16, 300), (1, 32, 9001),
                                               (5, 5, 12289), (1, 1, 151936), (2, 4, 151936)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_beam_select(groups, beams, vocab, dtype):
    g = torch.Generator().manual_seed(groups * beams + vocab)
    logits = (3 * torch.randn(groups, beams, vocab, generator=g)).to(dtype)
    scores = -5 * torch.rand(groups, beams, generator=g)
    finished = (torch.rand(groups, beams, generator=g) < 0.3).to(torch.uint8)
    _check(logits, scores, finished, eos=min(2, vocab - 1))
    _check(logits, scores, torch.zeros_like(finished), eos=-1)


def test_first_step_and_finished_beams():
    """Scores -inf: beams that do not exist yet; a group whose beams are all finished keeps them, in the order of their
    scores; finished beams without an eos id have no continuation."""
    logits = torch.randn(3, 4, 500, generator=torch.Generator().manual_seed(1))
    scores = torch.full((3, 4), -math.inf)
    scores[0, 0] = scores[2, 3] = 0.0
    scores[1] = torch.tensor([-3.0, -1.0, -2.0, -4.0])
    finished = torch.zeros(3, 4, dtype=torch.uint8)
    finished[1] = 1
    _check(logits, scores, finished, eos=7)
    _check(logits, scores, finished, eos=-1)


def test_ties_take_the_lower_index():
    """Equal logits everywhere, equal beams, a plateau wider than any buffer: the answer is the first indices."""
    from vault_b200 import beam_select
    flat = torch.zeros(2, 4, 10000)
    tokens, parents, best, _ = beam_select(flat.cuda(), torch.zeros(2, 4).cuda())
    assert tokens.cpu().tolist() == [[0, 1, 2, 3]] * 2 and parents.cpu().tolist() == [[0, 0, 0, 0]] * 2
    assert float((best.cpu() + math.log(10000)).abs().max()) <= 1e-5
    peak = torch.full((1, 3, 9000), -4.0)
    peak[:, :, 5000:8999] = 2.0
    peak[0, 1, 8999] = 3.0
    tokens, parents, _, _ = beam_select(peak.cuda(), torch.tensor([[0.0, 0.0, 0.0]]).cuda())
    assert tokens.cpu().tolist()[0][0] == 8999 and parents.cpu().tolist()[0][0] == 1
    assert tokens.cpu().tolist()[0][1:] == [5000, 5001] and parents.cpu().tolist()[0][1:] == [0, 0]
    ramp = torch.arange(20000.0)[None, None].repeat(1, 2, 1) / 1000
    for x in (ramp, ramp.flip(-1)):
        tokens, parents, _, _ = beam_select(x.cuda(), torch.tensor([[0.0, -1e-4]]).cuda())
        top = 19999 if x is ramp else 0
        assert tokens.cpu().tolist()[0] == [top, top] and parents.cpu().tolist()[0] == [0, 1]
    signed = torch.tensor([[[-0.0, 0.0, -1.0, 0.0]]])
    assert beam_select(signed.cuda(), torch.zeros(1, 1).cuda())[0].item() == 0


def test_masked_logits():
    """-inf and the type's lowest value hide tokens; NaN logits are skipped; a beam with an infinite logit or none finite has
    no continuation."""
    g = torch.Generator().manual_seed(3)
    logits = torch.randn(2, 3, 5000, generator=g)
    logits[:, :, 10:] = -math.inf
    logits[0, 1, 4] = math.nan
    logits[1, 0] = -math.inf
    logits[1, 1, 17] = math.inf
    _check(logits, torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.uint8), eos=3)
    low = torch.randn(1, 2, 5000, generator=g)
    low[:, :, 1:] = torch.finfo(torch.float32).min
    _check(low, torch.zeros(1, 2), torch.zeros(1, 2, dtype=torch.uint8), eos=3)
    _check(torch.full((1, 2, 50), math.nan), torch.zeros(1, 2), torch.zeros(1, 2, dtype=torch.uint8), eos=3)


def test_row_strides_and_streams():
    from vault_b200 import beam_select
    g = torch.Generator().manual_seed(4)
    wide = torch.randn(2, 3, 4111, generator=g).cuda()
    for lo, hi in ((0, 4096), (1, 4100), (3, 700)):
        view = wide[:, :, lo:hi]
        scores = torch.zeros(2, 3, device="cuda")
        want = beam_select(view.contiguous(), scores)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = beam_select(view, scores)
        side.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_beams_over_long_slices(dtype):
    """Enough beams that a slice has several steps, the last of them ragged; the best ones of a slice together in one
    thread's share, in rising and falling order; every slice of a wide group at the bound."""
    g = torch.Generator().manual_seed(5)
    groups, beams, vocab = 40, 32, 20001
    logits = (3 * torch.randn(groups, beams, vocab, generator=g)).to(dtype)
    logits[1] = torch.arange(vocab) / 1024
    logits[2] = torch.arange(vocab).flip(0) / 1024
    logits[3, :, 8192:8232] += 20
    logits[4, :, 256 * torch.arange(78)] += 20
    scores = -5 * torch.rand(groups, beams, generator=g)
    scores[5, 1:] = -math.inf
    finished = (torch.rand(groups, beams, generator=g) < 0.2).to(torch.uint8)
    _check(logits, scores, finished, eos=2)


def test_ties_of_many_slices():
    from vault_b200 import beam_select
    flat = torch.zeros(2, 32, 151936, device="cuda")
    tokens, parents, best, _ = beam_select(flat, torch.zeros(2, 32, device="cuda"))
    assert tokens.cpu().tolist() == [list(range(32))] * 2 and int(parents.abs().max()) == 0
    assert float((best + math.log(151936)).abs().max()) <= 2e-5
    live = torch.full((2, 32), -math.inf, device="cuda")
    live[:, 7] = -1.0
    tokens, parents, _, _ = beam_select(flat, live)
    assert tokens.cpu().tolist() == [list(range(32))] * 2 and parents.cpu().tolist() == [[7] * 32] * 2
