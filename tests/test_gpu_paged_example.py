"""GPU: examples/paged_beam_search.py, the paged-cache operators and beam selection in one loop."""
import importlib.util
import os

import pytest
import torch

from tests.conftest import REPO

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("paged_beam_search", os.path.join(REPO, "examples", "paged_beam_search.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.fixture(scope="module")
def model_file(example, tmp_path_factory):
    return example.synthetic_model(str(tmp_path_factory.mktemp("model")))


def _replay(dec, prompt, tokens):
    """Log-probability of `tokens` after `prompt`, fed one at a time to a cache of their own."""
    dev = dec.cache.device
    table = torch.arange(dec.cache.n_pages, dtype=torch.int32, device=dev)[None]
    i32 = dict(dtype=torch.int32, device=dev)
    logits = dec.forward(torch.tensor(prompt, device=dev), table, torch.tensor([len(prompt)], **i32), torch.tensor([0, len(prompt)], **i32))
    total, picks = 0.0, []
    for i, t in enumerate(tokens):
        lp = torch.log_softmax(logits[0].double(), -1)
        picks.append(int(lp.argmax()))
        total += float(lp[t])
        if i + 1 < len(tokens):
            logits = dec.forward(torch.tensor([t], device=dev), table, torch.tensor([len(prompt) + i + 1], **i32), torch.tensor([0, 1], **i32),
                                 max_q=1)
    return total, picks


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
def test_beam_scores_are_the_sequences_own(example, model_file, window, sinks):
    """Every beam's score is the log-probability of its tokens when they are fed again to a cache of their own: page sharing,
    copying and selection lost nothing.  Batch and single sequence sum their projections in another order, which can move
    single cache codes by one step (1/127 of their block's largest value) and with it a logit by a few thousandths."""
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 256, (n,), generator=g).tolist() for n in (3, 16, 75)]
    steps = 20
    dec = example.PagedDecoder(model_file, n_pages=128, page=16, window=window, n_sink=sinks)
    out, scores = example.beam_search(dec, prompts, beams=3, steps=steps, eos_id=-1)
    assert bool((scores[:, :-1] >= scores[:, 1:]).all())
    single = example.PagedDecoder(model_file, n_pages=8, page=16, window=window, n_sink=sinks)
    for p, prompt in enumerate(prompts):
        assert len({tuple(x) for x in out[p].tolist()}) == 3
        for j in range(3):
            total, _ = _replay(single, prompt, out[p, j].tolist())
            assert abs(total - float(scores[p, j])) <= 5e-3 * steps


def test_one_beam_is_greedy(example, model_file):
    """A single beam's tokens are the most probable ones of its own replay, except where two logits are within the replay's
    difference."""
    prompt = list(range(40, 90))
    dec = example.PagedDecoder(model_file, n_pages=16, page=16)
    out, scores = example.beam_search(dec, [prompt], beams=1, steps=12, eos_id=-1)
    _, picks = _replay(example.PagedDecoder(model_file, n_pages=16, page=16), prompt, out[0, 0].tolist())
    assert picks == out[0, 0].tolist()
