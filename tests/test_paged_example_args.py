"""What examples/paged_beam_search.py refuses before it runs anything."""
import importlib.util
import os

import pytest

from tests.conftest import REPO


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("paged_beam_search", os.path.join(REPO, "examples", "paged_beam_search.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("prompts", [[[]], [[1, 2], []], [[], [3]], []])
def test_prompts_of_no_token(example, prompts):
    """A prompt of no token has no last row to go on from: it would go on from another prompt's."""
    with pytest.raises(ValueError, match="prompt"):
        example.beam_search(None, prompts, beams=2, steps=3, eos_id=-1)
