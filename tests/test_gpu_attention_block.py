"""The four calls of a step together (examples/attention_block.py): chats of different lengths served side by side, another
prompt among token steps, samples behind a shared prefix; every row as if its chat's text had come at once."""
import importlib.util
import os

import pytest
import torch  # noqa: F401 -- its HIP runtime has to be in the process before libtrhip.so asks for one

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "attention_block.py")


# Rows are rounded to bf16 three times on the way (q/k/v, attention's weights and output; 2^-8 each at most, of values that
# the output projection sums with alternating signs): 2^-6 of a row's largest output
# covers them with room, and a key lost out of some hundred is several times that.
@pytest.mark.parametrize("prompts,late,steps,window,sinks", [((37, 200, 5), 90, 20, 0, 0), ((300, 40), 500, 6, 128, 4), ((1, 260), 2, 35, 0, 0)])
def test_steps_equal_the_whole_text(backend, prompts, late, steps, window, sinks):
    spec = importlib.util.spec_from_file_location("attention_block", PATH)
    block = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(block)
    assert block.run(backend, prompts, late, steps, window, sinks) <= 2.0 ** -6
