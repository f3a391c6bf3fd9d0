"""The example decoder: attention operators and the MoE FFN together, prompts and single tokens."""
import os
import sys

import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.gpu
@pytest.mark.parametrize("prompts,steps", [("70,1,300", 5), ("17", 48)])
def test_token_by_token_matches_the_prompt(prompts, steps):
    """bf16 projections of other shapes round otherwise: 2^-8 a value, a few times a layer, and an expert or a code of the
    cache chosen otherwise now and then; two layers stay below a tenth."""
    import attention_block
    assert attention_block.main(["--layers", "2", "--prompts", prompts, "--steps", str(steps)]) < 0.1
