"""More of what the attention operators refuse, without a GPU: scales beyond powers of two, and wrappers called with what is no
tensor of the right kind or no number of the right size."""
import pytest

from ovk_b200 import INVALID_ARGUMENT
from test_attention_refusals import attention, prompt


@pytest.mark.parametrize("scale", [2.4e38, -3.4e38, float("inf"), float("nan")])
def test_scales_that_are_not_finite_in_powers_of_two(scale):
    for rc, message in (attention(scale=scale), prompt(scale=scale)):
        assert rc == INVALID_ARGUMENT and "scale" in message, message


@pytest.mark.parametrize("scale", [2.3e38, -2.3e38, 0.0, 1e-45])
def test_finite_scales_pass(scale):
    for rc, message in (attention(scale=scale), prompt(scale=scale)):
        assert rc == INVALID_ARGUMENT and "null context" in message, message
