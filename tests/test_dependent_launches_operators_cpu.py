"""The rules for kernels launched as programmatic dependents, on the sources of the long-context operators."""
import pytest

import test_dependent_launches_cpu as rules

SOURCES = [rules.CSRC / "ops/rotary.cu", rules.CSRC / "ops/distill.cu", rules.CSRC / "ops/window_decode.cu",
           rules.CSRC / "ops/window_attention.cu"]
CHECKS = [rules.test_inputs_of_dependent_kernels_are_read_coherently, rules.test_dependent_launches_wait,
          rules.test_dependent_kernels_wait_before_they_touch_memory, rules.test_kernels_of_a_row_exchange_do_not_let_the_next_one_start]


@pytest.mark.parametrize("check", CHECKS, ids=lambda f: f.__name__[5:])
@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_rules(path, check):
    check(path)
