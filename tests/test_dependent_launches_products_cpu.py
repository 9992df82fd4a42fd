"""The rules for kernels launched as programmatic dependents, on the sources of the training step's operators."""
import re

import pytest

import test_dependent_launches_cpu as rules
import test_dependent_launches_operators_cpu as operators
import test_dependent_launches_strict_cpu as strict

SMALL = [rules.CSRC / "ops" / n for n in ("few_tokens.cu", "gated.cu", "head.cu", "orthogonal.cu")]


@pytest.mark.parametrize("check", operators.CHECKS, ids=lambda f: f.__name__[5:])
@pytest.mark.parametrize("path", SMALL + [rules.CSRC / "gemm/sm100_products.cu", rules.CSRC / "ops/orthogonal_small.cu"], ids=lambda p: p.name)
def test_rules(path, check):
    check(path)


@pytest.mark.parametrize("path", SMALL, ids=lambda p: p.name)
def test_strict_rules(path):
    assert strict.problems(re.sub(r"//[^\n]*|/\*.*?\*/", "", path.read_text(), flags=re.S)) == []


def test_every_kernel_is_known():
    names = {k for p in SMALL + [rules.CSRC / "gemm/sm100_products.cu", rules.CSRC / "ops/orthogonal_small.cu"] for k in rules.functions(rules._code(p), "__global__")}
    assert names == {"sum_parts_kernel", "sm100_chain_kernel", "orthogonal_small_kernel", "few_nn_kernel", "few_nt_kernel", "gated_act_kernel", "gated_act_bwd_kernel", "head_rows_kernel", "square_sums_kernel", "load_unit_kernel", "load_unit_transposed_kernel", "head_losses_kernel", "momentum_kernel",
                     "apply_update_kernel", "sm100_products_kernel"}
