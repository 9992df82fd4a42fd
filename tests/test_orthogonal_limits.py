"""Orthogonal update: where its result may lie."""
import pytest
import torch

import test_orthogonal as base
from meshslice_b200.ops import functional as F

gpu = pytest.mark.gpu
both = pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])


@both
@pytest.mark.parametrize("shape,strides", [((2, 8, 8), (32, 8, 1)), ((2, 8, 8), (8, 8, 1)), ((2, 8, 8), (1, 8, 1)), ((8, 8), (1, 1)), ((8, 8), (7, 1)),
                                           ((8, 8), (1, 7)), ((3, 8, 8), (8, 16, 1)), ((2, 1, 8), (7, 8, 1))])
def test_results_that_lie_on_one_another_are_refused(dev, shape, strides):
    out = torch.zeros(512, device=dev).as_strided(shape, strides)
    with pytest.raises(ValueError, match="element"):
        F.orthogonalize(torch.ones(shape, device=dev), out=out)


@both
@pytest.mark.parametrize("shape,strides", [((2, 8, 8), (64, 8, 1)), ((2, 8, 8), (8, 16, 1)), ((2, 8, 8), (64, 1, 8)), ((8, 2, 8), (1, 64, 8)), ((8, 8), (9, 1)),
                                           ((1, 8, 8), (0, 8, 1)), ((2, 1, 8), (8, 0, 1)), ((2, 1, 1), (1, 1, 1)), ((2, 8, 1), (8, 1, 1))])
def test_results_that_lie_among_one_another_are_taken(dev, shape, strides):
    g = torch.randn(shape, generator=torch.Generator().manual_seed(0)).to(dev)
    out = torch.zeros(512, device=dev).as_strided(shape, strides)
    assert F.orthogonalize(g, out=out) is out
    assert torch.equal(out, F.orthogonalize(g, out_dtype=torch.float32))


@both
@pytest.mark.parametrize("n", [130, 290])
def test_out_in_another_storage_over_the_same_memory(dev, n):
    """As in one storage: results that lie where matrices that are still to be read are."""
    g = base.matrices("noise", 4, 70, n).to(dev)
    want = F.orthogonalize(g[:3], out_dtype=torch.float32)
    for first, to in ((0, 1), (1, 0)):
        t = torch.zeros(4, 70, n, device=dev)
        t[first:first + 3] = g[:3]
        other = torch.from_dlpack(t[to:])
        F.orthogonalize(t[first:first + 3], out=other[:3])
        assert torch.equal(t[to:to + 3], want)


def test_memory_is_compared_by_its_addresses():
    from meshslice_b200.ops.orthogonal import _meet
    t = torch.zeros(4, 6)
    other = torch.from_dlpack(t[1:])
    assert other.untyped_storage().data_ptr() != t.untyped_storage().data_ptr()
    assert _meet(t[:2], other) and _meet(other[1:], t) and not _meet(t[:1], other) and not _meet(t[:1], t[1:])
