"""Sampler.project allocates its result, which holds nothing to add to."""
import pytest

from test_gpu_project import Problem

pytestmark = pytest.mark.gpu


def test_no_accumulation_on_new_memory(sampler):
    import torch
    p = Problem(20, 64, 48, 2, 8)
    with pytest.raises(ValueError, match="accumulate"):
        sampler.project(p.x, p.weight, accumulate=True, **p.kw())
    with pytest.raises(ValueError, match="weight"):
        sampler.project(p.x, None, **p.kw())
    want = sampler.project(p.x, p.weight, accumulate=False, **p.kw())
    out = torch.zeros_like(want)
    sampler.project_into(p.x, p.weight, out, accumulate=True, **p.kw())
    assert torch.equal(out, want)
