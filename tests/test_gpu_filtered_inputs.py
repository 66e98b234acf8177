"""sas_sample_filtered and sas_project write nothing but their results."""
import numpy as np
import pytest

from shared_amd import Adapters, FilterParams
from test_gpu_filtered import CUTS, device, run

pytestmark = pytest.mark.gpu


def test_logits_are_left_alone(sampler):
    import torch
    rng = np.random.default_rng(32)
    whole = device((rng.standard_normal((7, 10007)) * 3).astype(np.float32))
    before = whole.clone()
    for k, view in enumerate((whole[:, 3:9001], whole[1::2], whole[2:5, 1:], whole)):
        n = view.shape[0]
        run(sampler, view, [FilterParams(temperature=1.0, **CUTS[(k + r) % len(CUTS)]) for r in range(n)], rng.random(n))
    assert torch.equal(whole, before)


@pytest.mark.parametrize("rows", [3, 40, 200])
def test_projection_inputs_are_left_alone(sampler, rows):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(rows)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    x, w, a, b = normal(rows, 136), normal(300, 136).bfloat16(), normal(5, 24, 136).bfloat16(), normal(5, 300, 24).bfloat16()
    scales, ranks = normal(5), torch.tensor([3, 24, 0, 8, 17], dtype=torch.int32, device="cuda")
    which = (torch.arange(rows, device="cuda") % 6 - 1).to(torch.int32)
    inputs = (x, w, a, b, scales, ranks, which)
    before = [t.clone() for t in inputs]
    sampler.project(x, w, adapters=Adapters(a, b, scales=scales, ranks=ranks), row_adapter=which, softcap=5.0)
    assert all(torch.equal(t, old) for t, old in zip(inputs, before))
