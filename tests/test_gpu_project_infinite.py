"""sas_project with infinite weights: bf16 hidden states give what the sum
gives; f32 ones, which go in as three pieces, no finite number.  No other
output changes."""
import numpy as np
import pytest

from shared_amd import Adapters

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("x", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows", [2, 40, 200])
def test_infinite_weights(sampler, rows, x):
    import torch
    inf = float("inf")
    g = torch.Generator(device="cuda")
    g.manual_seed(rows)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    hidden, w = normal(rows, 256).to(getattr(torch, x)), normal(300, 256).bfloat16()
    a, b = normal(3, 16, 256).bfloat16(), normal(3, 300, 16).bfloat16()
    which = torch.from_numpy((np.arange(rows) % 3).astype(np.int32)).cuda()
    pool = Adapters(a, b)
    clean = sampler.project(hidden, w, adapters=pool, row_adapter=which)
    w[7, 100], w[250, 3] = inf, -inf
    got = sampler.project(hidden, w, adapters=pool, row_adapter=which)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[:, [7, 250]] = True
    assert torch.equal(got[~hit], clean[~hit]) and not torch.isfinite(got[hit]).any()
    if x == "bfloat16":
        sign = torch.sign(hidden.float())
        assert (hidden[:, [100, 3]] != 0).all()
        assert torch.equal(got[:, 7], sign[:, 100] * inf) and torch.equal(got[:, 250], -sign[:, 3] * inf)
    b[1, 40, 5] = inf
    got = sampler.project(hidden, w, adapters=pool, row_adapter=which)
    hit[which == 1, 40] = True
    assert torch.equal(got[~hit], clean[~hit]) and not torch.isfinite(got[hit]).any()
