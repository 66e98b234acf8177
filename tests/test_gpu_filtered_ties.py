"""sas_sample_filtered where ids share one value: shares of the mass are whole
numbers of ids, so a prefix's end is exact."""
import numpy as np
import pytest

from shared_amd import FilterParams
from test_gpu_filtered import device, run

pytestmark = pytest.mark.gpu


def exact_count(n, top_p):
    """The fewest of n equal masses that reach top_p of theirs (their sum's product
    rounded, as the definition's double)."""
    return max(1, int(np.ceil(top_p * float(n))))


# (lists hold the first; the ranges' ids the second and third; the values alone the last)
@pytest.mark.parametrize("n", [2, 10, 58, 1000, 3000, 9000])
@pytest.mark.parametrize("value", [0.3, -7.1, 23.7, 1000.1])
def test_equal_values(sampler, n, value):
    import torch
    rng = np.random.default_rng(n)
    print(f"[gpu] filtered ties n={n} value={value}", flush=True)
    for rest in (-np.inf, value - 200.0):  # no candidates, or candidates that weigh nothing
        for temperature in (0.9, 0.13, 2.7):
            vocab = 20000
            v = np.full((5, vocab), rest, np.float32)
            for r in range(5):
                v[r, rng.permutation(vocab)[:n]] = np.float32(value)
            for top_p in (0.5, 0.9, 0.75, 0.2):
                u = rng.random(5)
                p = FilterParams(temperature=temperature, top_p=top_p)
                out = sampler.sample_filtered(device(v), uniforms=torch.from_numpy(u).cuda(), params=p, full=True)
                counts, probs, ids = (out[k].cpu().numpy() for k in ("counts", "probs", "ids"))
                want = exact_count(n, top_p)
                assert (counts == want).all(), (rest, temperature, top_p, want, counts)
                assert np.array_equal(probs, np.full(5, 1.0 / want)), (want, probs)
                for r in range(5):
                    kept = np.nonzero(v[r] == np.float32(value))[0][:want]
                    at = min(int(u[r] * want), want - 1)
                    near = abs(u[r] * want - round(u[r] * want)) < 1e-9
                    assert near or ids[r] == kept[at], (r, ids[r], kept[at])


def test_the_largest_weighs_one(sampler):
    # whatever the values' distance from zero: the token's share is never above 1, and
    # 1 where it is alone
    import torch
    rng = np.random.default_rng(3)
    for offset in (0.0, 188.7, -2683.7, 49190.0, 345678.0):
        v = (rng.standard_normal((40, 3000)) * 3 + offset).astype(np.float32)
        v[:20, 17] = v[:20].max(1) + 1000.0
        for p in (FilterParams(temperature=0.55), FilterParams(temperature=0.55, top_p=0.5), FilterParams(temperature=0.55, min_p=0.3),
                  FilterParams(temperature=1.9, top_k=2)):
            out = sampler.sample_filtered(device(v), uniforms=torch.from_numpy(rng.random(40)).cuda(), params=p, full=True)
            probs = out["probs"].cpu().numpy()
            assert (probs <= 1).all() and (probs[:20] == 1.0).all() if p.temperature < 1 else (probs <= 1).all()


@pytest.mark.parametrize("offset", [49190.0, -135345.0, 976507.0])
def test_masses_far_from_zero(sampler, offset):
    # v - m is exact: a row far from zero has the masses of its differences
    rng = np.random.default_rng(5)
    v = (rng.standard_normal((9, 5000)) * 3 + offset).astype(np.float32)
    run(sampler, device(v), [FilterParams(temperature=1.0, top_k=k) for k in (1, 2, 3, 5, 8, 0, 0, 40, 100)], rng.random(9))
