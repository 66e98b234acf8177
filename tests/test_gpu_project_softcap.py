"""The softcap behind sas_project against tanh in 64 bits, in units of the last
place."""
import numpy as np
import pytest

from shared_amd import SasError

pytestmark = pytest.mark.gpu


def capped(sampler, x, cap):
    """cap * tanh(x / cap) of f32 values: a projection whose weight picks them."""
    import torch
    rows = np.zeros((x.size, 8), np.float32)
    rows[:, 0] = x
    pick = torch.zeros((1, 8), dtype=torch.bfloat16, device="cuda")
    pick[0, 0] = 1.0
    return sampler.project(torch.from_numpy(rows).cuda(), pick, softcap=cap).cpu().numpy()[:, 0]


def ulps(got, want):
    return np.abs(got.astype(np.float64) - want) / 2.0 ** (np.floor(np.log2(np.abs(want))) - 23)


# From 0.625 on, t = 1 - 2 / (e + 1) with e = e^2|x|, in ulps of 2^-24 (t >= 0.55): 1 ulp of
# exp2 and the roundings of its argument are (2 + 3 |x|) 2^-24 of e, times sech^2(x) / 2 at
# most 1.34; e + 1 rounded, times 2 / (e + 1), 0.45; 1 ulp of the reciprocal 0.89; the last
# step 0.5.  Below, the polynomial's terms are at most 0.13 of the result: 0.4 of their
# roundings, 0.1 of the fit, 0.5 of the last step.
BOUND = 3.2


def test_cap_of_one(sampler):
    # (x / 1 and 1 * tanh are exact)
    rng = np.random.default_rng(1)
    parts = [rng.uniform(0.0, 0.7, 150000), rng.uniform(0.6, 2.0, 150000), rng.uniform(2.0, 12.0, 100000),
             np.exp(rng.uniform(np.log(1e-30), 0.0, 50000)), 0.625 + np.arange(-20000, 20000) * 2.0 ** -24]
    x = np.concatenate(parts).astype(np.float32) * rng.choice(np.array([-1.0, 1.0], np.float32), sum(p.size for p in parts))
    off = ulps(capped(sampler, x, 1.0), np.tanh(x.astype(np.float64)))
    print(f"[gpu] tanh: {off.max():.2f} ulp, at {x[off.argmax()]!r}", flush=True)
    assert off.max() <= BOUND


def test_ends(sampler):
    x = np.array([0.0, -0.0, np.inf, -np.inf, 16.0, -16.0, 3e38, -3e38, 2.0 ** -100], np.float32)
    got = capped(sampler, x, 1.0)
    assert np.array_equal(got, np.array([0, 0, 1, -1, 1, -1, 1, -1, 2.0 ** -100], np.float32))
    got = capped(sampler, x, 30.0)
    assert np.array_equal(got[:2], [0, 0]) and np.array_equal(got[2:4], [30, -30]) and np.array_equal(got[6:8], [30, -30])
    assert np.isnan(capped(sampler, np.array([np.nan], np.float32), 30.0)).all()


def test_least_cap(sampler):
    # 1 / cap is finite from the smallest normal number on; below it 0 gave NaN
    least = float(np.finfo(np.float32).tiny)
    got = capped(sampler, np.array([0.0, 1.0, -1e30], np.float32), least)
    assert np.array_equal(got, np.array([0.0, least, -least], np.float32))
    with pytest.raises(SasError, match="softcap"):
        capped(sampler, np.zeros(1, np.float32), least / 2)


def test_cap_of_thirty(sampler):
    # 30 ulps of t are up to 30 / 16 of 30 t: 6; x / 30 is two roundings, which move the
    # result by 2^-23 of itself at most: 2; the product with 30 rounds once: 0.5
    rng = np.random.default_rng(2)
    x = rng.uniform(-150.0, 150.0, 300000).astype(np.float32)
    off = ulps(capped(sampler, x, 30.0), 30.0 * np.tanh(x.astype(np.float64) / 30.0))
    print(f"[gpu] capped: {off.max():.2f} ulp", flush=True)
    assert off.max() <= 30 / 16 * BOUND + 2.5
