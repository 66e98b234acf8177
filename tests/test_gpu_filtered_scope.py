"""sas_sample_filtered on rows whose values lie at the end of the value ranges'
scope (2^22 ranges of T / 16 to T / 8 from zero): parts on both sides of it."""
import numpy as np
import pytest

from shared_amd import FilterParams
from test_gpu_filtered import device, run

pytestmark = pytest.mark.gpu

CUTS = [dict(), dict(top_p=0.9), dict(min_p=0.2), dict(top_k=700), dict(top_k=3000, top_p=0.8, min_p=0.05)]


# (temperature, the scope's end: 2^22 times 2^floor(log2(T / 8)))
@pytest.mark.parametrize("temperature,end", [(1e-3, 512.0), (1.0, 524288.0), (1e-5, 4.0)])
@pytest.mark.parametrize("rows", [1, 40])
def test_parts_on_both_sides_of_the_scope(sampler, temperature, end, rows):
    rng = np.random.default_rng(int(rows + end))
    print(f"[gpu] filtered scope T={temperature} rows={rows}", flush=True)
    vocab = 100000 if rows > 1 else 8192
    part = 8192 if rows > 1 else 2048
    for sign in (-1.0, 1.0):
        # the largest value within a few T of the end, on its near side for a negative
        # row; every other part on the other side
        step = max(temperature / 4, float(np.spacing(np.float32(end))))
        v = np.empty((rows, vocab), np.float32)
        v[:, :part] = sign * end + step * rng.integers(1, 3, (rows, part))
        v[:, part:] = sign * end - step * rng.integers(0, 8, (rows, vocab - part))
        for c in CUTS:
            run(sampler, device(v), [FilterParams(temperature=temperature, **c)] * rows, rng.random(rows))


def test_far_parts_leave_a_row_where_it_was(sampler):
    # parts of the type's lowest value (a mask written into the logits) are out of scope
    # and weigh nothing
    rng = np.random.default_rng(31)
    v = (rng.standard_normal((6, 60000)) * 3).astype(np.float32)
    v[:, 8192:40000] = np.finfo(np.float32).min
    for c in CUTS:
        run(sampler, device(v), [FilterParams(temperature=0.8, **c)] * 6, rng.random(6))
