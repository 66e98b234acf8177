"""sas_sample_filtered's draw where most ids weigh nothing: every row writes
its token, also where the uniform falls on a stretch of ids whose masses all
round to zero though their sum does not."""
import numpy as np
import pytest

from shared_amd import FilterParams, pack_filter_params
from test_gpu_filtered import device, mass_shift, reference_row

pytestmark = pytest.mark.gpu

SENTINEL = 0x55555555


def draw(s, v, plist, u, dtype="float32"):
    """ids, probs, counts and flags of calls whose outputs hold a sentinel before."""
    import torch
    rows = v.shape[0]
    ids, counts, flags = (torch.full((rows,), SENTINEL, dtype=torch.int32, device="cuda") for _ in range(3))
    probs = torch.full((rows,), -7.0, dtype=torch.float64, device="cuda")
    s.sample_filtered_into(device(v, dtype), ids, uniforms=torch.from_numpy(np.asarray(u, np.float64)).cuda(),
                           row_params=torch.from_numpy(pack_filter_params(plist).view(np.uint8)).cuda(),
                           out_probs=probs, out_counts=counts, out_flags=flags)
    torch.cuda.synchronize()
    return [t.cpu().numpy() for t in (ids, probs, counts, flags)]


def check(s, v, plist, u, dtype="float32"):
    ids, probs, counts, flags = draw(s, v, plist, u, dtype)
    want = None
    for r in range(v.shape[0]):
        if want is None or (v[r] != v[r - 1]).any() or u[r] != u[r - 1]:
            want = reference_row(v[r], plist[r], u[r])
        got = (int(ids[r]), float(probs[r]), int(counts[r]), int(flags[r]))
        assert got[0] == want[0] and got[2] == want[2] and got[3] == 0, (r, u[r], want, got)
        # a mass is rounded to 2^-shift of the largest
        tol = (want[2] + 1) * 2.0 ** -(mass_shift(v.shape[1]) + 1) + 2.0 ** -50
        assert abs(got[1] - want[1]) <= tol, (r, u[r], want, got)


# (rows for each length of a part: 2,048, 4,096 and 8,192 ids)
@pytest.mark.parametrize("rows", [1, 8, 40])
def test_ids_that_weigh_nothing(sampler, rows):
    # exp(-24 / 0.75) is below half of 2^-44; a part of them sums to hundreds of units
    vocab = 262144
    print(f"[gpu] filtered draw rows={rows}", flush=True)
    p = FilterParams(temperature=0.75)
    last = 1 - 2.0 ** -53
    for where, us in (((0,), (0.0, 0.5, last)), ((vocab - 1,), (0.0, 0.5, last)), ((vocab // 2,), (0.0, 2.0 ** -40, 0.5, last)),
                      ((0, vocab - 1), (0.0, 0.25, 0.5 + 2.0 ** -30, 0.75, last)),
                      ((5, 100000, 200000), (1 / 3 + 2.0 ** -30, 2 / 3 + 2.0 ** -29, last))):
        one = np.full(vocab, -24.0, np.float32)
        one[list(where)] = 0.0
        v = np.repeat(one[None], rows, 0)
        for u in us:
            check(sampler, v, [p] * rows, [u] * rows)


def test_a_part_between_nothing_and_the_top(sampler):
    # part 0: one id and no other candidate; part 1: ids that weigh nothing
    v = np.full((3, 4096), -np.inf, np.float32)
    v[:, 2048:] = -36.0
    v[:, 0] = 0.0
    check(sampler, v, [FilterParams(temperature=1.0)] * 3, [0.0, 0.5, 1 - 2.0 ** -53])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_steep_rows_write_every_token(sampler, dtype):
    # low temperatures over ordinary values: parts from nothing to the top
    rng = np.random.default_rng(21)
    rows, vocab = 24, 50257
    v = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    v[:, ::4096] += np.float32(12.0)
    plist = [FilterParams(temperature=float(t)) for t in np.linspace(0.05, 1.0, rows)]
    for u in (0.0, 2.0 ** -50, 1 - 2.0 ** -53):
        ids, probs, counts, flags = draw(sampler, v, plist, [u] * rows, dtype)
        assert ((ids >= 0) & (ids < vocab)).all() and (counts == vocab).all() and (flags == 0).all()
        assert ((probs > 0) & (probs <= 1)).all()
