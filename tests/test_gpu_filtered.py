"""sas_sample_filtered against its definition in 64 bits (numpy): the token
ids and the kept counts are equal, the probabilities agree to the rounding of
the integer masses."""
import math

import numpy as np
import pytest

from shared_amd import FilterParams, pack_filter_params
from shared_amd._capi import ERR_INVALID, FLAG_EMPTY_ROW, MAX_HISTORY, SasError

pytestmark = pytest.mark.gpu


def softcapped(v, cap):
    q = (v / np.float32(cap)).astype(np.float32)
    return (np.float32(cap) * np.tanh(q.astype(np.float64)).astype(np.float32)).astype(np.float32)


def mass_shift(vocab):
    return 62 - max(0, math.ceil(math.log2(vocab)))


def reference_row(v, p, u, allowed=None, history=None):
    """(id, probability, kept) of one row; v float32."""
    v = v.astype(np.float32)
    if p.softcap > 0:
        v = softcapped(v, p.softcap)
    v = v.astype(np.float64)
    if history is not None and len(history):
        seen, times = np.unique(history[history < v.size], return_counts=True)
        old = v[seen]
        new = np.where(old > 0, old / p.repetition_penalty, old * p.repetition_penalty)
        v[seen] = (new - p.frequency_penalty * times - p.presence_penalty).astype(np.float32)
    if allowed is not None:
        v[~allowed] = -np.inf
    v[np.isnan(v)] = -np.inf
    n = int((v > -np.inf).sum())
    if n == 0:
        return -1, 0.0, 0
    order = np.argsort(-v, kind="stable")
    if not p.temperature > 0 or p.top_k == 1:
        return int(order[0]), 1.0, 1
    with np.errstate(invalid="ignore"):
        w = np.where(v == v[order[0]], 1.0, np.exp((v - v[order[0]]) / p.temperature))
    n = min(n, p.top_k) if p.top_k > 0 else n
    mass = np.cumsum(w[order[:n]])
    if p.top_p < 1:
        n = min(n, 1 + int(np.searchsorted(mass, max(p.top_p, 0.0) * mass[-1], side="left")))
    if p.min_p > 0:
        n = min(n, int((w[order[:n]] >= min(p.min_p, 1.0)).sum()))
    kept = np.sort(order[:n])
    # masses are integers of 2^-shift: those below half of one are none
    mass = np.cumsum(np.where(w[kept] < 2.0 ** -(mass_shift(v.size) + 1), 0.0, w[kept]))
    at = min(int(np.searchsorted(mass, u * mass[-1], side="right")), n - 1)
    return int(kept[at]), w[kept[at]] / mass[-1], n


def unpack(words, vocab):
    return np.unpackbits(words.view(np.uint8), bitorder="little")[:vocab].astype(bool)


def pack(allowed):
    bits = np.zeros((allowed.shape[0], (allowed.shape[1] + 31) // 32 * 32), np.uint8)
    bits[:, :allowed.shape[1]] = allowed
    return np.packbits(bits, axis=1, bitorder="little").view(np.uint32)


def run(s, logits, plist, u, *, allowed=None, shared=False, history=None, one=False, **kw):
    """GPU results of device logits (any type), checked row by row."""
    import torch
    rows, vocab = logits.shape
    args = {}
    if allowed is not None:
        m = torch.from_numpy(pack(allowed[:1] if shared else allowed).view(np.int32)).cuda()
        args["mask"] = m
    if history is not None:
        off = np.concatenate([[0], np.cumsum([len(h) for h in history])]).astype(np.int32)
        flat = np.concatenate([np.asarray(h, np.uint32) for h in history] + [np.zeros(1, np.uint32)])
        args["hist_ids"] = torch.from_numpy(flat.view(np.int32)).cuda()
        args["hist_offsets"] = torch.from_numpy(off).cuda()
    if one:
        args["params"] = plist[0]
    else:
        args["row_params"] = torch.from_numpy(pack_filter_params(plist).view(np.uint8)).cuda()
    if u is not None:
        args["uniforms"] = torch.from_numpy(np.asarray(u, np.float64)).cuda()
    got = s.sample_filtered(logits, full=True, **args, **kw)
    torch.cuda.synchronize()
    got = {k: v.cpu().numpy() for k, v in got.items()}
    host = logits.float().cpu().numpy()
    shift = mass_shift(vocab)
    for r in range(rows):
        ok = None if allowed is None else allowed[0 if shared else r]
        want = reference_row(host[r], plist[0] if one else plist[r], 0.0 if u is None else u[r], ok,
                             None if history is None else np.asarray(history[r], np.uint32))
        assert got["ids"][r] == want[0] and got["counts"][r] == want[2], (r, plist[0 if one else r], want, got["ids"][r], got["counts"][r])
        # every mass is rounded to 2^-shift of the largest (2^-(shift + 1) off),
        # its own exponential within 2 ulp
        tol = (want[2] + 1) * 2.0 ** -(shift + 1) + 2.0 ** -50
        assert abs(got["probs"][r] - want[1]) <= tol * max(want[1], 2.0 ** -20), (r, got["probs"][r], want[1])
        assert got["flags"][r] == (FLAG_EMPTY_ROW if want[0] < 0 else 0)
    return got


def peaked(rng, rows, vocab, top=18.0):
    v = rng.standard_normal((rows, vocab)) * 1.8
    for r in range(rows):
        hot = rng.integers(0, vocab, max(1, min(300, vocab // 3)))
        v[r, hot] = np.maximum(v[r, hot], top - (1 + rng.random()) * np.log(np.arange(1, hot.size + 1)))
    return v.astype(np.float32)


def device(v, dtype="float32"):
    import torch
    return torch.from_numpy(v).cuda().to(getattr(torch, dtype))


CUTS = [dict(), dict(top_p=0.9), dict(min_p=0.1), dict(top_k=40), dict(top_k=3000, top_p=0.97, min_p=1e-3),
        dict(top_k=2, top_p=0.999), dict(top_p=0.0), dict(min_p=1.0), dict(top_p=0.9999, min_p=1e-6)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("vocab", [1, 2, 3, 5, 31, 1000, 4097, 8192, 8193, 50257, 151936])
def test_against_definition(sampler, vocab, dtype):
    rng = np.random.default_rng(vocab)
    print(f"[gpu] filtered vocab={vocab} {dtype}", flush=True)
    rows = len(CUTS)
    for spread in ("peaked", "flat"):
        v = peaked(rng, rows, vocab) if spread == "peaked" else (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
        plist = [FilterParams(temperature=float(rng.choice([0.5, 1.0, 1.7])), **c) for c in CUTS]
        run(sampler, device(v, dtype), plist, rng.random(rows))


@pytest.mark.parametrize("rows,vocab", [(1, 262144), (3, 262144), (200, 5000), (40, 40000)])
def test_batch_shapes(sampler, rows, vocab):
    rng = np.random.default_rng(rows)
    print(f"[gpu] filtered rows={rows} vocab={vocab}", flush=True)
    for c in (dict(), dict(top_p=0.95, min_p=0.02), dict(top_k=100)):
        p = FilterParams(temperature=0.8, **c)
        run(sampler, device(peaked(rng, rows, vocab)), [p] * rows, rng.random(rows), one=True)


def test_large_vocabulary(sampler):
    rng = np.random.default_rng(5)
    vocab = (1 << 22) - 3
    v = (rng.standard_normal((2, vocab)) * 3).astype(np.float32)
    run(sampler, device(v, "float16"), [FilterParams(temperature=1.0, top_p=0.9), FilterParams(temperature=1.2)], rng.random(2))


@pytest.mark.parametrize("shared", [False, True])
def test_masks_and_empty_rows(sampler, shared):
    rng = np.random.default_rng(3)
    rows, vocab = 12, 20011
    v = peaked(rng, rows, vocab)
    allowed = rng.random((rows, vocab)) < 0.1
    if not shared:
        allowed[3] = False              # nothing allowed
        allowed[4] = False
        allowed[4, vocab - 1] = True    # the last id alone
        v[5] = np.nan                   # nothing but NaN
        v[6] = -np.inf                  # nothing but -inf
        v[7] = np.finfo(np.float32).min  # one value, the lowest, for all
        v[8, ~allowed[8]] = np.inf      # what is not allowed is infinite, or no number
        v[9, ~allowed[9]] = np.nan
    plist = [FilterParams(temperature=1.0, **CUTS[r % len(CUTS)]) for r in range(rows)]
    got = run(sampler, device(v), plist, rng.random(rows), allowed=allowed, shared=shared)
    if not shared:
        assert (got["ids"][[3, 5, 6]] == -1).all() and (got["counts"][[3, 5, 6]] == 0).all()


def test_special_values(sampler):
    rng = np.random.default_rng(4)
    vocab = 9000
    v = (rng.standard_normal((10, vocab)) * 2).astype(np.float32)
    v[0, [7, 8500]] = np.inf                       # infinite logits share the mass
    v[1] = 0.0                                     # one value for all
    v[1, ::2] = -0.0
    v[2] = np.where(rng.random(vocab) < 0.5, np.finfo(np.float32).min, v[2])
    v[3, 100:200] = np.finfo(np.float32).max       # ties of the largest value
    v[4] *= 1e-30                                  # differences below any temperature
    v[5] *= 1e30
    v[6] = np.round(v[6])                          # long ties
    v[7] = -np.abs(v[7]) - 50.0
    v[8, rng.random(vocab) < 0.5] = np.nan
    v[9] = np.linspace(0, -600, vocab)             # masses down to e^-600
    for c in CUTS:
        run(sampler, device(v), [FilterParams(temperature=0.9, **c)] * 10, rng.random(10))


def test_parameters_at_their_ends(sampler):
    rng = np.random.default_rng(6)
    nan, inf = float("nan"), float("inf")
    plist = [FilterParams(temperature=0.0), FilterParams(temperature=nan), FilterParams(temperature=-1.0),
             FilterParams(temperature=1.0, top_p=nan), FilterParams(temperature=1.0, top_p=-1.0),
             FilterParams(temperature=1.0, top_p=2.0), FilterParams(temperature=1.0, min_p=nan),
             FilterParams(temperature=1.0, min_p=3.0), FilterParams(temperature=1.0, min_p=-1.0),
             FilterParams(temperature=1.0, top_k=-5), FilterParams(temperature=1.0, top_k=1),
             FilterParams(temperature=1.0, top_k=1 << 30), FilterParams(temperature=1e-4), FilterParams(temperature=1e4),
             FilterParams(temperature=inf, top_p=0.5), FilterParams(temperature=1e-300, min_p=0.5),
             FilterParams(temperature=1.0, top_p=1 - 2.0 ** -53), FilterParams(temperature=1.0, top_p=1e-300)]
    v = peaked(rng, len(plist), 12345)
    run(sampler, device(v), plist, rng.random(len(plist)))


def test_uniforms_at_their_ends(sampler):
    rng = np.random.default_rng(7)
    v = peaked(rng, 8, 30000)
    v[:, 0] = -30.0
    v[:, -1] = -30.0
    u = [0.0, 2.0 ** -60, 1 - 2.0 ** -53, 0.5, 0.0, 1 - 2.0 ** -53, 2.0 ** -24, 1 - 2.0 ** -24]
    plist = [FilterParams(temperature=1.0, top_k=k) for k in (0, 0, 0, 0, 50, 50, 5000, 5000)]
    run(sampler, device(v), plist, u)


@pytest.mark.parametrize("length", [1, 300, 4096, MAX_HISTORY])
def test_penalties(sampler, length):
    rng = np.random.default_rng(length)
    rows, vocab = 6, 33000
    v = peaked(rng, rows, vocab)
    history = [rng.integers(0, vocab, length) for _ in range(rows)]
    history[1] = np.argsort(-v[1])[rng.integers(0, 20, length)]           # the likely ids, many times
    history[2] = np.full(length, int(np.argmax(v[2])))                    # one id, as often as can be
    history[3] = np.concatenate([history[3][:-1], [vocab + 7]])           # an id past the vocabulary
    history[4] = np.zeros(0, np.int64)
    plist = [FilterParams(temperature=0.9, repetition_penalty=1.3, presence_penalty=0.5, frequency_penalty=0.1,
                          **CUTS[r]) for r in range(rows)]
    plist[5].softcap = 15.0
    allowed = rng.random((rows, vocab)) < 0.5
    run(sampler, device(v), plist, rng.random(rows), allowed=allowed, history=history)


def test_softcap(sampler):
    rng = np.random.default_rng(8)
    v = peaked(rng, 9, 40001, top=60.0)
    run(sampler, device(v), [FilterParams(temperature=1.0, softcap=30.0, **c) for c in CUTS], rng.random(9))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strides_and_alignment(sampler, dtype):
    import torch
    rng = np.random.default_rng(9)
    whole = device(peaked(rng, 7, 10007), dtype)
    for view in (whole[:, 3:9001], whole[1::2], whole[2:5, 1:], whole[:, :6]):
        n = view.shape[0]
        run(sampler, view, [FilterParams(temperature=1.0, top_p=0.9)] * n, rng.random(n))
    assert torch.equal(whole, whole.clone())


def test_offsets_past_32_bits(sampler):
    import torch
    rng = np.random.default_rng(10)
    vocab, stride = 5000, (1 << 31) + 8
    flat = torch.empty(stride + vocab, dtype=torch.float16, device="cuda")
    view = flat.as_strided((2, vocab), (stride, 1))
    view.copy_(device(peaked(rng, 2, vocab), "float16"))
    run(sampler, view, [FilterParams(temperature=1.0, top_p=0.9)] * 2, rng.random(2))


def test_split_does_not_change_the_answer(sampler):
    # a row alone, in a small and in a large batch: other splits, the same bits
    import torch
    rng = np.random.default_rng(11)
    v = device((rng.standard_normal((150, 70001)) * 3).astype(np.float32))
    u = torch.from_numpy(rng.random(150)).cuda()
    p = FilterParams(temperature=1.1, top_p=0.95)
    whole = sampler.sample_filtered(v, uniforms=u, params=p, full=True)
    for n in (1, 2, 9, 40):
        part = sampler.sample_filtered(v[:n], uniforms=u[:n], params=p, full=True)
        for key in ("ids", "counts"):
            assert torch.equal(part[key], whole[key][:n]), (n, key)
        assert torch.allclose(part["probs"], whole["probs"][:n], rtol=1e-9, atol=0)


def test_same_bits_every_time(sampler):
    import torch
    rng = np.random.default_rng(12)
    v = device((rng.standard_normal((64, 50000)) * 3).astype(np.float32), "bfloat16")
    u = torch.from_numpy(rng.random(64)).cuda()
    p = FilterParams(temperature=1.0, top_k=9000, top_p=0.99)
    first = sampler.sample_filtered(v, uniforms=u, params=p, full=True)
    for _ in range(5):
        again = sampler.sample_filtered(v, uniforms=u, params=p, full=True)
        assert all(torch.equal(first[k], again[k]) for k in first)


def test_draws_follow_the_masses(sampler):
    # 20,000 draws over evenly spaced uniforms: each kept id as often as its share
    import torch
    n, vocab = 20000, 64
    rng = np.random.default_rng(13)
    one = (rng.standard_normal(vocab) * 2).astype(np.float32)
    v = device(one)[None].expand(n, vocab)
    u = (np.arange(n) + 0.5) / n
    ids = sampler.sample_filtered(v.contiguous(), uniforms=torch.from_numpy(u).cuda(), params=FilterParams(temperature=1.0, top_k=20))
    got = np.bincount(ids.cpu().numpy(), minlength=vocab)
    w = np.exp(one.astype(np.float64))
    w[np.argsort(-one, kind="stable")[20:]] = 0
    assert np.abs(got - n * w / w.sum()).max() <= 1.0   # a stratified count is off by less than one


def test_other_stream(sampler):
    import torch
    rng = np.random.default_rng(14)
    host = peaked(rng, 32, 100000)
    side = torch.cuda.Stream()
    u = torch.from_numpy(rng.random(32)).cuda()
    p = FilterParams(temperature=1.0, top_p=0.9)
    want = sampler.sample_filtered(device(host), uniforms=u, params=p)
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        a = sampler.sample_filtered(device(host), uniforms=u, params=p)
    b = sampler.sample_filtered(device(host), uniforms=u, params=p, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want)


def test_in_a_graph():
    import torch
    from shared_amd import Sampler
    rng = np.random.default_rng(15)
    with Sampler(0) as s:
        s.reserve_filtered(16, 151936)
        v = device(peaked(rng, 16, 151936))
        u = torch.from_numpy(rng.random(16)).cuda()
        ids = torch.empty(16, dtype=torch.int32, device="cuda")
        probs = torch.empty(16, dtype=torch.float64, device="cuda")
        p = FilterParams(temperature=1.0, top_p=0.9, min_p=0.01)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.sample_filtered_into(v, ids, uniforms=u, params=p, out_probs=probs)
        for k in range(4):
            v.copy_(device(peaked(rng, 16, 151936)))
            u.copy_(torch.from_numpy(rng.random(16)))
            g.replay()
            torch.cuda.synchronize()
            got = ids.clone(), probs.clone()
            want = s.sample_filtered(v, uniforms=u, params=p, full=True)
            torch.cuda.synchronize()
            assert torch.equal(got[0], want["ids"]) and torch.equal(got[1], want["probs"]), k


def test_refusals(sampler):
    import ctypes

    import torch
    from shared_amd import _capi
    v = torch.zeros((2, 100), device="cuda")
    u = torch.zeros(2, dtype=torch.float64, device="cuda")
    p = FilterParams(temperature=1.0)
    out = torch.empty(2, dtype=torch.int32, device="cuda")
    for bad in (dict(uniforms=None), dict(uniforms=u.float()), dict(uniforms=u[:1]), dict(vocab=101), dict(vocab=0),
                dict(mask=torch.zeros((2, 3), dtype=torch.int32, device="cuda")),
                dict(mask=torch.zeros((2, 4), dtype=torch.int64, device="cuda")),
                dict(hist_ids=torch.zeros(3, dtype=torch.int32, device="cuda")),
                dict(hist_ids=torch.zeros(3, dtype=torch.int32, device="cuda"),
                     hist_offsets=torch.zeros(2, dtype=torch.int32, device="cuda")),
                dict(row_params=torch.zeros(64, dtype=torch.uint8, device="cuda"))):
        with pytest.raises((ValueError, SasError)):
            sampler.sample_filtered_into(v, out, **{**dict(uniforms=u, params=p), **bad})
    for bad in (v.double(), v.t(), v.cpu(), v[0]):
        with pytest.raises(ValueError):
            sampler.sample_filtered_into(bad, out, uniforms=u, params=p)
    lib = _capi.load()
    good = _capi.SasFilterRows(logits=v.data_ptr(), logits_stride=100, vocab=100, rows=2, uniforms=u.data_ptr(),
                               params=p.to_c(), out_ids=out.data_ptr())
    for name, value, word in (("rows", -1, "rows"), ("vocab", 0, "vocab"), ("vocab", (1 << 22) + 1, "vocab"),
                              ("logits_type", 3, "logits_type"), ("logits_stride", 99, "logits_stride"),
                              ("logits", None, "logits"), ("out_ids", None, "out_ids"), ("uniforms", None, "uniforms"),
                              ("logits", v.data_ptr() + 2, "aligned")):
        d = _capi.SasFilterRows.from_buffer_copy(good)
        setattr(d, name, value)
        assert lib.sas_sample_filtered(sampler._h, ctypes.byref(d), None) == ERR_INVALID
        assert word in lib.sas_last_error(sampler._h).decode()
    d = _capi.SasFilterRows.from_buffer_copy(good)
    d.rows = 0
    assert lib.sas_sample_filtered(sampler._h, ctypes.byref(d), None) == 0
    with pytest.raises(SasError):
        sampler.reserve_filtered(4, 0)
