"""sas_project against its definition in 64 bits."""
import numpy as np
import pytest

from shared_amd import Adapters
from shared_amd._capi import ERR_INVALID, SasError

pytestmark = pytest.mark.gpu


class Problem:
    """Random inputs of one call."""

    def __init__(self, rows, dim, out, n=0, rank=16, *, x="float32", seed=0, ragged=False, share_none=0.2, grouped=False):
        import torch
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        rng = np.random.default_rng(seed)
        normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
        self.x = normal(rows, dim).to(getattr(torch, x))
        self.weight = (normal(out, dim) / dim ** 0.5).bfloat16()
        self.adapters = self.row_adapter = None
        if n:
            ranks = rng.integers(0, rank + 1, n) if ragged else np.full(n, rank)
            self.adapters = Adapters((normal(n, rank, dim) / dim ** 0.5).bfloat16(), normal(n, out, rank).bfloat16(),
                                     scales=torch.from_numpy(rng.uniform(-2, 2, n).astype(np.float32)).cuda(),
                                     ranks=torch.from_numpy(ranks.astype(np.int32)).cuda())
            which = np.where(rng.random(rows) < share_none, -1, rng.integers(0, n, rows))
            which = np.sort(which) if grouped else which
            self.row_adapter = torch.from_numpy(which.astype(np.int32)).cuda()

    def kw(self):
        return dict(adapters=self.adapters, row_adapter=self.row_adapter)

    def reference(self, cols=None):
        """y in 64 bits, and the sum of its terms' magnitudes."""
        import torch
        cols = slice(None) if cols is None else cols
        x = self.x.double()
        y = torch.zeros((x.shape[0], self.weight[cols].shape[0]), dtype=torch.float64, device="cuda")
        size = torch.zeros_like(y)
        w = self.weight[cols].double()
        y += x @ w.T
        size += x.abs() @ w.abs().T
        if self.adapters is not None:
            ad, which = self.adapters, self.row_adapter.cpu().numpy()
            for k in range(len(ad)):
                rows = np.nonzero(which == k)[0]
                if rows.size == 0:
                    continue
                r = int(ad.ranks[k]) if ad.ranks is not None else ad.a.shape[1]
                r = min(max(r, 0), ad.a.shape[1])
                scale = float(ad.scales[k]) if ad.scales is not None else 1.0
                i = torch.from_numpy(rows).cuda()
                a, b = ad.a[k, :r].double(), ad.b[k][cols][:, :r].double()
                y[i] += scale * (x[i] @ a.T @ b.T)
                size[i] += abs(scale) * (x[i].abs() @ a.abs().T @ b.abs().T)
        return y, size

    def check(self, got, cap=0.0, extra=0.0, cols=None):
        """|y - reference| within what f32 sums of its terms can be off by: one
        rounding (2^-23 for a cut one) a term of the longest chain, dim + 3
        ranks + the joins, and the result's own rounding."""
        import torch
        y, size = self.reference(cols)
        y = y + extra
        size = size + (extra.abs() if torch.is_tensor(extra) else abs(extra))
        dim = self.x.shape[1] * (3 if self.x.dtype == torch.float32 else 1)
        rank = 0 if self.adapters is None else self.adapters.a.shape[1]
        tol = (dim + 6 * rank + 16) * 2.0 ** -23 * size
        if cap:
            y = cap * torch.tanh(y / cap)
            tol = tol + 2.0 ** -20 * abs(cap)      # tanh, the division and the product in f32
        if got.dtype == torch.bfloat16:
            tol = tol + 2.0 ** -8 * y.abs() + 1e-38
        off = (got.double() - y).abs()
        bad = ~(off <= tol)
        assert not bad.any(), (int(bad.sum()), got[bad][:4], y[bad][:4], bad.nonzero()[:4])
        # and as sums of rounding errors are: far inside that bound on the whole
        if got.dtype == torch.float32 and not cap:
            assert float(off.norm()) <= 2.0 ** -20 * float(size.norm())


SHAPES = [(1, 2560, 2560), (1, 8, 1), (2, 16, 3), (3, 1000, 77), (15, 256, 16), (16, 64, 64), (17, 72, 65), (33, 520, 1000),
          (64, 2048, 257), (65, 264, 511), (128, 512, 1024), (130, 640, 300), (257, 1032, 515), (300, 136, 2049),
          (512, 256, 256), (1000, 200, 130), (5, 8, 70000)]


@pytest.mark.parametrize("x", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,dim,out", SHAPES)
def test_shapes(sampler, rows, dim, out, x):
    import torch
    print(f"[gpu] project {rows} x {dim} x {out} {x}", flush=True)
    for n, rank, grouped in ((0, 8, False), (3, 16, False), (rows, 8, False), (5, 24, True)):
        p = Problem(rows, dim, out, n, rank, x=x, seed=rows + n, grouped=grouped)
        p.check(sampler.project(p.x, p.weight, **p.kw()))
        p.check(sampler.project(p.x, p.weight, out_dtype=torch.bfloat16, **p.kw()))


@pytest.mark.parametrize("rank", [8, 16, 32, 40, 64, 128, 256])
@pytest.mark.parametrize("rows", [1, 20, 150])
def test_ranks(sampler, rank, rows):
    print(f"[gpu] project rank={rank} rows={rows}", flush=True)
    for x in ("float32", "bfloat16"):
        p = Problem(rows, 512, 300, 7, rank, x=x, seed=rank, ragged=True)
        p.check(sampler.project(p.x, p.weight, **p.kw()))


def test_no_scales_no_ranks_and_rows_without_adapter(sampler):
    import torch
    p = Problem(40, 256, 200, 4, 16)
    p.adapters = Adapters(p.adapters.a, p.adapters.b)
    p.check(sampler.project(p.x, p.weight, **p.kw()))
    for none in (-1, 4, 99, -2 ** 31):     # outside the pool: no adapter
        which = torch.full((40,), none, dtype=torch.int32, device="cuda")
        got = sampler.project(p.x, p.weight, adapters=p.adapters, row_adapter=which)
        assert torch.equal(got, sampler.project(p.x, p.weight))


def test_f32_values_keep_their_bits(sampler):
    # sums of few terms that f32 holds: nothing may be lost of 24 significant bits
    import torch
    rng = np.random.default_rng(1)
    for rows in (3, 40, 200):
        dim, out, n, rank = 64, 80, 3, 8
        x = np.zeros((rows, dim), np.float32)
        x[:, ::16] = rng.integers(-2 ** 22, 2 ** 22, (rows, 4)) | 1
        w = rng.integers(-1, 2, (out, dim)).astype(np.float32)
        a = np.zeros((n, rank, dim), np.float32)
        a[:, :, ::32] = rng.integers(-1, 2, (n, rank, 2))
        b = np.zeros((n, out, rank), np.float32)
        b[:, np.arange(out), rng.integers(0, rank, out)] = 1.0
        which = rng.integers(0, n, rows)
        dev = lambda t, d=torch.float32: torch.from_numpy(t).cuda().to(d)  # noqa: E731
        got = sampler.project(dev(x), dev(w, torch.bfloat16), adapters=Adapters(dev(a, torch.bfloat16), dev(b, torch.bfloat16)),
                              row_adapter=dev(which.astype(np.int32), torch.int32))
        want = x.astype(np.float64) @ w.T
        for r in range(rows):
            want[r] += b[which[r]] @ (a[which[r]] @ x[r].astype(np.float64))
        assert np.abs(want).max() < 2 ** 25
        fits = np.abs(want) < 2 ** 24
        assert np.array_equal(got.cpu().numpy()[fits], want[fits])


def test_values_that_are_not_finite_stay_where_they_are(sampler):
    import torch
    nan, inf = float("nan"), float("inf")
    for rows in (20, 150):
        for x in ("float32", "bfloat16"):
            p = Problem(rows, 256, 300, 4, 16, x=x, share_none=0.3, seed=3)
            clean = sampler.project(p.x, p.weight, **p.kw())
            which = p.row_adapter.cpu().numpy()
            p.x[5, 7] = inf
            p.weight[11, 3] = nan
            ad = p.adapters
            ad.a[1, 2, 5] = inf
            ad.b[2, 17, 3] = nan
            ad.ranks[3] = 5
            before = sampler.project(p.x, p.weight, **p.kw())
            ad.a[3, 5:], ad.b[3, :, 5:] = nan, inf       # behind the ranks in use
            got = sampler.project(p.x, p.weight, **p.kw())
            assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(before))
            rows_ok = torch.ones(rows, dtype=torch.bool, device="cuda")
            rows_ok[5] = False
            rows_ok[torch.from_numpy(np.nonzero((which == 1) | (which == 3))[0]).cuda()] = False
            two = torch.from_numpy(which == 2).cuda()
            col_ok = torch.ones(300, dtype=torch.bool, device="cuda")
            col_ok[11] = False
            same = (got == clean) | ~rows_ok[:, None] | ~col_ok[None, :]
            same[:, 17] |= two
            assert same.all()
            assert not torch.isfinite(got[5]).any() and not torch.isfinite(got[:, 11]).any()
            assert not torch.isfinite(got[two, 17]).any() or not two.any()


@pytest.mark.parametrize("rows", [1, 30, 200])
def test_softcap_and_accumulate(sampler, rows):
    import torch
    for dtype in (torch.float32, torch.bfloat16):
        p = Problem(rows, 256, 333, 4, 16, seed=rows)
        p.check(sampler.project(p.x, p.weight, softcap=3.0, out_dtype=dtype, **p.kw()), cap=3.0)
        old = torch.randn((rows, 333), device="cuda").to(dtype)
        out = old.clone()
        sampler.project_into(p.x, p.weight, out, accumulate=True, **p.kw())
        p.check(out, extra=old.double())
        out = old.clone()
        sampler.project_into(p.x, None, out, accumulate=True, softcap=2.0, **p.kw())
        p.weight = torch.zeros_like(p.weight)
        p.check(out, cap=2.0, extra=old.double())


def test_strides(sampler):
    import torch
    p = Problem(50, 128, 90, 3, 16, seed=9)
    want = sampler.project(p.x, p.weight, **p.kw())
    pad = lambda t, cols, dtype: torch.full((*t.shape[:-1], cols), float("nan"), dtype=dtype, device="cuda")  # noqa: E731
    x = pad(p.x, 132, torch.float32)
    x[:, :128] = p.x
    w = pad(p.weight, 136, torch.bfloat16)
    w[:, :128] = p.weight
    a, b = pad(p.adapters.a, 144, torch.bfloat16), pad(p.adapters.b, 24, torch.bfloat16)
    a[..., :128], b[..., :16] = p.adapters.a, p.adapters.b
    ad = Adapters(a[..., :128], b[..., :16], scales=p.adapters.scales, ranks=p.adapters.ranks)
    out = pad(want, 97, torch.float32)
    sampler.project_into(x[:, :128], w[:, :128], out[:, 3:93], adapters=ad, row_adapter=p.row_adapter)
    assert torch.equal(out[:, 3:93], want)
    assert torch.isnan(out[:, :3]).all() and torch.isnan(out[:, 93:]).all()
    big = torch.zeros((50, 90), dtype=torch.bfloat16, device="cuda")
    odd = torch.full((50, 91), 7.0, dtype=torch.bfloat16, device="cuda")
    sampler.project_into(p.x, p.weight, big, **p.kw())
    sampler.project_into(p.x, p.weight, odd[:, 1:], **p.kw())
    assert torch.equal(odd[:, 1:], big) and (odd[:, 0] == 7.0).all()


def test_offsets_past_32_bits(sampler):
    # a weight and a result of over 2^31 elements
    import torch
    p = Problem(20, 8192, 64, 2, 8, x="bfloat16", seed=4)
    out = (1 << 18) + 64
    weight = torch.zeros((out, 8192), dtype=torch.bfloat16, device="cuda")
    weight[-64:] = p.weight
    b = torch.zeros((2, out, 8), dtype=torch.bfloat16, device="cuda")
    b[:, -64:] = p.adapters.b
    ad = Adapters(p.adapters.a, b, scales=p.adapters.scales, ranks=p.adapters.ranks)
    y = sampler.project(p.x, weight, adapters=ad, row_adapter=p.row_adapter)
    assert not y[:, :-64].any()
    p.check(y[:, -64:])
    del weight, b, ad, y
    flat = torch.zeros((1 << 31) + 4096, dtype=torch.bfloat16, device="cuda")
    far = flat.as_strided((2, 64), (1 << 31, 1))
    sampler.project_into(p.x[:2], p.weight, far, adapters=p.adapters, row_adapter=p.row_adapter[:2])
    want = sampler.project(p.x[:2], p.weight, adapters=p.adapters, row_adapter=p.row_adapter[:2], out_dtype=torch.bfloat16)
    assert torch.equal(far, want)


def test_same_bits_and_other_stream(sampler):
    import torch
    p = Problem(70, 1024, 5000, 9, 16, seed=6)
    want = sampler.project(p.x, p.weight, **p.kw())
    side = torch.cuda.Stream()
    for _ in range(3):
        assert torch.equal(sampler.project(p.x, p.weight, **p.kw()), want)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        a = sampler.project(p.x, p.weight, **p.kw())
    side.synchronize()
    b = sampler.project(p.x, p.weight, stream=side, **p.kw())
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want)


def test_a_row_alone_is_the_row_in_a_batch(sampler):
    # rows do not depend on their neighbours but for the order of f32 sums
    p = Problem(90, 768, 1000, 5, 16, seed=8)
    whole = sampler.project(p.x, p.weight, **p.kw())
    p.check(whole)
    for i in (0, 17, 89):
        q = Problem(90, 768, 1000, 5, 16, seed=8)
        q.x, q.row_adapter = q.x[i:i + 1], q.row_adapter[i:i + 1]
        q.check(sampler.project(q.x, q.weight, **q.kw()))


def test_in_a_graph():
    import torch
    from shared_amd import Sampler
    with Sampler(0) as s:
        for rows in (4, 150):
            p = Problem(rows, 512, 1000, 4, 16, seed=2)
            s.reserve_project(rows, 512, rank=16)
            out = torch.empty((rows, 1000), device="cuda")
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                s.project_into(p.x, p.weight, out, **p.kw())
            for k in range(4):
                p.x.normal_()
                g.replay()
                torch.cuda.synchronize()
                got = out.clone()
                want = s.project(p.x, p.weight, **p.kw())
                torch.cuda.synchronize()
                assert torch.equal(got, want), k


def test_no_rows(sampler):
    import torch
    p = Problem(3, 64, 64, 2, 8)
    got = sampler.project(p.x[:0], p.weight, adapters=p.adapters, row_adapter=p.row_adapter[:0])
    torch.cuda.synchronize()
    assert got.shape == (0, 64)


def test_refusals(sampler):
    import ctypes

    import torch
    from shared_amd import _capi
    p = Problem(4, 64, 40, 2, 16)
    out = torch.empty((4, 40), device="cuda")
    for bad in (dict(x=p.x[:, :60]), dict(x=p.x.double()), dict(x=p.x[:, 1:57]), dict(weight=p.weight.float()),
                dict(weight=p.weight[:39]), dict(weight=None), dict(out=out[:3]), dict(out=out.half()), dict(out=out.t()),
                dict(row_adapter=None), dict(row_adapter=p.row_adapter[:3]), dict(row_adapter=p.row_adapter.long()),
                dict(softcap=-1.0), dict(softcap=float("nan")), dict(x=p.x.cpu())):
        args = {**dict(x=p.x, weight=p.weight, out=out, adapters=p.adapters, row_adapter=p.row_adapter), **bad}
        with pytest.raises((ValueError, SasError)):
            sampler.project_into(args.pop("x"), args.pop("weight"), args.pop("out"), **args)
    with pytest.raises(ValueError):
        Adapters(p.adapters.a, p.adapters.b[:, :, :8])
    with pytest.raises(ValueError):
        Adapters(p.adapters.a.float(), p.adapters.b)
    with pytest.raises(ValueError):
        Adapters(p.adapters.a, p.adapters.b, scales=torch.zeros(3, device="cuda"))
    lib = _capi.load()
    ad = p.adapters
    good = _capi.SasProjection(x=p.x.data_ptr(), x_stride=64, rows=4, weight=p.weight.data_ptr(), weight_stride=64, dim=64,
                               out_dim=40, adapters=2, rank=16, a=ad.a.data_ptr(), a_stride=64, a_adapter_stride=1024,
                               b=ad.b.data_ptr(), b_stride=16, b_adapter_stride=640, row_adapter=p.row_adapter.data_ptr(),
                               out=out.data_ptr(), out_stride=40)
    assert lib.sas_project(sampler._h, ctypes.byref(good), None) == 0
    torch.cuda.synchronize()
    for name, value, word in (("rows", -1, "rows"), ("rows", 1 << 20, "rows"), ("dim", 60, "dim"), ("dim", 0, "dim"),
                              ("out_dim", 0, "out_dim"), ("x_type", 2, "x_type"), ("out_type", 7, "out_type"),
                              ("adapters", -1, "adapters"), ("rank", 12, "rank"), ("rank", 264, "rank"), ("rank", 0, "rank"),
                              ("x_stride", 66, "x_stride"), ("x_stride", 56, "x_stride"), ("weight_stride", 60, "weight_stride"),
                              ("a_stride", 12, "a_stride"), ("b_stride", 12, "b_stride"), ("b_adapter_stride", 4, "b_stride"),
                              ("a_adapter_stride", -8, "a_stride"), ("out_stride", 39, "out_stride"), ("x", None, "x and out"),
                              ("out", None, "x and out"), ("a", None, "required"), ("row_adapter", None, "required"),
                              ("weight", None, "weight"), ("x", p.x.data_ptr() + 4, "aligned"),
                              ("weight", p.weight.data_ptr() + 2, "aligned"), ("out", out.data_ptr() + 2, "aligned"),
                              ("b", ad.b.data_ptr() + 2, "aligned")):
        d = _capi.SasProjection.from_buffer_copy(good)
        setattr(d, name, value)
        assert lib.sas_project(sampler._h, ctypes.byref(d), None) == ERR_INVALID, name
        assert word in lib.sas_last_error(sampler._h).decode(), name
    for bad in ((-1, 64, 8), (4, 60, 8), (4, 64, 12), (4, 64, 264)):
        with pytest.raises(SasError):
            sampler.reserve_project(bad[0], bad[1], rank=bad[2])
