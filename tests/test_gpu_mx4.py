"""MXFP4 tables against their definition in 64 bits: quantisation, lookup,
products, and the fused head."""
import numpy as np
import pytest

import mx4_reference as R
from shared_amd import Adapters, FilterParams, Mx4, Params, workloads as W
from shared_amd._capi import SasError

pytestmark = pytest.mark.gpu

TYPES = ["float32", "bfloat16", "float16"]


def table(rows, dim, seed=0, spread=8, pad=0):
    """A random table: every code, scales around 1, `pad` blocks between rows."""
    import torch
    rng = np.random.default_rng(seed)
    blocks = (dim + 31) // 32
    codes = rng.integers(0, 256, (rows, 16 * (blocks + pad)), dtype=np.uint8)
    last = codes.reshape(rows, -1)[:, :16 * blocks]
    nib = np.stack([last & 15, last >> 4], 2).reshape(rows, -1)
    nib[:, dim:] = 0
    last[:] = nib[:, 0::2] | nib[:, 1::2] << 4
    # what pads a row is NaN: nothing may come of it
    scales = np.full((rows, (blocks + 3) // 4 * 4 + 4 * pad), 255, np.uint8)
    scales[:, :blocks] = rng.integers(127 - spread, 128 + spread // 2, (rows, blocks))
    return Mx4(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), dim)


def table_values(t):
    return R.values(t.codes.cpu().numpy(), t.scales.cpu().numpy(), t.dim)


def check_quantized(sampler, x):
    """Codes and scales of x (device tensor) are the reference's, byte for byte,
    and nothing behind them is written."""
    import torch
    rows, dim = x.shape
    blocks = (dim + 31) // 32
    codes = torch.full((rows + 2, 16 * (blocks + 1)), 0xA5, dtype=torch.uint8, device="cuda")
    scales = torch.full((rows + 2, (blocks + 3) // 4 * 4 + 4), 0xA5, dtype=torch.uint8, device="cuda")
    sampler.quantize_mx4_into(x, Mx4(codes, scales, dim))
    want_codes, want_scales = R.quantize(x.double().cpu().numpy())
    codes, scales = codes.cpu().numpy(), scales.cpu().numpy()
    bad = np.argwhere(scales[:rows, :blocks] != want_scales)
    assert bad.size == 0, (bad[:4], scales[:rows, :blocks][tuple(bad[0])], want_scales[tuple(bad[0])])
    bad = np.argwhere(codes[:rows, :16 * blocks] != want_codes)
    assert bad.size == 0, (bad[:4], codes[tuple(bad[0])], want_codes[tuple(bad[0])])
    assert (scales[:rows, blocks:(blocks + 3) // 4 * 4] == 0).all()
    assert (scales[:rows, (blocks + 3) // 4 * 4:] == 0xA5).all() and (scales[rows:] == 0xA5).all()
    assert (codes[:rows, 16 * blocks:] == 0xA5).all() and (codes[rows:] == 0xA5).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 7), (2, 31), (5, 32), (4, 33), (7, 100), (1, 127), (6, 128), (3, 129), (2, 1000),
                                      (9, 2560), (130, 520), (1, 16391)])
def test_quantize_shapes(sampler, rows, dim, kind):
    import torch
    print(f"[gpu] quantize {rows} x {dim} {kind}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(rows * 7 + dim)
    x = torch.randn((rows, dim), generator=g, device="cuda")
    x = (x * torch.exp(2 * torch.randn((rows, dim), generator=g, device="cuda"))).to(getattr(torch, kind))
    check_quantized(sampler, x)
    # rows apart, and off 16 bytes
    wide = torch.zeros((rows, dim + 3), dtype=x.dtype, device="cuda")
    wide[:, 1:dim + 1] = x
    check_quantized(sampler, wide[:, 1:dim + 1])


def test_quantize_borders(sampler):
    """Every border between elements and its neighbours in f32, both signs, under
    scales from the smallest to the largest."""
    import torch
    middle = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, 0.125, 7.9999995], np.float32)
    near = np.concatenate([middle, np.nextafter(middle, 0), np.nextafter(middle, 8)]).astype(np.float32)
    near = near[near < 8]
    rows = []
    for e in list(range(-127, 126, 9)) + [-126, -125, 124, 125]:
        for top in (4.0, 7.5):    # sets the block's scale to 2^e
            for at in range(0, len(near), 15):
                row = np.zeros(32)
                part = near[at:at + 15]
                row[0] = top
                row[1:1 + len(part)] = part
                row[16:16 + len(part)] = -part
                rows.append(np.ldexp(row, e))
    x = np.array(rows)
    with np.errstate(over="raise"):
        x = x.astype(np.float32)
    check_quantized(sampler, torch.from_numpy(x).cuda())


def test_quantize_extremes(sampler):
    import torch
    tiny = 2.0 ** -149
    blocks = np.zeros((12, 32))
    blocks[1] = -0.0
    blocks[2, 3] = tiny                      # below half of the smallest element: 0
    blocks[3, :4] = [2.0 ** -128, 2.0 ** -129, 3 * 2.0 ** -130, -2.0 ** -127]
    blocks[4, 5] = np.finfo(np.float32).max
    blocks[5, :2] = [1.0, 2.0 ** -40]
    blocks[6, 31] = np.inf
    blocks[7, 0] = -np.inf
    blocks[8, 17] = np.nan
    blocks[9] = np.arange(32)
    blocks[10, 30] = -1e-30
    blocks[11] = 6.0
    x = torch.from_numpy(blocks.reshape(2, 192).astype(np.float32)).cuda()
    check_quantized(sampler, x)
    for kind in ("bfloat16", "float16"):
        b = x.clone()
        b[b.abs() > 3e38] = 60000.0
        check_quantized(sampler, b.to(getattr(torch, kind)))


def test_quantize_all_half_values(sampler):
    """Every 16-bit value, each with a partner that sets the scale."""
    import torch
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    for kind in ("bfloat16", "float16"):
        v = bits.view(getattr(torch, kind))
        check_quantized(sampler, v.view(-1, 128).cuda())
        check_quantized(sampler, v.view(128, -1).T.contiguous().cuda())


@pytest.mark.parametrize("kind", TYPES)
def test_lookup_every_code_and_scale(sampler, kind):
    import torch
    codes = np.tile(np.arange(256, dtype=np.uint8)[:, None, None], (1, 256, 16))      # a byte, a scale
    codes = codes.transpose(1, 0, 2).reshape(256, 4096)
    scales = np.tile(np.arange(256, dtype=np.uint8)[:, None], (1, 256))
    t = Mx4(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), 8192)
    got = sampler.lookup_mx4(t, out_dtype=getattr(torch, kind))
    want = torch.from_numpy(table_values(t))[:253].to(torch.float32).to(getattr(torch, kind))
    assert torch.equal(got[:253].cpu(), want)
    assert got[255].isnan().all() and got.shape == (256, 8192)


@pytest.mark.parametrize("dim", [1, 8, 31, 33, 64, 100, 777, 2560])
def test_lookup_ids(sampler, dim):
    import torch
    t = table(70, dim, seed=dim, pad=1)
    ids = torch.tensor([0, 69, 5, 5, -1, 70, 2 ** 31 - 1, 33, -2 ** 31, 1], dtype=torch.int32, device="cuda")
    want = torch.from_numpy(table_values(t)).float().cuda()
    rows = torch.stack([want[i] if 0 <= i < 70 else torch.zeros_like(want[0]) for i in ids.tolist()])
    for kind in TYPES:
        ty = getattr(torch, kind)
        assert torch.equal(sampler.lookup_mx4(t, ids, out_dtype=ty), rows.to(ty))
        # rows apart and off 16 bytes; what lies between them stays
        out = torch.full((12, dim + 5), 7.0, dtype=ty, device="cuda")
        sampler.lookup_mx4_into(t, out[:10, 1:dim + 1], ids)
        assert torch.equal(out[:10, 1:dim + 1], rows.to(ty))
        out[:10, 1:dim + 1] = 7.0
        assert (out == 7.0).all()
        assert torch.equal(sampler.lookup_mx4(t, out_dtype=ty), want.to(ty))
    out = torch.empty((3, dim), device="cuda")
    sampler.lookup_mx4_into(t, out)
    assert torch.equal(out, want[:3])


def test_round_trip_keeps_quantised_values(sampler):
    import torch
    x = torch.randn((50, 700), device="cuda")
    once = sampler.lookup_mx4(sampler.quantize_mx4(x))
    assert torch.equal(sampler.lookup_mx4(sampler.quantize_mx4(once)), once)


class Product:
    """Inputs of one product: x_kind float32, bfloat16 or mx4."""

    def __init__(self, rows, dim, out, x_kind, seed=0):
        import torch
        g = torch.Generator(device="cuda").manual_seed(seed)
        if x_kind == "mx4":
            self.x = table(rows, dim, seed=seed + 1, spread=4)
            self.value = torch.from_numpy(table_values(self.x)).cuda()
        else:
            self.x = torch.randn((rows, dim), generator=g, device="cuda").to(getattr(torch, x_kind))
            self.value = self.x.double()
        self.w = table(out, dim, seed=seed + 2)
        self.weight = torch.from_numpy(table_values(self.w)).cuda()

    def check(self, got, cap=0.0, extra=None):
        """Within what f32 sums of exact products can be off by: a rounding of
        2^-23 (a cut one) of the terms' size for each of dim terms (times the pieces
        of an f32 value), and of the joins of the waves' sums."""
        import torch
        y, size = self.value @ self.weight.T, self.value.abs() @ self.weight.abs().T
        if extra is not None:
            y, size = y + extra, size + extra.abs()
        terms = self.weight.shape[1] * (3 if got.dtype != torch.float64 and isinstance(self.x, torch.Tensor) and
                                        self.x.dtype == torch.float32 else 1)
        tol = (terms + 32) * 2.0 ** -23 * size
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


SHAPES = [(1, 2560, 2560), (1, 8, 1), (2, 16, 3), (3, 1000, 77), (5, 264, 100), (6, 512, 40), (15, 256, 16), (16, 64, 64), (17, 72, 65),
          (33, 520, 1000), (64, 2048, 257), (65, 264, 511), (128, 512, 1024), (130, 640, 300), (257, 1032, 515), (300, 136, 2049),
          (512, 256, 256), (1000, 200, 130), (5, 8, 70000), (4, 4096, 33000), (16, 256, 50000), (48, 128, 40000), (100, 96, 30011),
          (520, 384, 2100), (700, 40, 1111)]


@pytest.mark.parametrize("x_kind", ["float32", "bfloat16", "mx4"])
@pytest.mark.parametrize("rows,dim,out", SHAPES)
def test_project_shapes(sampler, rows, dim, out, x_kind):
    import torch
    print(f"[gpu] project_mx4 {rows} x {dim} x {out} {x_kind}", flush=True)
    p = Product(rows, dim, out, x_kind, seed=rows + out)
    p.check(sampler.project_mx4(p.x, p.w))
    p.check(sampler.project_mx4(p.x, p.w, out_dtype=torch.bfloat16))
    p.check(sampler.project_mx4(p.x, p.w, softcap=20.0), cap=20.0)


@pytest.mark.parametrize("rows,dim,out", [(1, 1, 1), (3, 33, 40), (70, 1001, 130), (20, 31, 40000), (300, 129, 600)])
def test_project_four_bits_any_dim(sampler, rows, dim, out):
    p = Product(rows, dim, out, "mx4", seed=dim)
    p.check(sampler.project_mx4(p.x, p.w))


@pytest.mark.parametrize("x_kind", ["float32", "bfloat16", "mx4"])
@pytest.mark.parametrize("rows,out", [(2, 50), (40, 300), (33, 33333), (600, 1111)])
def test_project_accumulate_strides(sampler, rows, out, x_kind):
    """Accumulates on what out holds, through strides of every operand; what lies
    between rows stays, whatever it holds."""
    import torch
    dim = 328
    p = Product(rows, dim, out, x_kind, seed=out)
    p.w = table(out, dim, seed=5, pad=2)
    p.weight = torch.from_numpy(table_values(p.w)).cuda()
    x = p.x
    if x_kind == "mx4":
        p.x = x = table(rows, dim, seed=6, spread=4, pad=1)
        p.value = torch.from_numpy(table_values(x)).cuda()
    else:
        store = torch.full((rows, dim + 24), float("nan"), dtype=x.dtype, device="cuda")
        store[:, :dim] = x
        x = store[:, :dim]
    for kind in ("float32", "bfloat16"):
        held = torch.randn((rows + 3, out + 7), device="cuda").to(getattr(torch, kind))
        got = held.clone()
        view = got[:rows, 3:3 + out]
        before = view.double()
        sampler.project_mx4_into(x, p.w, view, accumulate=True)
        p.check(view, extra=before)
        got[:rows, 3:3 + out] = held[:rows, 3:3 + out]
        assert torch.equal(got, held)


@pytest.mark.parametrize("x_kind", ["float32", "bfloat16", "mx4"])
@pytest.mark.parametrize("rows,out", [(3, 40), (50, 200), (17, 33000), (400, 900)])
def test_project_not_finite_stays(sampler, rows, out, x_kind):
    import torch
    dim = 160
    p = Product(rows, dim, out, x_kind, seed=3)
    clean = sampler.project_mx4(p.x, p.w)
    p.w.scales[out // 2, 4] = 255
    if x_kind == "mx4":
        p.x.scales[rows // 2, 0] = 255
    else:
        p.x[rows // 2, 3] = float("nan")
    got = sampler.project_mx4(p.x, p.w)
    assert got[rows // 2].isnan().all() and got[:, out // 2].isnan().all()
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[rows // 2] = False
    keep[:, out // 2] = False
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("x_kind", ["float32", "bfloat16"])
def test_project_infinite_hidden_state(sampler, x_kind):
    """An infinite value gives what the definition gives: infinities of the
    weights' signs, NaN where a weight is 0."""
    import torch
    p = Product(9, 64, 500, x_kind, seed=8)
    p.x[4, 10] = float("inf")
    got = sampler.project_mx4(p.x, p.w)
    w = p.weight[:, 10]
    want = torch.where(w == 0, float("nan"), torch.where(w > 0, float("inf"), -float("inf"))).float()
    if x_kind == "bfloat16":      # (f32: the other pieces of infinity are 0, its products with w stay infinite)
        assert torch.equal(got[4].nan_to_num(5.0, 1.0, -1.0), want.nan_to_num(5.0, 1.0, -1.0))
    else:
        assert torch.equal(got[4].nan_to_num(5.0, 1.0, -1.0), want.nan_to_num(5.0, 1.0, -1.0))
    assert got[torch.arange(9, device="cuda") != 4].isfinite().all()


def test_project_scales_over_their_range(sampler):
    """Scales from 2^-127 to 2^125 against hidden states that bring the products
    back into range: each product alone in its sum, so exact."""
    import torch
    out = 253
    codes = np.zeros((out, 16), np.uint8)
    codes[:, 0] = 0x57                                  # 6, 3
    codes[:, 15] = 0x91                                 # the last two: 0.5, -0.5
    scales = np.zeros((out, 4), np.uint8)
    scales[:, 0] = np.arange(out)
    w = Mx4(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), 32)
    for column, element in ((0, 6.0), (1, 3.0), (30, 0.5), (31, -0.5)):
        for e in (-20, 0, 20):
            x = np.zeros((7, 32), np.float32)
            x[:, column] = 2.0 ** e
            y = element * np.exp2(np.arange(out) - 127.0 + e)
            want = np.where((np.abs(y) >= 2.0 ** -126) & (np.abs(y) < 2.0 ** 128), y, np.nan)
            for t in (torch.from_numpy(x).cuda(), torch.from_numpy(x).cuda().bfloat16(),
                      sampler.quantize_mx4(torch.from_numpy(x).cuda())):
                got = sampler.project_mx4(t, w).double().cpu().numpy()
                ok = np.isnan(want) | (got == want)
                assert ok.all(), (column, e, np.argwhere(~ok)[:3], got[~ok][:3])


def test_f32_hidden_states_keep_their_bits(sampler):
    import torch
    rng = np.random.default_rng(1)
    for rows in (2, 5, 6, 40, 200):
        for out in (80, 33000):
            dim = 64
            x = np.zeros((rows, dim), np.float32)
            x[:, ::16] = rng.integers(-2 ** 22, 2 ** 22, (rows, 4)) | 1
            w = sampler.quantize_mx4(torch.from_numpy(rng.integers(-1, 2, (out, dim)).astype(np.float32)).cuda())
            want = x.astype(np.float64) @ table_values(w).T
            got = sampler.project_mx4(torch.from_numpy(x).cuda(), w)
            assert np.abs(want).max() <= 2 ** 24 and np.array_equal(got.double().cpu().numpy(), want)


def test_repeats_bit_for_bit_and_rows_do_not_mix(sampler):
    import torch
    for rows, dim, out in ((4, 512, 33000), (40, 512, 400), (600, 512, 512)):
        for kind in ("float32", "bfloat16", "mx4"):
            p = Product(rows, dim, out, kind, seed=1)
            a = sampler.project_mx4(p.x, p.w)
            assert torch.equal(a, sampler.project_mx4(p.x, p.w))
            order = torch.randperm(rows, device="cuda")
            x = Mx4(p.x.codes[order], p.x.scales[order], dim) if kind == "mx4" else p.x[order]
            assert torch.equal(sampler.project_mx4(x, p.w), a[order])


# -------------------------------------------------------- the fused head --

def head_inputs(rows, dim, vocab, seed=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn((vocab, dim), generator=g, device="cuda") * (2.0 / dim ** 0.5)
    hid = torch.randn((rows, dim), generator=g, device="cuda")
    return hid, w


@pytest.mark.parametrize("rows,dim,vocab", [(1, 256, 1000), (2, 512, 33), (3, 2560, 50257), (4, 2560, 5000), (1, 12288, 700),
                                            (4, 2816, 262144)])
def test_head_logits_and_tokens(sampler, rows, dim, vocab):
    """The logits are the product's, and the tokens what sas_sample makes of
    them."""
    import torch
    print(f"[gpu] mx4 head {rows} x {dim} x {vocab}", flush=True)
    hid, w = head_inputs(rows, dim, vocab, seed=rows)
    head = sampler.quantize_mx4(w)
    u = torch.rand(rows, dtype=torch.float64, device="cuda")
    mask = torch.randint(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32), device="cuda", dtype=torch.int64).to(torch.int32)
    hist = torch.randint(0, vocab, (20 * rows,), device="cuda", dtype=torch.int32)
    off = torch.arange(0, 20 * rows + 1, 20, device="cuda", dtype=torch.int32)
    kw = dict(uniforms=u, mask=mask, hist_ids=hist, hist_offsets=off,
              params=Params(temperature=0.9, top_k=40, top_p=0.95, repetition_penalty=1.2, presence_penalty=0.3, softcap=30.0))
    r = sampler.lm_head_sample(hid, head, full=True, logits=True, **kw)
    p = Product.__new__(Product)
    p.x, p.w, p.value, p.weight = hid, head, hid.double(), torch.from_numpy(table_values(head)).cuda()
    p.check(r["logits"])
    again = sampler.sample(r["logits"], full=True, **kw)
    for k in ("ids", "probs", "cand_ids", "counts", "flags"):
        assert torch.equal(r[k], again[k]), k
    assert torch.equal(r["logits"], sampler.project_mx4(hid, head))
    # without out_logits, and rows apart at an address of 4 bytes
    store = torch.zeros((rows, dim + 5), device="cuda")
    store[:, 1:dim + 1] = hid
    assert torch.equal(sampler.lm_head_sample(store[:, 1:dim + 1], head, dim=dim, **kw), r["ids"])


def test_head_greedy_matches_the_definition(sampler):
    import torch
    hid, w = head_inputs(3, 512, 20000, seed=4)
    head = sampler.quantize_mx4(w)
    ids = sampler.lm_head_sample(hid, head, params=Params())
    y = hid.double() @ torch.from_numpy(table_values(head)).cuda().T
    top = torch.topk(y, 2, dim=1)
    sure = top.values[:, 0] - top.values[:, 1] > 1e-3
    assert sure.any() and torch.equal(ids.long()[sure], top.indices[sure, 0])


def test_refusals(sampler):
    import torch
    t, x = table(10, 64), torch.zeros((2, 64), device="cuda")
    out = torch.zeros((2, 10), device="cuda")
    u8 = lambda *shape: torch.zeros(shape, dtype=torch.uint8, device="cuda")  # noqa: E731
    with pytest.raises(ValueError, match="uint8"):
        Mx4(t.codes.int(), t.scales, 64)
    with pytest.raises(ValueError, match="32 bytes"):
        Mx4(t.codes[:, :16], t.scales, 64)
    with pytest.raises(ValueError, match="same rows"):
        Mx4(t.codes[:5], t.scales, 64)
    with pytest.raises(SasError, match="codes must be 16-byte aligned"):
        sampler.project_mx4(x, Mx4(u8(10, 48)[:, 8:], t.scales, 64))
    with pytest.raises(SasError, match="codes_stride"):
        sampler.project_mx4(x, Mx4(u8(10, 40), t.scales, 64))
    with pytest.raises(SasError, match="scales_stride"):
        sampler.project_mx4(x, Mx4(t.codes, u8(10, 7), 64))
    with pytest.raises(SasError, match="scales must be 4-byte aligned"):
        sampler.project_mx4(x, Mx4(t.codes, u8(10, 8)[:, 2:], 64))
    with pytest.raises(SasError, match="multiple of 8"):
        sampler.project_mx4(torch.zeros((2, 60), device="cuda"), table(10, 60))
    with pytest.raises(SasError, match="x must be 16-byte aligned"):
        sampler.project_mx4(torch.zeros((2, 72), device="cuda")[:, 1:65], t)
    with pytest.raises(SasError, match="x_stride"):
        sampler.project_mx4(torch.zeros((2, 66), dtype=torch.bfloat16, device="cuda")[:, :64], t)
    for bad in (-1.0, float("inf"), float("nan"), 1e-40):
        with pytest.raises(SasError, match="softcap"):
            sampler.project_mx4(x, t, softcap=bad)
    with pytest.raises(ValueError, match="fit together"):
        sampler.project_mx4(x[:, :32], t)
    with pytest.raises(ValueError, match="accumulate"):
        sampler.project_mx4(x, t, accumulate=True)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        sampler.project_mx4(x.half(), t)
    with pytest.raises(ValueError, match="x's dim"):
        sampler.quantize_mx4_into(x, t.__class__.empty(2, 65))
    with pytest.raises(ValueError, match="rows of x's dim"):
        sampler.quantize_mx4_into(x, Mx4.empty(1, 64))
    with pytest.raises(SasError, match="without ids"):
        sampler.lookup_mx4_into(t, torch.zeros((11, 64), device="cuda"))
    with pytest.raises(ValueError, match="one id per row"):
        sampler.lookup_mx4_into(t, torch.zeros((3, 64), device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="integer"):
        sampler.lookup_mx4(t, torch.zeros(2, dtype=torch.int64, device="cuda"))
    hid = torch.zeros((1, 256), device="cuda")
    with pytest.raises(ValueError, match="dim differs"):
        sampler.lm_head_sample(hid, t, params=Params())
    with pytest.raises(ValueError, match="needs an Mx4"):
        sampler.lm_head_sample(hid, u8(10, 128), fmt=4, params=Params())
    with pytest.raises(ValueError, match="HEAD_MX4"):
        sampler.lm_head_sample(hid, table(10, 256), fmt=W.HEAD_Q6_K, params=Params())
    with pytest.raises(SasError, match="scales_stride"):
        sampler.lm_head_sample(hid, Mx4(u8(10, 128), u8(10, 9), 256), params=Params())
    with pytest.raises(ValueError, match="vocab exceeds"):
        sampler.lm_head_sample(hid, table(10, 256), vocab=11, params=Params())
    with pytest.raises(ValueError, match="must be an Mx4"):
        sampler.project_mx4(x, torch.zeros((10, 64), device="cuda"))
    # nothing of no rows
    assert sampler.project_mx4(x[:0], t).shape == (0, 10)
    assert sampler.quantize_mx4(x[:0]).shape == (0, 64)
    assert sampler.lookup_mx4(t, torch.zeros(0, dtype=torch.int32, device="cuda")).shape == (0, 64)


def test_a_tied_head_in_four_bits(sampler):
    """The operators as they are used: the table laid out once, the tokens'
    embeddings looked up, a batch's logits with the adapters' terms behind
    them, filtered sampling, the next embeddings; eager and as a graph, on a
    stream of its own, with other work between the replays."""
    import torch
    rows, dim, vocab = 12, 256, 5003
    g = torch.Generator(device="cuda").manual_seed(2)
    normal = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    weight = normal(vocab, dim) * 0.1
    pool = Adapters((normal(3, 8, dim) / 16).bfloat16(), normal(3, vocab, 8).bfloat16())
    which = torch.tensor([i % 4 - 1 for i in range(rows)], dtype=torch.int32, device="cuda")
    u = torch.rand(rows, dtype=torch.float64, device="cuda")
    ids = torch.randint(0, vocab, (rows,), dtype=torch.int32, device="cuda")
    first = ids.clone()
    held = Mx4.empty(vocab, dim)
    acts = Mx4.empty(rows, dim)
    hidden, logits = torch.empty((rows, dim), device="cuda"), torch.empty((rows, vocab), device="cuda")

    def step():
        sampler.lookup_mx4_into(held, hidden, ids)
        hidden.mul_(8.0)
        sampler.quantize_mx4_into(hidden, acts)
        sampler.project_mx4_into(acts, held, logits)
        sampler.project_into(hidden, None, logits, adapters=pool, row_adapter=which, accumulate=True, softcap=30.0)
        sampler.sample_filtered_into(logits, ids, uniforms=u, params=FilterParams(temperature=0.8, top_p=0.9, min_p=0.02))

    sampler.quantize_mx4_into(weight, held)
    sampler.reserve_project(rows, dim, rank=8)
    sampler.reserve_filtered(rows, vocab)
    want = []
    for _ in range(4):
        step()
        want.append((ids.clone(), logits.clone()))
    w = torch.from_numpy(table_values(held)).cuda()
    x = torch.from_numpy(R.values(*R.quantize((8 * w[first.long()]).cpu().numpy()), dim)).cuda()
    y, size = x @ w.T, x.abs() @ w.abs().T
    for r in range(rows):
        if which[r] >= 0:
            a, b, h = pool.a[which[r]].double(), pool.b[which[r]].double(), 8 * w[first[r].long()]
            y[r] += b @ (a @ h)
            size[r] += b.abs() @ (a.abs() @ h.abs())
    # f32 sums of dim terms, of 3 dim and 3 x 8 in the adapters' terms; the cap
    tol = (4 * dim + 64) * 2.0 ** -23 * size + 2.0 ** -20 * 30.0
    assert ((want[0][1].double() - 30.0 * torch.tanh(y / 30.0)).abs() <= tol).all()
    stream = torch.cuda.Stream()
    ids.copy_(first)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    ids.copy_(first)
    torch.cuda.synchronize()
    for n in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ids, want[n][0]) and torch.equal(logits, want[n][1])
        sampler.project_mx4(hidden, held)                        # eager work between the replays
        torch.zeros(1 << 20, device="cuda").sum().item()


def test_head_in_a_captured_decode_loop(sampler):
    """sas_lm_head_sample_step with an MXFP4 head, its scratch reserved and no
    eager call before the capture: the tokens of eager steps."""
    import torch
    from shared_amd import DecodeState, Sampler
    rows, dim, vocab, steps = 2, 512, 3000, 5
    hid, w = head_inputs(rows, dim, vocab, seed=9)
    head = sampler.quantize_mx4(w)
    embed = w.mul(4.0)
    params = Params(temperature=1.0, top_k=30, top_p=0.95, presence_penalty=0.5)

    def run(s, graph):
        st = DecodeState(rows, max_steps=steps, seeds=np.arange(7, 7 + rows, dtype=np.uint32))
        h, ids = hid.clone(), torch.empty(rows, dtype=torch.int32, device="cuda")

        def step():
            s.lm_head_step_into(h, head, ids, st, params=params)
            h.copy_(embed.index_select(0, ids))
        if not graph:
            for _ in range(steps):
                step()
        else:
            g = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(g):
                step()
            for _ in range(steps):
                g.replay()
                torch.cuda.synchronize()
                torch.ones(1 << 16, device="cuda").cumsum(0)
        torch.cuda.synchronize()
        return st.sampled.cpu().numpy()
    want = run(sampler, False)
    with Sampler(0) as s:
        s.reserve(rows=rows, vocab=vocab, lm_head_rows=rows, hist_ids=rows * 512)
        assert np.array_equal(run(s, True), want)


def test_offsets_past_32_bits(sampler):
    """Tables and hidden states of more than 4 GiB: the last rows are what they are
    alone."""
    import torch
    rows, dim = 3_400_000, 2560
    small = table(300, dim, seed=4)
    big = Mx4(torch.zeros((rows, 1280), dtype=torch.uint8, device="cuda"), torch.zeros((rows, 80), dtype=torch.uint8, device="cuda"), dim)
    big.codes[-300:], big.scales[-300:] = small.codes, small.scales
    ids = torch.tensor([rows - 1, 0, rows - 300, rows], dtype=torch.int32, device="cuda")
    got, want = sampler.lookup_mx4(big, ids), sampler.lookup_mx4(small)
    assert torch.equal(got[0], want[299]) and torch.equal(got[2], want[0]) and not got[1].any() and not got[3].any()
    for n, kind in ((2, torch.float32), (12, torch.bfloat16), (70, torch.bfloat16)):
        x = torch.randn((n, dim), device="cuda").to(kind)
        y = sampler.project_mx4(x, big, out_dtype=torch.bfloat16)
        p = Product.__new__(Product)
        p.x, p.value, p.weight = x, x.double(), torch.from_numpy(table_values(small)).cuda()
        p.check(y[:, -300:])
        assert not y[:, :-300].any()
        del y
    del big
    x = torch.zeros((rows // 4, dim), device="cuda")     # 8.7 GB of f32
    x[-3:] = torch.randn((3, dim), device="cuda")
    q, alone = sampler.quantize_mx4(x), sampler.quantize_mx4(x[-3:])
    assert torch.equal(q.codes[-3:], alone.codes) and torch.equal(q.scales[-3:], alone.scales)
    assert not q.codes[:-3].any() and not q.scales[:-3].any()


def test_more_rows_than_a_launch_has_threads_for(sampler):
    """2^28 rows and more of one value: 16 lanes each would be 2^32 threads."""
    import torch
    rows = (1 << 28) + 77
    x = torch.zeros((rows, 1), dtype=torch.bfloat16, device="cuda")
    x[0], x[-1], x[rows // 2], x[1 << 26] = 3.0, -0.75, 5.0, 1.5
    q = sampler.quantize_mx4(x)
    out = torch.full_like(x, 7.0)
    sampler.lookup_mx4_into(q, out)
    want = sampler.lookup_mx4(sampler.quantize_mx4(x[rows // 2:rows // 2 + 1]), out_dtype=torch.bfloat16)
    x[rows // 2] = want[0]
    assert torch.equal(out, x)
    f32 = torch.full((rows, 1), 7.0, device="cuda")
    sampler.lookup_mx4_into(q, f32)
    assert torch.equal(f32, x.float())


@pytest.mark.parametrize("rows", [3, 20, 50])
def test_rows_far_apart(sampler, rows):
    """Strides that pass the kernels' 32-bit offsets within a tile."""
    import torch
    dim, out = 64, 9000
    p = Product(rows, dim, out, "bfloat16", seed=rows)
    far = torch.empty(((rows - 1) << 24) + dim, dtype=torch.bfloat16, device="cuda").as_strided((rows, dim), (1 << 24, 1))
    far.copy_(p.x)
    p.check(sampler.project_mx4(far, p.w))
    there = torch.empty(((rows - 1) << 25) + out, device="cuda").as_strided((rows, out), (1 << 25, 1))
    sampler.project_mx4_into(p.x, p.w, there)
    p.check(there)


def test_accumulate_then_cap_and_nan_in_bf16(sampler):
    import torch
    for rows, out in ((2, 9000), (40, 64), (40, 40000)):
        for kind in ("float32", "bfloat16", "mx4"):
            p = Product(rows, 256, out, kind, seed=out)
            held = torch.randn((rows, out), device="cuda")
            got = held.clone()
            sampler.project_mx4_into(p.x, p.w, got, accumulate=True, softcap=10.0)
            p.check(got, cap=10.0, extra=held.double())
            p.w.scales[7, 2] = 255
            y = sampler.project_mx4(p.x, p.w, out_dtype=torch.bfloat16, softcap=10.0)
            assert y[:, 7].isnan().all() and y[:, :7].isfinite().all() and y[:, 8:].isfinite().all()


def test_other_streams(sampler):
    """On a stream of the caller's, behind work that fills the inputs there."""
    import torch
    st = torch.cuda.Stream()
    x = torch.zeros((64, 2048), device="cuda")
    src = torch.randn((64, 2048), device="cuda")
    w = table(4000, 2048)
    want = sampler.project_mx4(sampler.quantize_mx4(src), w)
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        for _ in range(50):
            x.add_(1.0)
        x.copy_(src)
    q = sampler.quantize_mx4(x, stream=st)
    got = sampler.project_mx4(q, w, stream=st)
    back = sampler.lookup_mx4(q, stream=st)
    st.synchronize()
    assert torch.equal(got, want) and torch.equal(back, sampler.lookup_mx4(sampler.quantize_mx4(src)))
