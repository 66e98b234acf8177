"""MXFP4 products at shapes chosen by the kernel that takes them (256 CUs),
wherever the shapes of the other tests take another: every form that a call can
reach, over several super-runs of 512 values and several groups of outputs a
block, with and without a last block cut short; and the largest strides that the
kernels' 32-bit offsets take."""
import pytest

from shared_amd import Mx4, Params
from test_gpu_mx4_scales import values

pytestmark = pytest.mark.gpu


def table(rows, dim, seed, pad=0):
    """Every code, scales around 1; NaN scales behind the rows' last blocks."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    blocks = (dim + 31) // 32
    codes = torch.randint(0, 256, (rows, 16 * (blocks + pad)), generator=g, device="cuda", dtype=torch.uint8)
    if dim % 32:
        last = codes[:, 16 * (blocks - 1):16 * blocks]
        keep = dim - 32 * (blocks - 1)                       # values of the last block
        at = torch.arange(16, device="cuda")
        last &= torch.where(2 * at + 1 < keep, 255, torch.where(2 * at < keep, 15, 0)).to(torch.uint8)
    scales = torch.full((rows, (blocks + 3) // 4 * 4 + 4 * pad), 255, dtype=torch.uint8, device="cuda")
    scales[:, :blocks] = torch.randint(121, 131, (rows, blocks), generator=g, device="cuda", dtype=torch.uint8)
    return Mx4(codes, scales, dim)


def hidden(rows, dim, kind, seed):
    """Hidden states and their float64 values."""
    import torch
    if kind == "mx4":
        x = table(rows, dim, seed)
        return x, values(x.codes, x.scales, dim)
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, dim), generator=g, device="cuda").to(getattr(torch, kind))
    return x, x.double()


def some(n, most, seed):
    """Indexes below n: all of them, or the first and last and a sample between."""
    import torch
    if n <= most:
        return torch.arange(n, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(seed)
    edge = most // 4
    return torch.cat([torch.arange(edge, device="cuda"), edge + torch.randperm(n - 2 * edge, generator=g, device="cuda")[:most - 2 * edge],
                      torch.arange(n - edge, n, device="cuda")])


def check(got, value, w, dim, terms, rows=None):
    """Sampled rows and outputs against the 64-bit product: f32 sums of exact
    products, a rounding of 2^-23 (a cut one) a term and 32 for the joins of the
    waves' sums, and half a step of bf16 results."""
    import torch
    cols = some(got.shape[1], 1536, got.shape[1])
    rows = some(got.shape[0], 256, got.shape[0]) if rows is None else rows
    weight = values(w.codes[cols], w.scales[cols], dim)
    value = value[rows]
    want, size = value @ weight.T, value.abs() @ weight.abs().T
    part = got[rows[:, None], cols].double()
    tol = (terms + 32) * 2.0 ** -23 * size
    if got.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * want.abs()
    off = (part - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), part[bad][:4].tolist(), want[bad][:4].tolist())
    # a block of 32 left out or taken twice would show here
    if got.dtype == torch.float32:
        assert float(off.norm()) <= 2.0 ** -20 * float(size.norm())
    assert got.isfinite().all()


# rows, dim, outputs, hidden states, the kernel (waves' rows and outputs in 16s)
KERNELS = [
    # split: <1, 1>, <1, 2> for up to 5 f32 rows, <2, 2>, <4, 2>
    (5, 1096, 4000, "float32", "split 1 1"), (16, 3000, 4096, "bfloat16", "split 1 1"), (9, 2081, 1000, "mx4", "split 1 1"),
    (1, 5120, 20000, "float32", "split 1 2"), (3, 5120, 20000, "float32", "split 1 2"), (5, 12288, 9000, "float32", "split 1 2"),
    (2, 8200, 4700, "float32", "split 1 2"),
    (24, 2560, 2560, "float32", "split 2 2"), (24, 2600, 2560, "bfloat16", "split 2 2"), (32, 2560, 2561, "mx4", "split 2 2"),
    (64, 4096, 4000, "float32", "split 4 2"), (61, 2600, 4001, "bfloat16", "split 4 2"), (100, 4097, 2000, "mx4", "split 4 2"),
    # stream: packed f32, bf16, MXFP4 rows of one, two and four subtiles
    (5, 4096, 50000, "float32", "stream packed"), (2, 1544, 9000, "float32", "stream packed"),
    (16, 4096, 30000, "bfloat16", "stream 1"), (7, 1544, 9000, "bfloat16", "stream 1"),
    (16, 8192, 30000, "mx4", "stream 1"), (32, 8192, 9000, "mx4", "stream 2"), (20, 1537, 9000, "mx4", "stream 2"),
    (61, 4096, 11007, "mx4", "stream 4"), (50, 2081, 70000, "mx4", "stream 4"),
    # the largest products that are timed
    (16, 2560, 151936, "float32", "wide 1 3"), (2048, 4096, 4096, "bfloat16", "wide 8 2"), (8192, 4096, 11008, "mx4", "wide 8 2"),
    (2048, 1024, 4096, "float32", "wide 4 2"),
]
# wide, of 16 rows up to 128: dims past what the other kernels hold, whole super-runs
# and not; outputs for one to three 16s a wave, blocks with several groups of them
for sub, most, dims in ((1, 3, dict(float32=(2048, 1544), bfloat16=(4608, 4616), mx4=(16896, 16500))),
                        (2, 2, dict(float32=(2048, 1544), bfloat16=(2048, 1544), mx4=(8704, 8449))),
                        (4, 2, dict(float32=(2048, 1544), bfloat16=(2048, 1544), mx4=(4608, 4353))),
                        (8, 2, dict(bfloat16=(2048, 1544), mx4=(2048, 1537)))):
    for kind, (whole, cut) in dims.items():
        for n, out in enumerate((20000 if sub == 1 else 70000, 128256, 151936)[:most], 1):
            KERNELS += [(16 * sub, whole, out, kind, f"wide {sub} {n}"), (16 * sub - 5, cut, out, kind, f"wide {sub} {n}")]
# many tiles of rows
for kind, dims, sub in (("float32", (2048, 1544), 4), ("bfloat16", (2048, 1544), 8), ("mx4", (1536, 1537), 8)):
    for dim in dims:
        KERNELS += [(300, dim, 4000, kind, f"wide {sub} 1"), (700, dim, 9000, kind, f"wide {sub} 2")]


@pytest.mark.parametrize("rows,dim,out,kind,kernel", KERNELS)
def test_every_kernel(sampler, rows, dim, out, kind, kernel):
    import torch
    print(f"[gpu] project_mx4 {rows} x {dim} x {out} {kind}: {kernel}", flush=True)
    w = table(out, dim, seed=rows + out)
    x, value = hidden(rows, dim, kind, seed=dim)
    terms = dim * (3 if kind == "float32" else 1)
    got = sampler.project_mx4(x, w)
    check(got, value, w, dim, terms)
    half = sampler.project_mx4(x, w, out_dtype=torch.bfloat16)
    # the same sums, rounded once
    assert torch.equal(half, got.bfloat16())


@pytest.mark.parametrize("rows,dim,vocab", [(1, 5120, 50257), (1, 8192, 20000), (2, 6144, 9000)])
def test_heads_past_the_streams_lds(sampler, rows, dim, vocab):
    import torch
    print(f"[gpu] mx4 head {rows} x {dim} x {vocab}", flush=True)
    w = table(vocab, dim, seed=vocab)
    x, value = hidden(rows, dim, "float32", seed=dim)
    u = torch.rand(rows, dtype=torch.float64, device="cuda")
    kw = dict(uniforms=u, params=Params(temperature=0.9, top_k=40, top_p=0.95))
    r = sampler.lm_head_sample(x, w, logits=True, **kw)
    check(r["logits"], value, w, dim, 3 * dim)
    assert torch.equal(r["ids"], sampler.sample(r["logits"], **kw))


@pytest.mark.parametrize("rows,kind,x_far,out_far", [
    # far strides go to the split kernel, whatever the shape
    (3, "float32", 0, 1 << 25), (12, "float32", 1 << 23, 0), (20, "float32", 1 << 23, 0), (50, "float32", 0, 1 << 25), (5, "float32", 1 << 24, 0),
    (10, "mx4", 1 << 23, 0), (20, "mx4", 0, 1 << 25), (70, "mx4", 1 << 24, 0), (70, "bfloat16", 1 << 23, 1 << 25),
    # the largest that the other kernels take
    (3, "float32", (1 << 23) - 4, (1 << 25) - 1), (16, "float32", (1 << 23) - 4, (1 << 25) - 1), (64, "float32", (1 << 23) - 4, 0),
    (130, "float32", (1 << 23) - 4, 0), (16, "bfloat16", (1 << 23) - 8, (1 << 25) - 1), (128, "bfloat16", (1 << 23) - 8, 0),
    (140, "bfloat16", (1 << 23) - 8, (1 << 25) - 1), (16, "mx4", (1 << 23) - 16, 0), (61, "mx4", (1 << 23) - 16, (1 << 25) - 1),
    (200, "mx4", (1 << 23) - 16, 0)])
def test_strides_around_the_32_bit_offsets(sampler, rows, kind, x_far, out_far):
    """x_far: elements (MXFP4: bytes) between rows of hidden states, out_far between
    rows of the result (0: as they come)."""
    import torch
    dim, out = 64, 9000
    print(f"[gpu] project_mx4 {rows} x {dim} x {out} {kind}, rows {x_far} and {out_far} apart", flush=True)
    w = table(out, dim, seed=rows)
    x, value = hidden(rows, dim, kind, seed=rows + 1)

    def apart(t, stride):
        far = torch.empty((rows - 1) * stride + t.shape[1], dtype=t.dtype, device="cuda").as_strided(t.shape, (stride, 1))
        far.copy_(t)
        return far
    if x_far:
        x = Mx4(apart(x.codes, x_far), apart(x.scales, x_far), dim) if kind == "mx4" else apart(x, x_far)
    if out_far:
        y = torch.empty((rows - 1) * out_far + out, device="cuda").as_strided((rows, out), (out_far, 1))
    else:
        y = torch.empty((rows, out), device="cuda")
    sampler.project_mx4_into(x, w, y)
    check(y, value, w, dim, dim * (3 if kind == "float32" else 1))
