"""MXFP4 products with the largest scales: a value that a block holds is finite,
and what another block's codes would be under its scale is not."""
import pytest

from shared_amd import Mx4

pytestmark = pytest.mark.gpu

# 0 0.5 1 1.5 2 3 4 6, then their negatives
ELEMENTS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def values(codes, scales, dim):
    """float64 [n][dim] of a table's rows."""
    import torch
    n, blocks = codes.shape[0], (dim + 31) // 32
    c = codes[:, :16 * blocks].int()
    pair = torch.stack((c & 15, c >> 4), 2).view(n, 32 * blocks)
    element = torch.tensor(ELEMENTS + [-v for v in ELEMENTS], dtype=torch.float64, device=codes.device)
    unit = torch.exp2(scales[:, :blocks].double() - 127)
    return (element[pair.long()].view(n, blocks, 32) * unit[:, :, None]).view(n, -1)[:, :dim]


def spiked_table(rows, dim, seed):
    """Blocks of 6 and -6 under scales up to 2^120; in each row one block of the
    scale 2^127 with elements up to 1.5, or of 2^126 with elements up to 3: 6
    under either passes f32's range."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    blocks = (dim + 31) // 32
    pair = torch.where(torch.rand((rows, blocks, 32), generator=g, device="cuda") < 0.5, 7, 15)
    scales = torch.full((rows, (blocks + 3) // 4 * 4), 255, device="cuda")
    scales[:, :blocks] = torch.randint(240, 248, (rows, blocks), generator=g, device="cuda")
    at = torch.randint(0, blocks, (rows,), generator=g, device="cuda")
    top = torch.randint(253, 255, (rows,), generator=g, device="cuda")
    row = torch.arange(rows, device="cuda")
    scales[row, at] = top
    small = torch.rand((rows, 32), generator=g, device="cuda") * torch.where(top == 254, 4, 6)[:, None]
    pair[row, at] = small.long() + 8 * torch.randint(0, 2, (rows, 32), generator=g, device="cuda")
    pair = pair.view(rows, -1)
    pair[:, dim:] = 0
    return Mx4((pair[:, 0::2] + 16 * pair[:, 1::2]).to(torch.uint8), scales.to(torch.uint8), dim)


@pytest.mark.parametrize("x_kind", ["float32", "bfloat16", "mx4"])
@pytest.mark.parametrize("rows,dim,out", [(1, 2560, 300), (3, 1064, 77), (3, 2560, 9000), (4, 5120, 9000), (12, 2600, 500), (24, 2600, 300),
                                          (50, 2560, 600), (16, 4608, 5000), (60, 520, 9000), (300, 2600, 3001)])
def test_scales_near_the_top_stay_in_their_blocks(sampler, rows, dim, out, x_kind):
    """Hidden states around 2^-100 bring the sums back into range (all f32 bits
    of them are kept there).  f32 sums of exact products: a rounding of 2^-23 a term,
    three terms a product with f32 hidden states, and of the joins of the waves'
    sums."""
    import torch
    print(f"[gpu] project_mx4 {rows} x {dim} x {out} {x_kind}, scales near the top", flush=True)
    w = spiked_table(out, dim, seed=rows + dim)
    g = torch.Generator(device="cuda").manual_seed(dim)
    x = torch.randn((rows, dim), generator=g, device="cuda") * 2.0 ** -100
    if x_kind == "mx4":
        x = sampler.quantize_mx4(x)
        value = values(x.codes, x.scales, dim)
    else:
        x = x.to(getattr(torch, x_kind))
        value = x.double()
    weight = values(w.codes, w.scales, dim)
    want, size = value @ weight.T, value.abs() @ weight.abs().T
    tol = ((3 if x_kind == "float32" else 1) * dim + 32) * 2.0 ** -23 * size
    assert want.isfinite().all() and float(weight.abs().max()) > 2.0 ** 127
    got = sampler.project_mx4(x, w).double()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), got[bad][:4].tolist(), want[bad][:4].tolist())


@pytest.mark.parametrize("rows,dim,vocab", [(1, 2560, 300), (3, 4096, 900), (1, 5120, 9000)])
def test_a_head_with_scales_near_the_top(sampler, rows, dim, vocab):
    import torch
    from shared_amd import Params
    head = spiked_table(vocab, dim, seed=dim)
    x = torch.randn((rows, dim), device="cuda") * 2.0 ** -100
    r = sampler.lm_head_sample(x, head, params=Params(), logits=True)
    weight = values(head.codes, head.scales, dim)
    want, size = x.double() @ weight.T, x.double().abs() @ weight.abs().T
    assert ((r["logits"].double() - want).abs() <= (3 * dim + 32) * 2.0 ** -23 * size).all()
    assert torch.equal(r["ids"].long(), r["logits"].argmax(1))


@pytest.mark.parametrize("rows", [2, 20])
def test_small_f32_hidden_states_keep_their_bits_down_to_bf16s_last(sampler, rows):
    """A value alone in its sum, under a weight of 2^100: exact but for bits below
    2^-133, which are cut off."""
    import torch
    codes = torch.zeros((40, 16), dtype=torch.uint8, device="cuda")
    codes[:, 0] = 2                                                   # 1
    w = Mx4(codes, torch.full((40, 4), 227, dtype=torch.uint8, device="cuda"), 32)
    for e in range(-126, -99):
        x = torch.zeros((rows, 32), device="cuda")
        x[:, 0] = 2.0 ** e * (2 - 2.0 ** -23)
        got = sampler.project_mx4(x, w).double()
        want = torch.floor(x[0, 0].double() * 2.0 ** 133) * 2.0 ** -33
        assert (got == want).all(), (e, float(got[0, 0]), float(want))
