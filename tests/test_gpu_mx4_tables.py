"""MXFP4 tables of sizes at the ends of what the calls take."""
import pytest

from shared_amd import Mx4
from test_gpu_mx4_scales import values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["float32", "bfloat16", "float16"])
def test_lookup_in_a_table_of_no_rows(sampler, kind):
    """Every id lies past it: zeros."""
    import torch
    ids = torch.tensor([0, -1, 5], dtype=torch.int32, device="cuda")
    out = sampler.lookup_mx4(Mx4.empty(0, 100), ids, out_dtype=getattr(torch, kind))
    assert out.shape == (3, 100) and not out.any()
    assert sampler.lookup_mx4(Mx4.empty(0, 100)).shape == (0, 100)


@pytest.mark.parametrize("rows,out,kind", [(1, (1 << 27) + 77, "bfloat16"), (3, (1 << 27) + 77, "mx4"), (20, (1 << 28) + 77, "bfloat16")])
def test_more_outputs_than_a_launch_has_threads_for(sampler, rows, out, kind):
    """2^23 tiles of outputs and more, 512 threads each: 2^32.  Every 8 outputs in
    turn, and the last ones, are one small table's."""
    import torch
    dim = 32
    print(f"[gpu] project_mx4 {rows} x {dim} x {out} {kind}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(rows)
    small = torch.randint(0, 256, (8, 16), generator=g, device="cuda", dtype=torch.uint8)
    codes = torch.empty((out, 16), dtype=torch.uint8, device="cuda")
    codes[:out // 8 * 8].view(-1, 128).copy_(small.view(1, 128).expand(out // 8, 128))
    codes[out // 8 * 8:] = small[:out % 8]
    w = Mx4(codes, torch.full((out, 4), 127, dtype=torch.uint8, device="cuda"), dim)
    x = torch.randint(-3, 4, (rows, dim), generator=g, device="cuda").bfloat16()
    # small whole numbers and halves: every sum is exact
    want = (x.double() @ values(small, w.scales[:8], dim).T).bfloat16()
    if kind == "mx4":
        x = sampler.quantize_mx4(x)
    got = sampler.project_mx4(x, w, out_dtype=torch.bfloat16)
    for r in range(rows):
        assert (got[r, :out // 8 * 8].view(-1, 8) == want[r]).all()
        assert torch.equal(got[r, out // 8 * 8:], want[r, :out % 8])
