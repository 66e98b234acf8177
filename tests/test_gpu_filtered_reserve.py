"""sas_reserve_filtered covers every call of at most its rows and vocabulary:
smaller vocabularies, which may be cut into more parts, included."""
import gc

import numpy as np
import pytest

from shared_amd import FilterParams, Sampler

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_collection():
    # a graph that the collector destroys while another is being recorded aborts
    gc.collect()
    gc.disable()
    yield
    gc.enable()


# A row's parts hold 8,192 ids, and 4,096 or 2,048 where fewer than two parts a CU would
# come of that: shapes just below those limits for 256 CUs need the most scratch.
@pytest.mark.parametrize("rows,vocab,smaller", [
    (16, 262144, [(16, 250000), (16, 126976), (16, 122880), (15, 137217), (1, 262144), (16, 131072)]),
    (64, 50257, [(63, 30721), (64, 28672), (64, 28673), (63, 32768), (33, 30720)]),
    (96, 32000, [(96, 18433), (96, 18432), (96, 20480), (85, 24576), (51, 20480)]),
    (1, 300000, [(1, 299999), (1, 5)]),
    (600, 9000, [(600, 8192), (300, 8192), (512, 8193), (256, 4096), (511, 2048)])])
def test_smaller_calls_are_captured(rows, vocab, smaller):
    import torch
    p = FilterParams(temperature=1.0, top_p=0.9)
    rng = np.random.default_rng(rows)
    for n, width in smaller:
        print(f"[gpu] reserve {rows} x {vocab}, call {n} x {width}", flush=True)
        v = torch.randn((n, width), device="cuda") * 3
        u = torch.from_numpy(rng.random(n)).cuda()
        ids = torch.full((n,), -5, dtype=torch.int32, device="cuda")
        with Sampler(0) as fresh, Sampler(0) as eager:
            fresh.reserve_filtered(rows, vocab)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                fresh.sample_filtered_into(v, ids, uniforms=u, params=p)
            for _ in range(2):
                g.replay()
                torch.cuda.synchronize()
                want = eager.sample_filtered(v, uniforms=u, params=p)
                torch.cuda.synchronize()
                assert torch.equal(ids, want)
                v.normal_().mul_(3)


def test_a_call_out_of_reserve_names_the_way_out():
    import torch
    from shared_amd import SasError
    v = torch.zeros((4, 30000), device="cuda")
    u = torch.zeros(4, dtype=torch.float64, device="cuda")
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    x, w = torch.zeros((4, 64), device="cuda"), torch.zeros((32, 64), dtype=torch.bfloat16, device="cuda")
    y = torch.zeros((4, 32), device="cuda")
    with Sampler(0) as s:
        for call, name in ((lambda: s.sample_filtered_into(v, ids, uniforms=u, params=FilterParams(temperature=1.0)),
                            "sas_reserve_filtered"), (lambda: s.project_into(x, w, y), "sas_reserve_project")):
            g = torch.cuda.CUDAGraph()
            with pytest.raises(SasError, match=name):
                with torch.cuda.graph(g):
                    call()
            torch.cuda.synchronize()
