"""sas_project on both sides of the choice between its kernels (tiles of up to 128
rows x 256 outputs against the compute units), for every tile height."""
import pytest

from test_gpu_project import Problem

pytestmark = pytest.mark.gpu


def shapes():
    for rows in (5, 16, 17, 32, 33, 48, 64, 70, 90, 112, 128, 130, 250, 300, 1000, 1920, 2500):
        tiles = ((rows + 15) // 16 + 7) // 8
        for units in ((96, 256) if rows <= 32 else (96,)):
            outs = -(-units // tiles) * 256
            # the least outputs that fill so many tiles (an odd number), and a tile less
            yield rows, outs - 255
            yield rows, outs - 256


@pytest.mark.parametrize("x", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,out", list(shapes()))
def test_both_sides(sampler, rows, out, x):
    import torch
    print(f"[gpu] project tiles {rows} x {out} {x}", flush=True)
    for dim, n, rank, grouped in ((72, 0, 8, False), (328, 7, 16, False), (640, 3, 40, True)):
        p = Problem(rows, dim, out, n, rank, x=x, seed=rows + n, grouped=grouped)
        p.check(sampler.project(p.x, p.weight, **p.kw()))
        p.check(sampler.project(p.x, p.weight, out_dtype=torch.bfloat16, **p.kw()))
