"""Decode steps of a batch whose requests use adapters of their own.

Each step takes the batch's final-normed hidden states through the shared
head with every request's low-rank adapter (Sampler.project), then draws one
token a request with its own temperature, top-k, top-p and min-p
(Sampler.sample_filtered).  The hidden states are synthetic; a model would
compute them from the tokens fed back.  Both calls are recorded into one HIP
graph after the scratch is sized, and replayed.

    python examples/multi_adapter_decode.py --rows 32 --steps 8
"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from shared_amd import Adapters, FilterParams, Sampler, pack_filter_params  # noqa: E402


def decode(rows=32, steps=8, vocab=32000, dim=2560, adapters=8, rank=16, seed=0, graph=True):
    """Token ids [steps][rows] of `steps` decode steps."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    head = (normal(vocab, dim) * (2.0 / dim ** 0.5)).bfloat16()
    pool = Adapters((normal(adapters, rank, dim) / dim ** 0.5).bfloat16(), normal(adapters, vocab, rank).bfloat16())
    # requests without an adapter have -1
    row_adapter = torch.from_numpy(rng.integers(-1, adapters, rows).astype(np.int32)).cuda()
    requests = [FilterParams(temperature=float(rng.choice([0.0, 0.7, 1.0])), top_p=float(rng.choice([0.9, 1.0])),
                             min_p=float(rng.choice([0.0, 0.05])), top_k=int(rng.choice([0, 50]))) for _ in range(rows)]
    params = torch.from_numpy(pack_filter_params(requests).view(np.uint8)).cuda()
    hidden, uniforms = torch.empty((rows, dim), device="cuda"), torch.empty(rows, dtype=torch.float64, device="cuda")
    logits, ids = torch.empty((rows, vocab), device="cuda"), torch.empty(rows, dtype=torch.int32, device="cuda")
    out = []
    with Sampler(0) as s:
        s.reserve_project(rows, dim, rank=rank)
        s.reserve_filtered(rows, vocab)

        def step():
            s.project_into(hidden, head, logits, adapters=pool, row_adapter=row_adapter, softcap=30.0)
            s.sample_filtered_into(logits, ids, uniforms=uniforms, row_params=params)

        if graph:
            recorded = torch.cuda.CUDAGraph()
            with torch.cuda.graph(recorded):
                step()
        for _ in range(steps):
            hidden.normal_(generator=g)
            uniforms.copy_(torch.from_numpy(rng.random(rows)))
            recorded.replay() if graph else step()
            out.append(ids.clone())
        torch.cuda.synchronize()
    return torch.stack(out)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--rows", type=int, default=32)
    ap.add_argument("--steps", type=int, default=8)
    a = ap.parse_args()
    for t, tokens in enumerate(decode(rows=a.rows, steps=a.steps).tolist()):
        print(f"step {t}: {tokens}")
