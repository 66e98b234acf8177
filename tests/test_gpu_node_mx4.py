"""The Node layer's MXFP4 calls against the Python mirror on the same inputs: the
same bits."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

from shared_amd import Params

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_node_mx4(tmp_path, sampler):
    if shutil.which("node") is None:
        pytest.skip("node is not installed")
    import torch
    rows, vocab, dim, n = 3, 4099, 512, 9
    rng = np.random.default_rng(3)
    x = rng.standard_normal((rows, dim)).astype(np.float32)
    w = torch.from_numpy((0.1 * rng.standard_normal((vocab, dim))).astype(np.float32)).bfloat16()
    ids = rng.integers(0, vocab, n).astype(np.uint32)
    ids[4] = 0xFFFFFFFF
    u = rng.random(rows)
    for name, data in (("x.f32", x), ("w.u16", w.view(torch.int16).numpy()), ("ids.u32", ids), ("u.f64", u)):
        np.ascontiguousarray(data).tofile(tmp_path / name)
    (tmp_path / "meta.json").write_text(json.dumps(dict(rows=rows, vocab=vocab, dim=dim, ids=n)))
    print("[gpu] node mx4", flush=True)
    run = subprocess.run(["node", os.path.join(ROOT, "tests", "node", "mx4_gpu.js"), str(tmp_path)], capture_output=True,
                         text=True, timeout=100)
    assert run.returncode == 0, run.stdout + run.stderr
    dev = lambda t: torch.from_numpy(t).cuda()  # noqa: E731
    head = sampler.quantize_mx4(w.cuda())
    f32 = lambda name, *shape: np.fromfile(tmp_path / name, np.float32).reshape(shape)  # noqa: E731
    assert np.array_equal(f32("wide.f32", rows, vocab), sampler.project_mx4(dev(x), head, softcap=30.0).cpu().numpy())
    once = sampler.project_mx4(sampler.quantize_mx4(dev(x)), head)
    assert np.array_equal(f32("twice.f32", rows, vocab), (once + once).cpu().numpy())
    assert np.array_equal(f32("rows.f32", n, dim), sampler.lookup_mx4(head, dev(ids.view(np.int32))).cpu().numpy())
    got = sampler.lm_head_sample(dev(x), head, uniforms=dev(u), params=Params(temperature=0.9, top_k=40, top_p=0.95))
    assert np.array_equal(np.fromfile(tmp_path / "ids.out", np.int32), got.cpu().numpy())
    assert np.array_equal(np.fromfile(tmp_path / "greedy.out", np.int32), sampler.lm_head_sample(dev(x), head, params=Params()).cpu().numpy())
