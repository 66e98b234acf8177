"""The Node layer's project and sampleFiltered against the Python mirror on the
same inputs: the same bits."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

from shared_amd import Adapters, FilterParams, pack_filter_params

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_node_decode(tmp_path, sampler):
    if shutil.which("node") is None:
        pytest.skip("node is not installed")
    import torch
    rows, vocab, dim, n, rank = 6, 4099, 256, 3, 8
    rng = np.random.default_rng(2)
    x = rng.standard_normal((rows, dim)).astype(np.float32)
    w, a, b = (torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).bfloat16()
               for shape in ((vocab, dim), (n, rank, dim), (n, vocab, rank)))
    which = rng.integers(-1, n, rows).astype(np.int32)
    u = rng.random(rows)
    allowed = rng.random((rows, (vocab + 31) // 32 * 32)) < 0.3
    allowed[:, vocab:] = False
    mask = np.packbits(allowed, axis=1, bitorder="little").view(np.uint32)
    params = [dict(temperature=1.0 + 0.1 * r, topP=0.9, minP=0.01, topK=100 * r) for r in range(rows)]
    for name, data in (("x.f32", x), ("w.u16", w.view(torch.int16).numpy()), ("a.u16", a.view(torch.int16).numpy()),
                       ("b.u16", b.view(torch.int16).numpy()), ("which.i32", which), ("u.f64", u), ("mask.u32", mask)):
        np.ascontiguousarray(data).tofile(tmp_path / name)
    (tmp_path / "meta.json").write_text(json.dumps(dict(rows=rows, vocab=vocab, dim=dim, adapters=n, rank=rank, params=params)))
    print("[gpu] node decode", flush=True)
    run = subprocess.run(["node", os.path.join(ROOT, "tests", "node", "decode_gpu.js"), str(tmp_path)], capture_output=True,
                         text=True, timeout=100)
    assert run.returncode == 0, run.stdout + run.stderr
    dev = lambda t: torch.from_numpy(t).cuda()  # noqa: E731
    logits = sampler.project(dev(x), w.cuda(), adapters=Adapters(a.cuda(), b.cuda()), row_adapter=dev(which), softcap=30.0)
    assert np.array_equal(np.fromfile(tmp_path / "logits.f32", np.float32).reshape(rows, vocab), logits.cpu().numpy())
    plist = [FilterParams(temperature=p["temperature"], top_p=p["topP"], min_p=p["minP"], top_k=p["topK"]) for p in params]
    one = sampler.sample_filtered(logits, uniforms=dev(u), params=plist[0], full=True)
    assert np.array_equal(np.fromfile(tmp_path / "one_ids.u32", np.int32), one["ids"].cpu().numpy())
    assert np.array_equal(np.fromfile(tmp_path / "one_probs.f64", np.float64), one["probs"].cpu().numpy())
    each = sampler.sample_filtered(logits, uniforms=dev(u), row_params=dev(pack_filter_params(plist).view(np.uint8)),
                                   mask=dev(mask.view(np.int32)), full=True)
    assert np.array_equal(np.fromfile(tmp_path / "each_ids.u32", np.int32), each["ids"].cpu().numpy())
    assert np.array_equal(np.fromfile(tmp_path / "each_counts.i32", np.int32), each["counts"].cpu().numpy())
