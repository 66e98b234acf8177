"""The Node layer's sampleFiltered honours SampleParams.allowedTokenIds as
sampleRows does: one list for every row, a list a row, and its refusals."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

from shared_amd import FilterParams, pack_filter_params

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_allowed_ids(tmp_path, sampler):
    if shutil.which("node") is None:
        pytest.skip("node is not installed")
    import torch
    rows, vocab = 5, 3001
    rng = np.random.default_rng(4)
    v = (rng.standard_normal((rows, vocab)) * 2).astype(np.float32)
    u = rng.random(rows)
    params = [dict(temperature=1.0 + 0.1 * r, topP=0.95, minP=0.001, topK=20 * r) for r in range(rows)]
    lists = [sorted(int(i) for i in rng.choice(vocab, 40, replace=False)) for _ in range(rows)]
    lists[3] = []     # none: the row is free
    v.tofile(tmp_path / "logits.f32")
    u.tofile(tmp_path / "u.f64")
    (tmp_path / "meta.json").write_text(json.dumps(dict(rows=rows, vocab=vocab, params=params, lists=lists)))
    print("[gpu] node sampleFiltered lists", flush=True)
    run = subprocess.run(["node", os.path.join(ROOT, "tests", "node", "lists_gpu.js"), str(tmp_path)], capture_output=True,
                         text=True, timeout=100)
    assert run.returncode == 0, run.stdout + run.stderr
    dev = lambda t: torch.from_numpy(t).cuda()  # noqa: E731
    plist = [FilterParams(temperature=p["temperature"], top_p=p["topP"], min_p=p["minP"], top_k=p["topK"]) for p in params]

    def want(ids, params):
        allowed = np.zeros((rows, (vocab + 31) // 32 * 32), bool)
        for r in range(rows):
            allowed[r, ids[r] or slice(0, vocab)] = True
        mask = np.packbits(allowed, axis=1, bitorder="little").view(np.int32)
        out = sampler.sample_filtered(dev(v), uniforms=dev(u), mask=dev(mask), full=True,
                                      row_params=dev(pack_filter_params(params).view(np.uint8)))
        return out["ids"].cpu().numpy(), out["counts"].cpu().numpy()
    for name, (ids, counts) in (("each", want(lists, plist)), ("shared", want([lists[0]] * rows, [plist[1]] * rows)),
                                ("same", want([lists[0]] * rows, plist)), ("free", want([[]] * rows, plist))):
        assert np.array_equal(np.fromfile(tmp_path / f"{name}_ids.u32", np.int32), ids), name
        assert np.array_equal(np.fromfile(tmp_path / f"{name}_counts.i32", np.int32), counts), name
