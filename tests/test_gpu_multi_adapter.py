"""The example that runs sas_project and sas_sample_filtered together: eager
and recorded steps draw the same tokens."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("rows", [1, 5, 40])
def test_example(rows):
    import torch
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import multi_adapter_decode as example
    print(f"[gpu] multi-adapter decode rows={rows}", flush=True)
    eager = example.decode(rows=rows, steps=5, vocab=5003, dim=256, graph=False)
    recorded = example.decode(rows=rows, steps=5, vocab=5003, dim=256, graph=True)
    assert torch.equal(eager, recorded)
    assert ((eager >= 0) & (eager < 5003)).all()
