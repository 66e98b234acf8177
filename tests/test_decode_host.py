"""sas_project and sas_sample_filtered without a GPU: the structures' layout,
the entries' answers to calls without a handle, and the Python mirror's
parameter packing."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

from shared_amd import FilterParams, _capi, pack_filter_params

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_layout_matches_the_c_compiler(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("gcc is not installed")
    structs = {"sas_projection": _capi.SasProjection, "sas_filter_params": _capi.SasFilterParams,
               "sas_filter_rows": _capi.SasFilterRows}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "shared_amd_sampler.h"', "int main(void) {"]
    for cname, cls in structs.items():
        lines.append(f'  printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0; }"]) + "\n")
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(l.split() for l in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for cname, cls in structs.items():
        assert int(got[cname]) == ctypes.sizeof(cls), cname
        for f, _ in cls._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(cls, f).offset, (cname, f)


def test_calls_without_a_handle_are_refused():
    lib = _capi.load()
    assert lib.sas_project(None, None, None) == _capi.ERR_INVALID
    assert b"handle is NULL" in lib.sas_last_error(None)
    assert lib.sas_sample_filtered(None, None, None) == _capi.ERR_INVALID
    assert b"sas_sample_filtered: handle is NULL" in lib.sas_last_error(None)
    assert lib.sas_reserve_project(None, 1, 64, 8) == _capi.ERR_INVALID
    assert lib.sas_reserve_filtered(None, 1, 64) == _capi.ERR_INVALID


def test_parameters_pack_as_the_c_struct():
    p = FilterParams(temperature=0.7, top_p=0.9, min_p=0.05, repetition_penalty=1.1, presence_penalty=0.5,
                     frequency_penalty=0.2, softcap=30.0, top_k=40)
    a = pack_filter_params([FilterParams(), p])
    assert a.itemsize == ctypes.sizeof(_capi.SasFilterParams)
    assert a[1].tobytes() == bytes(p.to_c())
    assert a[0]["top_k"] == 0 and a[0]["top_p"] == 1.0 and a[0]["min_p"] == 0.0
    assert np.float32(a[1]["softcap"]) == np.float32(30.0)
