"""MXFP4 without a GPU: the structures' layout, the entries' answers to calls
without a handle, and the tests' own reference."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

import mx4_reference as R
from shared_amd import HEAD_MX4, Mx4, _capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_layout_matches_the_c_compiler(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("gcc is not installed")
    structs = {"sas_mx4": _capi.SasMx4, "sas_mx4_quantization": _capi.SasMx4Quantization, "sas_mx4_lookup": _capi.SasMx4Lookup,
               "sas_mx4_projection": _capi.SasMx4Projection, "sas_lm_head": _capi.SasLmHead}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "shared_amd_sampler.h"', "int main(void) {",
             '  printf("consts %d %d %d\\n", SAS_HEAD_MX4, SAS_TYPE_MX4, SAS_MX4_BLOCK);']
    for cname, cls in structs.items():
        lines.append(f'  printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0; }"]) + "\n")
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(l.split(" ", 1) for l in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    assert got["consts"] == f"{HEAD_MX4} {_capi.TYPE_MX4} 32"
    for cname, cls in structs.items():
        assert int(got[cname]) == ctypes.sizeof(cls), cname
        for f, _ in cls._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(cls, f).offset, (cname, f)


def test_calls_without_a_handle_are_refused():
    lib = _capi.load()
    for name in ("sas_quantize_mx4", "sas_lookup_mx4", "sas_project_mx4"):
        assert getattr(lib, name)(None, None, None) == _capi.ERR_INVALID
        assert name.encode() + b": handle is NULL" in lib.sas_last_error(None)


def test_mx4_refuses_host_tensors():
    import torch
    with pytest.raises(ValueError, match="device tensor"):
        Mx4(torch.zeros((2, 16), dtype=torch.uint8), torch.zeros((2, 4), dtype=torch.uint8), 32)


def test_reference_of_the_format():
    # 7 lies past the last border: the scale is 1, and 7 stays at 6
    codes, scales = R.quantize([[0.25, 0.75, -1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 0.0, -0.3]])
    assert scales.tolist() == [[127]]
    assert codes[0, :5].tolist() == [0x20, 0x4A, 0x64, 0x76, 0x90] and not codes[0, 5:].any()
    assert R.values(codes, scales, 10).tolist() == [[0.0, 1.0, -1.0, 2.0, 2.0, 4.0, 4.0, 6.0, 0.0, -0.5]]
    codes, scales = R.quantize([[0.0] * 32 + [np.inf] + [2.0 ** -140] * 32])
    assert scales.tolist() == [[0, 255, 0]] and not codes.any()
    every = np.arange(16, dtype=np.uint8)
    v = R.values((every | every << 4)[None], np.array([[128]]), 32)
    assert v[0, ::2].tolist() == [0, 1, 2, 3, 4, 6, 8, 12, 0, -1, -2, -3, -4, -6, -8, -12]


def test_quantisation_refuses_scales_without_their_padding():
    """A row's scale bytes are written up to a multiple of four: a view that holds
    fewer would have what lies beside it overwritten."""
    import torch
    from shared_amd import Sampler

    class Device(torch.Tensor):
        is_cuda = property(lambda self: True)

    def dev(*shape, dtype=torch.uint8):
        return torch.zeros(shape, dtype=dtype).as_subclass(Device)
    s = Sampler.__new__(Sampler)
    s._lib, s._h = _capi.load(), None
    table = dev(10, 5)         # rows of 5 blocks, one behind another
    for rows, scales in ((1, table[4:5]), (1, dev(1, 7)[:, :5]), (3, dev(3, 12)[:, :5])):
        out = Mx4(dev(rows, 80), scales, 160)
        with pytest.raises(ValueError, match="8 bytes a row"):
            s.quantize_mx4_into(dev(rows, 160, dtype=torch.float32), out, stream=0)
    # with the padding the call goes on to the library, which has no handle here
    with pytest.raises(_capi.SasError, match="handle"):
        s.quantize_mx4_into(dev(3, 160, dtype=torch.float32), Mx4(dev(3, 80), dev(3, 12)[:, :8], 160), stream=0)


def test_quantisation_of_no_rows_needs_no_padding():
    import torch
    from shared_amd import Sampler

    class Device(torch.Tensor):
        is_cuda = property(lambda self: True)
    s = Sampler.__new__(Sampler)
    s._lib, s._h = _capi.load(), None
    u8 = lambda *shape: torch.zeros(shape, dtype=torch.uint8).as_subclass(Device)  # noqa: E731
    # (it reaches the library, which has no handle here)
    with pytest.raises(_capi.SasError, match="handle"):
        s.quantize_mx4_into(torch.zeros((0, 160)).as_subclass(Device), Mx4(u8(2, 80), u8(2, 5), 160), stream=0)
