"""What a paged cache and sampling refuse before anything reaches a GPU, their C structs, and the table of angles."""
import ctypes
import math
import os
import re
import subprocess

import pytest
import torch

import pimaicompiler_amd as P
from pimaicompiler_amd import _lib as L
from pimaicompiler_amd.paged import _overlaps

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_tensors_off_the_gpu_are_refused():
    pages, x = torch.zeros(2, 1, 16, 64, dtype=torch.float16), torch.zeros(2, 64)
    for call in (lambda: P.PagedCache(pages, pages), lambda: P.PagedCache(None, None), lambda: P.sample_tokens(x, torch.zeros(2)), lambda: P.sample_tokens(None, None)):
        with pytest.raises(P.NNRuntimeException, match="GPU"):
            call()


def test_the_structs_of_the_binding_are_the_header_s(tmp_path):
    """Sizes and offsets as a C compiler lays them out."""
    fields = {"PimHipPagedCache": L.PagedCache, "PimHipPagedBatch": L.PagedBatch, "PimHipPagedRows": L.PagedRows, "PimHipSampleSettings": L.SampleSettings}
    lines = []
    for name, struct in fields.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f}));' for f, _ in struct._fields_]
    src = tmp_path / "offsets.c"
    src.write_text('#include "pimhip.h"\n#include <stddef.h>\n#include <stdio.h>\nint main(void)\n{\n' + "\n".join(lines) + "\nreturn 0;\n}\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "offsets")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "offsets")], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for struct in fields.values():
        want.append(ctypes.sizeof(struct))
        want += [getattr(struct, f).offset for f, _ in struct._fields_]
    assert got == want


def test_limits_in_python_and_c_agree():
    from pimaicompiler_amd import paged, sampling
    csrc = os.path.join(ROOT, "pimaicompiler_amd", "csrc")
    assert int(re.search(r"kDimMost = (\d+)", open(os.path.join(csrc, "api_paged.hip")).read()).group(1)) == paged.HEAD_DIM_MOST
    assert eval(re.search(r"kSampleMost = ([\d <]+);", open(os.path.join(csrc, "sample_kernels.h")).read()).group(1)) == sampling.VOCAB_MOST


@pytest.mark.parametrize("base,scale", [(10000.0, 1.0), (500000.0, 1.0), (10000.0, 4.0)])
def test_the_table_of_angles(base, scale):
    t = P.rotary_table(1000, 96, base, scale)
    assert t.shape == (1000, 96) and t.dtype == torch.float32
    for p, i in ((0, 0), (1, 0), (999, 0), (999, 47), (500, 13)):
        angle = p / scale * base ** (-2 * i / 96)
        # cos and sin of an angle of up to 1000 that is off by two roundings of 2^-53, then a rounding to fp32
        for got, want in ((t[p, i], math.cos(angle)), (t[p, 48 + i], math.sin(angle))):
            assert abs(float(got) - want) <= abs(want) * 2.0**-24 + 1000 * 2.0**-51
    for wrong in (lambda: P.rotary_table(0, 64), lambda: P.rotary_table(10, 63), lambda: P.rotary_table(10, 0), lambda: P.rotary_table(10, 64, base=0.0),
                  lambda: P.rotary_table(10, 64, scale=-1.0)):
        with pytest.raises(P.NNRuntimeException):
            wrong()


def test_overlapping_elements_are_found():
    x = torch.zeros(4, 3, 16, 64)
    assert not _overlaps(x) and not _overlaps(x.transpose(1, 2)) and not _overlaps(x[::2, :, :, :8]) and not _overlaps(x[:1].expand(1, 3, 16, 64))
    assert _overlaps(x[:1].expand(4, 3, 16, 64)) and _overlaps(x.as_strided((4, 3, 16, 64), (x.stride(0) - 64, 1024, 64, 1)))
