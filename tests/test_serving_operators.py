"""What the expert layer and the log probabilities refuse before anything reaches a GPU, and their C structs."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

import pimaicompiler_amd as P
from pimaicompiler_amd import _lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_tensors_off_the_gpu_are_refused():
    x = torch.zeros(2, 64, dtype=torch.float16)
    for call in (lambda: P.token_log_probs(x, torch.zeros(2, dtype=torch.int64)), lambda: P.token_log_probs(None),
                 lambda: P.MoeLayerPlan((x, None), x.view(2, 1, 64), x.view(2, 64, 1))):
        with pytest.raises(P.NNRuntimeException):
            call()


def test_the_c_interface_checks_its_arguments():
    lib = L.load()
    n = ctypes.c_uint64()
    assert lib.pimhip_moe_layer_workspace_bytes(None, 1, ctypes.byref(n)) == L.PIMHIP_ERR_INVALID_ARGUMENT
    assert lib.pimhip_moe_layer_plan_destroy(None) == L.PIMHIP_OK
    handle = ctypes.c_void_p(8)
    assert lib.pimhip_moe_layer_plan_destroy(handle) == L.PIMHIP_ERR_INVALID_ARGUMENT


def test_the_structs_of_the_binding_are_the_header_s(tmp_path):
    """Sizes and offsets as a C compiler lays them out."""
    fields = {"PimHipMx4Matrix": L.Mx4Matrix, "PimHipMoeLayerDesc": L.MoeLayerDesc}
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
    from pimaicompiler_amd import log_probs, moe_layer
    src = "".join(open(os.path.join(ROOT, "pimaicompiler_amd", "csrc", f)).read() for f in ("logprob_kernels.h", "moe_layer_kernels.h"))
    assert int(re.search(r"kTopMost = (\d+)", src).group(1)) == log_probs.TOP_MOST
    assert int(re.search(r"kMoeLayerTokens = (\d+)", src).group(1)) == moe_layer.TOKENS_MOST


def test_a_plan_that_is_none_is_refused():
    n = ctypes.c_uint64()
    assert L.load().pimhip_moe_layer_workspace_bytes(ctypes.c_void_p(64), 1, ctypes.byref(n)) == L.PIMHIP_ERR_INVALID_ARGUMENT
