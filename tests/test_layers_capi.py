"""The C ABI of the layers around attention without a GPU: the headers declare
what the binding lists and the library exports, and are plain C."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADERS = ("layer_norm.h", "linear.h", "logprobs.h")


@pytest.fixture(scope="module")
def capi():
    from mobilefinetuner_amd import capi as M
    M.lib()
    return M


def declared():
    text = "".join(open(os.path.join(ROOT, "include", "mft", h)).read() for h in HEADERS)
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(mft_[a-z0-9_]+)\s*\(", text)))


def test_headers_binding_and_library_agree(capi):
    assert sorted(capi.LAYER_EXPORTS) == declared()
    out = subprocess.run(["nm", "-D", "--defined-only", capi.LIB_PATH], capture_output=True, text=True,
                         check=True).stdout
    exported = {line.split()[-1] for line in out.splitlines() if " T " in line}
    assert set(declared()) <= exported


def test_limits_and_enumerators_agree(capi, tmp_path):
    """The binding's constants are the headers', which compile as C99 by themselves."""
    src = tmp_path / "t.c"
    src.write_text("".join(f'#include "mft/{h}"\n' for h in HEADERS) + "#include <stdio.h>\n"
                   'int main(void) { printf("%d %d %d %d %d %zu %zu %zu\\n", MFT_LOGPROBS_MAX_TOP, MFT_ACT_NONE, '
                   "MFT_ACT_RELU, MFT_ACT_GELU_TANH, MFT_ACT_SILU, sizeof(mft_layer_norm_desc), "
                   "sizeof(mft_linear_desc), sizeof(mft_logprobs_desc)); return 0; }\n")
    exe = tmp_path / "t"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROOT, "include"),
                    "-I", "/opt/rocm/include", str(src), "-o", str(exe)], check=True, capture_output=True, text=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    import ctypes as C
    assert got == [capi.LOGPROBS_MAX_TOP, capi.MFT_ACT_NONE, capi.MFT_ACT_RELU, capi.MFT_ACT_GELU_TANH,
                   capi.MFT_ACT_SILU, C.sizeof(capi.LayerNormDesc), C.sizeof(capi.LinearDesc),
                   C.sizeof(capi.LogprobsDesc)]
