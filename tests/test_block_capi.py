"""The C ABI of the RMS norm, the gated linear layer and the AdamW step without a GPU: the headers declare what
the binding lists and the library exports, and are plain C."""
import ctypes as C
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADERS = ("rms_norm.h", "gated_linear.h", "adamw.h")


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
    assert sorted(capi.BLOCK_EXPORTS) == declared()
    out = subprocess.run(["nm", "-D", "--defined-only", capi.LIB_PATH], capture_output=True, text=True,
                         check=True).stdout
    exported = {line.split()[-1] for line in out.splitlines() if " T " in line}
    assert set(declared()) <= exported


def test_limits_and_layouts_agree(capi, tmp_path):
    """The binding's constants and structures are the headers', which compile as C99 by themselves."""
    structs = (("mft_rms_norm_desc", capi.RmsNormDesc), ("mft_gated_linear_desc", capi.GatedLinearDesc),
               ("mft_adamw_desc", capi.AdamWDesc), ("mft_adamw_tensor", capi.AdamWTensor))
    fields = [(s, f) for s, t in structs for f, _ in t._fields_]
    src = tmp_path / "t.c"
    src.write_text("".join(f'#include "mft/{h}"\n' for h in HEADERS) + "#include <stddef.h>\n#include <stdio.h>\n"
                   'int main(void) { printf("%d\\n", MFT_ADAMW_GROUP);\n' +
                   "".join(f'printf("%zu\\n", sizeof({s}));\n' for s, _ in structs) +
                   "".join(f'printf("%zu\\n", offsetof({s}, {f}));\n' for s, f in fields) + "return 0; }\n")
    exe = tmp_path / "t"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROOT, "include"),
                    "-I", "/opt/rocm/include", str(src), "-o", str(exe)], check=True, capture_output=True, text=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    of = dict(structs)
    assert got == ([capi.ADAMW_GROUP] + [C.sizeof(t) for _, t in structs] +
                   [getattr(of[s], f).offset for s, f in fields])
