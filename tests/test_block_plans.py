"""Every kernel that the gated linear layer's products and the RMS norm's rows can take, against the formulas in
64 bits: which one a size takes is asked of the planners themselves (native/block_plans.cpp), over a sweep of
sizes, and the sizes below have to reach each.  Bounds are those of test_gated_linear.py and test_rms_norm.py."""
import os
import subprocess

import pytest
import torch

import test_gated_linear as G
import test_rms_norm as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# N, in, ff, with either layout of the weights: dx joined along both weights and the forward on each tile, whole and
# cut along k; a training step's backward
BF16 = [(200, 4864, 768), (16384, 1408, 256), (1500, 4864, 896), (4096, 1152, 2048), (300, 6912, 6912), (300, 16384, 6912),
        (6000, 320, 6912), (2800, 11008, 768), (4096, 16384, 320), (2800, 16384, 1600), (4096, 1152, 6912)]
# fp32: 128 x 128 tiles of each product, whole and cut; dx as two products, the second added; odd sizes of both
F32 = [(2048, 4096, 64), (200, 64, 16384), (3, 11008, 320), (3, 6912, 320), (3, 1600, 5120), (300, 11008, 256),
       (300, 1153, 2001), (1001, 1153, 2050), (2048, 1152, 6912)]
E4M3 = [(64, 72, 64), (16384, 72, 256), (400, 1152, 16384)]
WIDTHS = [300, 301, 1000, 2304, 2561, 4096, 5120, 5121, 8192, 16384, 16392]


def ids(s):
    return "x".join(map(str, s))


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    """plans(of, sizes): the entries of each of the sizes."""
    lib = os.path.join(ROOT, "mobilefinetuner_amd", "lib")
    if not os.path.exists(os.path.join(lib, "libmft_attn.so")):
        pytest.skip("libmft_attn.so not built")

    def ask(of, sizes):
        exe = tmp_path_factory.mktemp(of) / "block_plans"
        # host code alone: the kernels' own code is not linked, and nothing is launched
        subprocess.run(["/opt/rocm/bin/hipcc", "-x", "hip", "--offload-arch=gfx950", "--cuda-host-only", "-O1", "-std=c++17",
                        f"-DOF_{of}", "-I", os.path.join(ROOT, "include"),
                        "-I", os.path.join(ROOT, "mobilefinetuner_amd", "csrc"),
                        os.path.join(ROOT, "tests", "native", "block_plans.cpp"), "-o", str(exe), "-L", lib, "-lmft_attn",
                        f"-Wl,-rpath,{lib}", "-Wl,--unresolved-symbols=ignore-all"],
                       check=True, capture_output=True, text=True)
        out = subprocess.run([str(exe)], input="\n".join(" ".join(map(str, s)) for s in sizes), capture_output=True, text=True,
                             check=True, env={**os.environ, "HIP_VISIBLE_DEVICES": ""}).stdout
        lines = [set(line.split()) for line in out.splitlines()]
        assert len(lines) == len(sizes)
        return lines

    return ask


NS = [3, 5, 9, 16, 17, 33, 64, 96, 128, 200, 256, 300, 400, 512, 700, 1000, 1024, 1500, 2000, 2048, 2800, 4096, 6000, 8192, 16384]
SIDES = [64, 72, 100, 128, 256, 320, 512, 640, 768, 896, 1024, 1152, 1408, 1600, 2048, 2304, 2560, 4096, 4864, 5120, 6912, 8192,
         11008, 16384]


@pytest.mark.parametrize("of,tested", [("GATED", G.SHAPES + BF16), ("F32", G.SHAPES + F32), ("E4M3", G.SHAPES + E4M3)])
def test_every_product_is_tested(plans, of, tested):
    if of != "F32":  # the large shapes of test_gated_linear.py
        more = {"GATED": G.test_large_products, "E4M3": G.test_eight_bits}[of]
        tested = tested + [s for m in more.pytestmark if m.args and m.args[0] == "shape" for s in m.args[1]]
    sweep = [(n, i, f) for n in NS for i in SIDES for f in SIDES if n * i * f <= 1 << 38]
    reached = set().union(*plans(of, sweep))
    assert len(reached) > 10
    missed = reached.difference(*plans(of, tested))
    assert not missed


def test_every_row_kernel_is_tested(plans):
    reached = set().union(*plans("RMS", [(d,) for d in range(1, 80000, 7)] + [(d,) for d in range(40, 80000, 40)]))
    assert len(reached) > 30
    missed = reached.difference(*plans("RMS", [(d,) for d in R.WIDTHS + WIDTHS]))
    assert not missed


@pytest.mark.gpu
@pytest.mark.parametrize("w_t", [False, True], ids=["in_ff", "ff_in"])
@pytest.mark.parametrize("dtype,shape", [("bf16", s) for s in BF16] + [("f32", s) for s in F32],
                         ids=lambda s: s if isinstance(s, str) else ids(s))
def test_gated_products(dev, dtype, shape, w_t):
    G.check(dev, *shape, dtype, "silu", w_t, 23)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", E4M3, ids=ids)
def test_eight_bits(dev, shape):
    G.check_e4m3(dev, *shape, "silu", 24)
    G.check_e4m3(dev, *shape, "silu", 24, near=True)


# operands off 16 bytes: the forward's tiles through registers, and dx by copies of both weights
@pytest.mark.gpu
@pytest.mark.parametrize("w_t", [False, True], ids=["in_ff", "ff_in"])
@pytest.mark.parametrize("shape", BF16[:8] + [(4100, 264, 2056), (4096, 1152, 6912)], ids=ids)
def test_gated_products_off_16_bytes(dev, shape, w_t):
    from mobilefinetuner_amd import gated_linear as L
    print(f"[case] {shape} {w_t}", flush=True)
    d = {}
    for k, v in G.make(*shape, "bf16", 25, w_t).items():
        flat = torch.empty(v.numel() + 1, dtype=v.dtype, device=dev)[1:]
        d[k] = flat.view(v.shape).copy_(v) if k in ("W_gate", "W_up") else v.to(dev)
    up = {k: v.double() for k, v in d.items()}
    Wg, Wu = (up[k].t() if w_t else up[k] for k in ("W_gate", "W_up"))
    got = L.gated_linear(d["x"], d["W_gate"], d["W_up"], "gelu_tanh", w_t, True)
    gate, tg, rise, tu, h, th = G.ref_forward(up["x"], Wg, Wu, "gelu_tanh", torch.bfloat16)
    for name, g, r, t in zip(("h", "gate", "up"), got, (h, gate, rise), (th, tg, tu)):
        G.within(g, r, t, name)
    del gate, tg, rise, tu, h, th, got
    dx, dWg, dWu = L.gated_linear_backward(d["x"], d["W_gate"], d["W_up"], d["gate"], d["up"], d["dh"], "gelu_tanh", w_t)
    ref = G.ref_backward(up["x"], Wg, Wu, up["gate"], up["up"], up["dh"], "gelu_tanh", torch.bfloat16)
    G.within(dx, ref[0], ref[1], "dx")
    for name, g, r, t in (("dW_gate", dWg, *ref[2:4]), ("dW_up", dWu, *ref[4:])):
        G.within(g, r.t() if w_t else r, t.t() if w_t else t, name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", WIDTHS)
def test_norms(dev, D, dtype):
    R.test_forward_and_backward(dev, D, dtype)
    R.test_eight_bits(dev, D, dtype)
