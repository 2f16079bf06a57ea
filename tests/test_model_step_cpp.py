"""The model-step operators' C and C++ headers, and the example that runs them together."""
from __future__ import annotations

import runpy
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
SRC = ROOT / "tests" / "cpp" / "model_api_test.cpp"
CUDA = Path("/usr/local/cuda")
LIBDIR = ROOT / "luisacompute-parallelprimitive_b200" / "lcpp_b200"


def _gxx():
    gxx = shutil.which("g++")
    if gxx is None or not (CUDA / "include" / "cuda_runtime.h").exists():
        pytest.skip("g++ or the CUDA headers are missing")
    return gxx


def test_headers_compile(tmp_path):
    r = subprocess.run([_gxx(), "-std=c++17", "-fsyntax-only", "-Wall", "-Wextra", "-Werror",
                        f"-I{ROOT / 'include'}", f"-I{CUDA / 'include'}", str(SRC)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    c = tmp_path / "t.c"
    c.write_text('#include "lcpp_b200_model.h"\nint main(void){return 0;}\n')
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", str(ROOT / "include"), "-c", str(c), "-o",
                    str(tmp_path / "t.o")], check=True)


@pytest.mark.gpu
def test_cpp_program_runs(tmp_path):
    exe = tmp_path / "model_api_test"
    r = subprocess.run([_gxx(), "-std=c++17", "-O2", f"-I{ROOT / 'include'}", f"-I{CUDA / 'include'}", str(SRC), "-o",
                        str(exe), f"-L{LIBDIR}", "-llcpp_b200", f"-L{CUDA / 'lib64'}", "-lcudart",
                        f"-Wl,-rpath,{LIBDIR}", f"-Wl,-rpath,{CUDA / 'lib64'}"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr
    assert run.stdout.startswith("OK "), run.stdout


@pytest.mark.gpu
def test_example_runs():
    """The example's layer fits its target, and the balance loss does not rise above an even batch's by much more
    than at the start (it is 1 for even counts and shares)."""
    first, last = runpy.run_path(str(ROOT / "examples" / "paged_moe_step.py"))["main"]()
    assert last[0] < 0.8 * first[0]
    assert last[1] < first[1] + 0.05


@pytest.mark.gpu
def test_example_gradient():
    """The layer's gradient of its input against differences of the 64-bit forward pass through the same choice:
    rows and logits are rounded to 16 bits on the way (2^-9 each), so a few 1e-2 of the largest entry."""
    torch = pytest.importorskip("torch")
    module = runpy.run_path(str(ROOT / "examples" / "paged_moe_step.py"))
    torch.manual_seed(3)
    t, h, e, k = 24, 32, 4, 2
    layer = module["Layer"](t, h, e, k, align=8)
    x = torch.randn(t, h, device="cuda").to(torch.bfloat16)
    requests = torch.where(torch.arange(t, device="cuda") < 20, 0, -1).to(torch.int32)
    layer.forward(x, requests)
    g = torch.randn(t, h, device="cuda").to(torch.bfloat16)
    grad = layer.backward(g, balance=0.5)[2].double()

    x64 = x.double().requires_grad_(True)
    chosen = layer.chosen.clamp(min=0).long()
    live = (requests >= 0).double()
    logits = x64 @ layer.router.double()
    share = torch.softmax(logits, 1)
    weights = torch.softmax(torch.gather(logits, 1, chosen), 1) * live[:, None]
    products = torch.einsum("th,ehg->teg", x64, layer.experts.double())
    out = (weights[:, :, None] * torch.gather(products, 1, chosen[:, :, None].expand(-1, -1, h))).sum(1)
    n = live.sum()
    loss = e * ((share * live[:, None]).sum(0) / n * layer.counts.double() / (k * n)).sum()
    want = torch.autograd.grad((out * g.double()).sum() + 0.5 * loss, x64)[0]
    assert (grad - want).abs().max() <= 0.03 * want.abs().max()
    assert not grad[20:].any()
