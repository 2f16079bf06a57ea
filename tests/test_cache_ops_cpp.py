"""The paged cache's C++ classes, and the example that runs the operators together."""
from __future__ import annotations

import runpy
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
SRC = ROOT / "tests" / "cpp" / "cache_api_test.cpp"
CUDA = Path("/usr/local/cuda")
LIBDIR = ROOT / "luisacompute-parallelprimitive_b200" / "lcpp_b200"
EXAMPLE = str(ROOT / "examples" / "paged_cache_decode.py")


def _gxx():
    gxx = shutil.which("g++")
    if gxx is None or not (CUDA / "include" / "cuda_runtime.h").exists():
        pytest.skip("g++ or the CUDA headers are missing")
    return gxx


def test_program_compiles():
    r = subprocess.run([_gxx(), "-std=c++17", "-fsyntax-only", "-Wall", "-Wextra", "-Werror",
                        f"-I{ROOT / 'include'}", f"-I{CUDA / 'include'}", str(SRC)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


@pytest.mark.gpu
def test_program_runs(tmp_path):
    exe = tmp_path / "cache_api_test"
    r = subprocess.run([_gxx(), "-std=c++17", "-O2", f"-I{ROOT / 'include'}", f"-I{CUDA / 'include'}", str(SRC), "-o",
                        str(exe), f"-L{LIBDIR}", "-llcpp_b200", f"-L{CUDA / 'lib64'}", "-lcudart",
                        f"-Wl,-rpath,{LIBDIR}", f"-Wl,-rpath,{CUDA / 'lib64'}"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr
    assert run.stdout.startswith("OK "), run.stdout


@pytest.mark.gpu
def test_example_runs():
    runpy.run_path(EXAMPLE)["main"](steps=70)


@pytest.mark.gpu
def test_example_decode_agrees_with_training():
    """Before anything is evicted, a request's answer from the cache is the training pass's last row: both in 32 bits,
    sums of a few hundred terms, so 1e-4 of the largest entry."""
    torch = pytest.importorskip("torch")
    module = runpy.run_path(EXAMPLE)
    torch.manual_seed(1)
    layer = module["Layer"](dtype=torch.float32)
    cache = module["Cache"](layer, 3, pages=30)
    lengths = [31, 70, 2]
    x = torch.randn(sum(lengths), layer.qkv.shape[0], device="cuda")
    ends = torch.tensor(lengths).cumsum(0) - 1
    was = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        want = layer.train_forward(x, lengths)[ends]
        got = cache.step(x, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    finally:
        torch.backends.cuda.matmul.allow_tf32 = was
    assert (got - want).abs().max() <= 1e-4 * want.abs().max()


@pytest.mark.gpu
def test_example_gradient():
    """The layer's gradient of its input against that of the same layer in 64 bits, by torch's own operations: all in
    32 bits, so 1e-4 of the largest entry."""
    torch = pytest.importorskip("torch")
    module = runpy.run_path(EXAMPLE)
    torch.manual_seed(2)
    layer = module["Layer"](hidden=32, heads=4, kv_heads=2, dim=16, dtype=torch.float32)
    lengths = [13, 1, 20]
    x = torch.randn(sum(lengths), 32, device="cuda")
    g = torch.randn_like(x)
    leaf = x.clone().requires_grad_(True)
    layer.train_forward(leaf, lengths).backward(g)

    y = x.double().requires_grad_(True)
    q, k, v = (y @ layer.qkv.double()).split((64, 32, 32), 1)
    angle = torch.cat([torch.arange(n, device="cuda") for n in lengths]).double()[:, None] * layer.frequencies
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]

    def turn(t):
        a, b = t.unflatten(1, (-1, 16)).chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    q, k, v = turn(q), turn(k), v.unflatten(1, (-1, 16))
    rows, at = [], 0
    for n in lengths:
        for t in range(n):
            head = []
            for h in range(4):
                x_t = k[at:at + t + 1, h // 2] @ q[at + t, h] / 4
                head.append(torch.softmax(x_t, 0) @ v[at:at + t + 1, h // 2])
            rows.append(torch.cat(head))
        at += n
    want = torch.autograd.grad((torch.stack(rows) @ layer.out.double() * g.double()).sum(), y)[0]
    assert (leaf.grad.double() - want).abs().max() <= 1e-4 * want.abs().max()
