"""First calls made by several threads at once (ctypes releases the interpreter lock): what a call prepares once per device
is written by one thread, and ordered before every other's use."""
import glob
import os
import re
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "nvidia-x-gpu-mode-kernels_b200", "csrc")


def test_once_per_device_under_the_thread_sanitizer(tmp_path):
    exe = tmp_path / "once_client"
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=thread", "-pthread", "-I", CSRC,
                    os.path.join(ROOT, "tests", "c_client", "once_client.cpp"), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    if "unexpected memory mapping" in run.stderr:       # the sanitizer wants the addresses that it knows
        run = subprocess.run(["setarch", "-R", str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout == "wrong 0\n", run.stdout + run.stderr


def test_no_unordered_first_call_flags():
    for path in glob.glob(os.path.join(CSRC, "*.cu*")):
        assert not re.search(r"static\s+bool\s+\w+\s*\[", open(path).read()), path


THREADS = """
import sys, threading, torch
sys.path.insert(0, {root!r})
import __graft_entry__
pkg = __graft_entry__.load_package()
g = torch.Generator(device="cuda").manual_seed(1)
half = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.float16)
byte = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, device="cuda", dtype=torch.uint8)
def lora(T):
    a = (half(T, 64), half(T, 64), half(3, 16, 64), half(3, 64, 16), torch.arange(T, device="cuda", dtype=torch.int32) % 4)
    return lambda: pkg.lora_add(*a, out=torch.empty_like(a[0]))
def moe(T):
    a = (half(T, 128), torch.randint(0, 4, (T, 2), generator=g, device="cuda", dtype=torch.int32),
         torch.rand(T, 2, generator=g, device="cuda"), byte(0, 256, 4, 128, 64), byte(0, 256, 4, 128, 64), byte(0, 256, 4, 128, 64),
         byte(2, 11, 4, 1024), byte(2, 11, 4, 1024), byte(2, 11, 4, 1024))
    return lambda: pkg.moe_mlp(*a)
def skinny(T):
    a = (byte(0, 256, T, 64), byte(0, 256, 128, 64), byte(2, 11, 1024), byte(2, 11, 1024))
    return lambda: pkg.skinny_gemm(*a, torch.empty((T, 128), dtype=torch.float16, device="cuda"))
calls = [f(T) for f, T in ((lora, 5), (lora, 300), (moe, 5), (moe, 600), (skinny, 5), (skinny, 40)) for _ in range(2)]
torch.cuda.synchronize()
first, start, failed = [None] * len(calls), threading.Barrier(len(calls)), []
def run(i):
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            start.wait()
            first[i] = calls[i]()
            torch.cuda.current_stream().synchronize()
    except Exception as e:
        failed.append(e)
threads = [threading.Thread(target=run, args=(i,)) for i in range(len(calls))]
[t.start() for t in threads]
[t.join() for t in threads]
assert not failed, failed
for f, got in zip(calls, first):
    assert torch.equal(f(), got)
torch.cuda.synchronize()
assert pkg._lib.device_errors() == 0
print("same")
"""


@pytest.mark.gpu
def test_first_calls_of_twelve_threads(cuda):
    run = subprocess.run([sys.executable, "-c", THREADS.format(root=ROOT)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == "same", run.stdout + run.stderr
