"""Scratch on hipStreamPerThread, a handle that is another stream in each thread: the pool's rule on the CPU
(tests/scratch_thread_model.cpp), and the norm's gradients and paged attention called so from several threads."""
import ctypes as C
import shutil
import subprocess
import threading
from pathlib import Path

import pytest
import torch

from torchvulkan_amd import _abi

ROOT = Path(__file__).resolve().parent.parent
PER_THREAD = 2   # hipStreamPerThread


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_scratch_thread_model(tmp_path):
    exe = tmp_path / "scratch_thread_model"
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-pthread", f"-I{ROOT / 'torchvulkan_amd' / 'csrc'}",
                    str(ROOT / "tests" / "scratch_thread_model.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stderr
    assert out.stdout.strip() == "ok"


def in_threads(work, count=4):
    """work(i) in `count` threads; the first exception of any."""
    failed = []

    def run(i):
        try:
            work(i)
        except BaseException as e:   # noqa: BLE001  (raised again below)
            failed.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(count)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if failed:
        raise failed[0]


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [1024, 20000])
def test_norm_gradients_from_threads(gpu, cols):
    rows, lib = 3000 if cols == 1024 else 300, _abi.load()
    calls = []
    for i in range(4):
        g = torch.Generator(device="cuda").manual_seed(i)
        dy, h = (torch.randn((rows, cols), generator=g, device="cuda").to(torch.float16) for _ in range(2))
        w = torch.randn(cols, generator=g, device="cuda")
        dx, dw = torch.empty_like(h), torch.empty_like(w)
        want = _abi.rms_norm_bwd(dy, h, w)
        calls.append((_abi.make_rms_norm_bwd_desc(dy, h, w, dx, dw, stream=PER_THREAD), dx, dw, want, (dy, h, w)))
    torch.cuda.synchronize()

    def work(i):
        d, dx, dw, want, _ = calls[i]
        for _ in range(20):
            _abi.check(lib.tvk_rms_norm_bwd(C.byref(d)))
        torch.cuda.synchronize()
        assert torch.equal(dx, want[0]) and torch.equal(dw, want[1])

    in_threads(work)


@pytest.mark.gpu
def test_paged_attention_from_threads(gpu):
    # long sequences are cut there as on any stream (joined by a second launch, with the same bits)
    lens, page, hkv, dim, lib = [20000, 700], 16, 2, 128, _abi.load()
    table = torch.arange(2 * 1250, dtype=torch.int32).view(2, 1250).cuda()
    seq = torch.tensor(lens, dtype=torch.int32).cuda()
    calls = []
    for i in range(4):
        g = torch.Generator(device="cuda").manual_seed(i)
        k, v = (torch.randn((2500, page, hkv, dim), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
        q = torch.randn((2, 1, 8, dim), generator=g, device="cuda").to(torch.bfloat16)
        want, _ = _abi.paged_attention(q, k, v, seq, table)
        out = torch.empty_like(q)
        calls.append((_abi.make_paged_attention_desc(q, k, v, out, seq, table, stream=PER_THREAD), out, want, (q, k, v)))
    torch.cuda.synchronize()

    def work(i):
        d, out, want, _ = calls[i]
        for _ in range(20):
            out.fill_(float("nan"))
            torch.cuda.synchronize()
            _abi.check(lib.tvk_paged_attention(C.byref(d)))
            torch.cuda.synchronize()
            assert torch.equal(out, want)

    in_threads(work)
