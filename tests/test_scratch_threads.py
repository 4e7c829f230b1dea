"""Host threads that call operators on one stream share the stream's scratch memory: a call keeps it until its last launch
is queued.  scratch_threads.cc checks that on the host, with stand-ins for the CUDA runtime's calls; the GPU test runs the
mixture-of-experts operators, whose launches hand data to each other through it, from several threads at once."""
import os
import shutil
import subprocess
import threading

import pytest
import torch

from sparsetir_b200 import ops
from sparsetir_b200 import build as B

HERE = os.path.dirname(os.path.abspath(__file__))


def test_scratch_is_held_until_the_call_is_queued(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    include = os.path.join(os.path.dirname(os.path.dirname(nvcc)), "include")
    if not os.path.exists(os.path.join(include, "cuda_runtime.h")):
        pytest.skip("no CUDA headers")
    exe = str(tmp_path / "scratch_threads")
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", B.INCLUDE, "-I", B.CSRC, "-isystem", include,
                    os.path.join(HERE, "scratch_threads.cc"), os.path.join(B.CSRC, "runtime.cc"), "-o", exe],
                   check=True, capture_output=True, text=True)
    res = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0 and res.stdout == "ok\n", res.stdout


def _job(seed, tokens, experts, top_k, rows, groups, fi, fo, device):
    """Inputs of one thread, and its calls with their results: a router of two launches, products whose operands are copied to
    aligned rows, and a gradient whose depth several units share."""
    g = torch.Generator(device=device).manual_seed(seed)
    z = torch.randn(tokens, experts, device=device, generator=g)
    x, w = (torch.randn(n, device=device, generator=g).half() for n in (rows * fi, groups * fi * fo))
    ptr = (torch.arange(groups + 1, device=device) * rows // groups).int()

    def calls():
        i32 = dict(dtype=torch.int32, device=device)
        gates = torch.zeros(tokens * top_k, device=device)
        chosen, slots, indptr = torch.zeros(tokens * top_k, **i32), torch.zeros(tokens * top_k, **i32), torch.zeros(experts + 1, **i32)
        y, dw = torch.zeros(rows * fo, device=device), torch.zeros(fi * fo, device=device)
        ops.moe_route(z.view(-1), gates, chosen, slots, indptr, experts, top_k)
        ops.grouped_mm(x, w, y, ptr, groups, fi, fo)
        ops.grouped_mm_grad_w(x, y.half(), dw, None, 1, fi, fo)
        return gates, chosen, slots, indptr, y, dw

    return calls


@pytest.mark.gpu
def test_threads_on_one_stream(cuda_device):
    stream = torch.cuda.Stream(priority=-1)
    jobs = [_job(1, 5000, 64, 6, 700, 3, 203, 131, cuda_device), _job(2, 300, 17, 2, 5000, 2, 35, 67, cuda_device),
            _job(3, 20000, 200, 8, 90, 1, 1001, 999, cuda_device)]
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    errors, gate = [], threading.Barrier(len(jobs))

    def work(job, want):
        try:
            torch.cuda.set_device(cuda_device)
            with torch.cuda.stream(stream):
                gate.wait()
                for _ in range(40):
                    got = job()
                    stream.synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(got, want))
        except Exception as e:  # surfaced by the main thread
            errors.append(repr(e))
            gate.abort()

    threads = [threading.Thread(target=work, args=pair) for pair in zip(jobs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
