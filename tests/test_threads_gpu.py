"""The training operators on threads that have made no CUDA call of their own: another host thread, autograd's first call."""
import pathlib
import subprocess
import sys
import threading

import pytest
import torch

from atomic_gdn2 import gated_scan, last_status, linear

pytestmark = pytest.mark.gpu
ROOT = pathlib.Path(__file__).resolve().parents[1]


def _in_a_thread(f):
    got = []

    def run():
        try:
            got.append(f())
        except Exception as e:                            # told where the test can see it
            got.append(e)

    t = threading.Thread(target=run)
    t.start()
    t.join()
    if isinstance(got[0], Exception):
        raise got[0]
    return got[0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_new_host_thread(dtype):
    """The same bits as from the thread that the tensors' memory came from; the outputs' is in the allocator's cache."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    make = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dtype)
    x, w, a, g = make(1024, 512), make(512, 768), make(2, 500, 64), -make(2, 500, 64).abs()
    for f in (lambda: linear(x, w), lambda: gated_scan(a, g)[0]):
        want = f().clone()
        f()
        torch.cuda.synchronize()
        for _ in range(2):
            assert torch.equal(_in_a_thread(f), want)
    assert last_status() == 0


SCRIPT = """
import torch
from atomic_gdn2 import linear, last_status
w = torch.zeros(2048, 2048, dtype=torch.bfloat16, device="cuda", requires_grad=True)
x = torch.ones(4096, 2048, dtype=torch.bfloat16, device="cuda")
dy = torch.ones(4096, 2048, dtype=torch.bfloat16, device="cuda")
(dw,) = torch.autograd.grad(linear(x, w), w, dy)
assert bool((dw == 4096.0).all()) and last_status() == 0
print("fine")
"""


def test_autograds_thread_begins_with_a_product():
    """A backward of one bf16 product is the first that autograd's thread of a new process does on the GPU."""
    r = subprocess.run([sys.executable, "-c", SCRIPT], cwd=ROOT / "atomic-ops_b200", capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("fine"), r.stderr[-2000:]


def _steps(seed):
    """Some calls of each operator, both ways, on a stream of the caller's own."""
    from atomic_gdn2.training import AdamW
    stream, got = torch.cuda.Stream(), []
    with torch.cuda.stream(stream):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        make = lambda *s: torch.randn(*s, generator=gen, device="cuda")
        for i, (M, K, N) in enumerate([(200, 300, 400), (64, 2000, 64), (700, 1500, 900), (5, 700, 900)]):
            dtype = torch.bfloat16 if (i + seed) % 2 else torch.float32
            leaves = [make(*s).to(dtype).requires_grad_(True) for s in ((M, K), (K, N), (N,))]
            y = linear(*leaves, act="gelu")
            got += [y.detach(), *torch.autograd.grad(y.float().square().sum(), leaves)]
            x, g = make(3, 400 + i, 65).to(dtype).requires_grad_(True), (-make(3, 400 + i, 65).abs()).to(dtype).requires_grad_(True)
            h, last = gated_scan(x, g)
            got += [h.detach(), last.detach(), *torch.autograd.grad(h.float().square().sum() + last.sum(), (x, g))]
            weights = [torch.nn.Parameter(make(300 + i, 77)) for _ in range(5)]
            for p in weights:
                p.grad = make(300 + i, 77)
            AdamW(weights, lr=1e-2, clip=1.0, state_bits=8 if i % 2 else 32).step()
            got += [p.detach() for p in weights]
        stream.synchronize()
    return got


def test_threads_at_once():
    """Four threads, each on a stream of its own, get the bits that each gets by itself."""
    alone = [_steps(s) for s in range(4)]
    for _ in range(2):
        got = {}
        threads = [threading.Thread(target=lambda s=s: got.update({s: _steps(s)})) for s in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        for s in range(4):
            assert s in got and all(torch.equal(a, b) for a, b in zip(alone[s], got[s])), s
    assert last_status() == 0
