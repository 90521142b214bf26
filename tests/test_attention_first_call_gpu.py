"""GPU tests of the process's first call, each in a process of its own: captured into a graph (the set-up
of the device runs inside the capture), or made by several threads at once."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]

SET_UP = """
import sys
import threading

import torch

sys.path.insert(0, "mini-flash-attention_b200")
import mini_flash_attention as mfa

g = torch.Generator(device="cuda").manual_seed(1)
new = lambda *shape: torch.randn(shape, device="cuda", generator=g).half()
whole = lambda *x: torch.tensor(x, device="cuda", dtype=torch.int32)
q, k, v, dout = new(1, 4, 300, 64), new(1, 2, 300, 64), new(1, 2, 300, 64), new(1, 4, 300, 64)
one, rows, k_cache, v_cache = new(2, 4, 64), new(4, 2, 64), new(40, 2, 16, 64), new(40, 2, 16, 64)
table = torch.arange(36, device="cuda", dtype=torch.int32).reshape(2, 18)
lse = torch.randn((1, 4, 300), device="cuda", generator=g)


def extend():
    mine = table.clone()
    return mine, *mfa.extend_block_tables(mine, whole_200, whole_30, table[0], 16, 60)


whole_200, whole_30, slots = whole(200, 100), whole(30, 20), whole(3, 9, -1, 77)


def append():
    mine = k_cache.clone(), v_cache.clone()
    mfa.append_kv(rows, rows, *mine, slots)
    return mine


calls = {
    "forward": lambda: (mfa.forward(q, q, q, True),),
    "backward": lambda: mfa.backward(q, q, q, q, lse, dout),
    "forward_window": lambda: (mfa.forward_window(q, k, v, 50, 2),),
    "backward_window": lambda: mfa.backward_window(q, k, v, q, lse, dout, 50, 2),
    "paged_attention": lambda: (mfa.paged_attention(one, k_cache, v_cache, table, whole_200),),
    "shared_prefix_attention": lambda: (mfa.shared_prefix_attention(
        one, k_cache, v_cache, table[0], 250, table, whole_200),),
    "extend_block_tables": extend,
    "append_kv": append,
}
call = calls[sys.argv[1]]
torch.cuda.synchronize()
"""

CAPTURED = SET_UP + """
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = call()
graph.replay()
want = call()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("same")
"""

THREADS = SET_UP + """
got, gate = [None] * 4, threading.Barrier(4)


def work(i):
    with torch.cuda.stream(torch.cuda.Stream()):
        gate.wait()
        got[i] = call()
        torch.cuda.current_stream().synchronize()


threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
for t in threads:
    t.start()
for t in threads:
    t.join()
want = call()
assert all(torch.equal(a, b) for x in got for a, b in zip(x, want))
print("same")
"""

NAMES = ["forward", "backward", "forward_window", "backward_window", "paged_attention",
         "shared_prefix_attention", "extend_block_tables", "append_kv"]


def child(code, name):
    r = subprocess.run([sys.executable, "-c", code, name], cwd=ROOT, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stderr[-2000:]


@pytest.mark.parametrize("name", NAMES)
def test_captured(name):
    child(CAPTURED, name)


@pytest.mark.parametrize("name", ["backward_window", "paged_attention", "append_kv"])
def test_threads(name):
    child(THREADS, name)
