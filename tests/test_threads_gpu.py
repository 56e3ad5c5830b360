"""First calls of a process from several threads at once, each on a stream of its own: the entry points run without the interpreter lock."""

import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent

PROGRAM = """
import threading
import torch
from tensorfold_b200 import lane_evict, lane_window, speculative

BF = torch.bfloat16
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")

def inputs(seed, d):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=gen).cuda()
    used = 20
    return dict(k=rand(1, 2 * used, 2, 16, d).to(BF), v=rand(1, 2 * used, 2, 16, d).to(BF), mass=rand(1, 2 * used, 2, 16).abs(), pos=i32([0] * (64 * used)).reshape(1, 2 * used, 2, 16),
                q=rand(6, 8, d).to(BF), kn=rand(6, 2, d).to(BF), vn=rand(6, 2, d).to(BF), logits=rand(6, 3000).to(BF), near=rand(6, 3000).to(BF),
                tokens=torch.randint(0, 3000, (6,), generator=gen).to(torch.int32).cuda(), u=torch.rand((6, 2), generator=gen, dtype=torch.float64).cuda(),
                table=torch.arange(2 * used, dtype=torch.int32).reshape(2, used).cuda(), lens=i32([300, 77]), start=i32([0, 4, 6]), row_pos=i32([1] * 6))

def calls(c):
    lse = torch.empty((1, 6, 8), device="cuda")
    out = lane_window.window_attention(c["q"], c["kn"], c["vn"], c["k"][0], c["v"][0], c["table"], c["lens"], c["start"], scale=0.1, max_window=4, max_context=310, lse=lse[0])
    keep, token = speculative.verify_drafts(c["logits"], c["tokens"], c["start"], c["u"], draft_logits=c["near"])
    lane_evict.attention_mass(c["q"][None], lse, c["k"], c["table"], c["lens"], c["start"], keep, c["row_pos"], c["mass"], c["pos"], scale=0.1, max_window=4, max_context=310)
    moved = lane_evict.evict(c["k"], c["v"], c["table"], c["lens"], c["lens"], c["mass"], c["pos"], 100, recent=5, sinks=2, max_context=310)
    return [out, lse, keep, token, moved, *(c[n] for n in ("mass", "pos", "k", "v"))]

sets = [(seed, 128 if seed % 2 else 256) for seed in range(6)]
held = [inputs(*x) for x in sets]
torch.cuda.synchronize()
results, begin = [None] * len(sets), threading.Barrier(len(sets))

def work(i):
    with torch.cuda.stream(torch.cuda.Stream()):
        begin.wait()
        results[i] = calls(held[i])
        torch.cuda.current_stream().synchronize()

threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sets))]
for t in threads: t.start()
for t in threads: t.join()
for x, got in zip(sets, results):
    want = calls(inputs(*x))
    assert all(torch.equal(a, b) for a, b in zip(got, want)), x
print("same")
"""


def test_first_calls_from_several_threads(lib):
    done = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip().endswith("same"), done.stdout + done.stderr
