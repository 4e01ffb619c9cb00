"""First calls of a process from several threads at once: the native call path lets go of the interpreter's lock, so what the
library finds out once per device (cluster counts, function attributes, the SiLU table) is found out side by side."""
import pathlib
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

THREADS = """
import threading
import torch
from kb_nano_b200 import moe, ops
d = torch.device("cuda")
torch.manual_seed(0)
k, n = 512, 4096
xs = [torch.randn(m, k, device=d).to(torch.bfloat16) for m in (2, 64, 1300)]
long = torch.randn(40, 14336, device=d).to(torch.bfloat16)
w = torch.randint(0, 256, (n, k // 2), device=d, dtype=torch.uint8)
wl = torch.randint(0, 256, (64, 14336 // 2), device=d, dtype=torch.uint8)
sf = {id(q): torch.full((ops.packed_mxfp4_bytes(q.shape[0], 2 * q.shape[1]),), 120, dtype=torch.uint8, device=d) for q in (w, wl)}
gate = torch.randn(3, 2 * k, device=d).to(torch.bfloat16)
gate[0, :4] = -70.0
lg = torch.randn(2, 4, device=d)
e13, e2 = torch.randint(0, 256, (4, 256, k // 2), device=d, dtype=torch.uint8), torch.randint(0, 256, (4, k, 64), device=d, dtype=torch.uint8)
c13, c2 = torch.full((4, 256, k // 32), 120, dtype=torch.uint8, device=d), torch.full((4, k, 4), 120, dtype=torch.uint8, device=d)

def calls():
    outs = []
    for x, b in [(x, w) for x in xs] + [(long, wl)]:
        m, kk = x.shape
        q, a = torch.empty(m, kk // 2, dtype=torch.uint8, device=d), torch.empty(ops.packed_mxfp4_bytes(m, kk), dtype=torch.uint8, device=d)
        outs.append(torch.empty(m, b.shape[0], dtype=torch.bfloat16, device=d))
        ops.mxfp4_linear(x, q, a, b, sf[id(b)], outs[-1])
    q, s = torch.empty(3, k // 2, dtype=torch.uint8, device=d), torch.empty(3, k // 32, dtype=torch.uint8, device=d)
    ops.silu_mul_quant_mxfp4(gate, q, s)
    return outs + [q, s, moe.few_tokens_moe(xs[0], lg, e13, c13, e2, c2, 2)]

torch.cuda.synchronize()
start, got, failed = threading.Barrier(6), [None] * 6, []

def work(i):
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            start.wait()
            got[i] = calls()
            torch.cuda.current_stream().synchronize()
    except Exception as e:
        failed.append(e)

threads = [threading.Thread(target=work, args=(i,)) for i in range(6)]
for t in threads:
    t.start()
for t in threads:
    t.join()
assert not failed, failed
want = calls()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for g in got for a, b in zip(g, want)) and all(torch.isfinite(o.float()).all() for o in want) and ops.gemm_status(d) == 0
print("same")
"""


def test_first_calls_of_a_process_from_six_threads(cuda_dev):
    r = subprocess.run([sys.executable, "-c", THREADS], capture_output=True, text=True, timeout=240, cwd=pathlib.Path(__file__).parents[1])
    assert r.returncode == 0 and "same" in r.stdout, r.stdout + r.stderr
