"""A launch that the CUDA runtime refuses is reported by the call that made it and by no later one."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
pytest.importorskip("torch")

# Launches on a stream whose capture has been invalidated (here by a synchronisation inside it) are refused by the runtime on the host.
# In a process of its own: the abandoned capture would outlive the test.
_CHILD = """
import torch
from accera_b200 import runtime as rt

zeros = lambda *shape, dtype=torch.float32: torch.zeros(*shape, device="cuda", dtype=dtype)
f8 = torch.float8_e4m3fn
table, ids, rows = zeros(10, 16), zeros(4, dtype=torch.int64), zeros(4, 16)
many, long_rows = zeros(4000, dtype=torch.int64), zeros(4000, 16)
q, s, C = zeros(4, 16, dtype=f8), zeros(4, 1), zeros(4, 4)
scale = s[:1].t().contiguous()
calls = {
    "embedding": lambda: rt.embedding(table, ids, rows),
    "few": lambda: rt.embedding_grad(rows, ids, table),
    "sorted": lambda: rt.embedding_grad(long_rows, many, table),
    "quantize": lambda: rt.quantize_fp8(rows, q, s),
    "gemm": lambda: rt.gemm_fp8(q, q.t(), C, s, scale, beta=0.0),
    "simt": lambda: rt.gemm_fp8(q, q.t(), C, s, scale, beta=0.0, compute="simt"),
}
data, where, out = zeros(8, 16), zeros(3, 1, dtype=torch.int64), zeros(3, 1, 16)
for call in calls.values():
    call()
rt.gather_rank2(data, where, out)
rt.synchronize()

graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
torch.cuda.synchronize()
with torch.cuda.stream(stream):
    graph.capture_begin(capture_error_mode="relaxed")
    try:
        stream.synchronize()
        raise SystemExit("the capture was not invalidated")
    except RuntimeError:
        pass
for name, call in calls.items():
    with torch.cuda.stream(stream):
        try:
            call()
            raise SystemExit(name + ": accepted")
        except rt.AccbError as e:
            assert e.code == rt.ERR_CUDA, (name, e)
    rt.gather_rank2(data, where, out)          # on the default stream: nothing is wrong with it
    print(name, flush=True)
import os
os._exit(0)                                    # without the graph's destructor
"""


def test_a_refused_launch_leaves_nothing_for_the_next_call():
    r = subprocess.run([sys.executable, "-c", _CHILD], capture_output=True, text=True, timeout=300,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0 and r.stdout.split() == ["embedding", "few", "sorted", "quantize", "gemm", "simt"], r.stdout + r.stderr
