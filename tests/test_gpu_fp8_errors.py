"""A launch that the driver refuses fails its own call and no later one."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

REPO = Path(__file__).resolve().parents[1]

# A capture that a host call has made invalid refuses every launch; nothing reaches the GPU. In a
# process of its own, whose capture state goes with it.
CODE = """
import torch
from aios_b200 import _lib
from aios_b200.kernel import ops

x = torch.randn(8, 256, device="cuda").to(torch.bfloat16)
g = torch.ones(256, dtype=torch.bfloat16, device="cuda")
q, s = ops.quantize_fp8(x)
wq, ws = ops.quantize_weight_fp8(torch.randn(64, 256, device="cuda").to(torch.bfloat16))
want = ops.linear_fp8(q, s, wq, ws)
out = torch.empty_like(want)
torch.cuda.synchronize()
side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
with torch.cuda.stream(side):
    graph.capture_begin()
    try:
        side.synchronize()
    except RuntimeError:
        pass
    lib = _lib.load()
    rc = lib.aiosb_quantize_fp8(x.data_ptr(), 8, 256, 256, q.data_ptr(), s.data_ptr(), side.cuda_stream)
    assert rc == _lib.ERR_LAUNCH, rc
    rc = lib.aiosb_linear_fp8(q.data_ptr(), 256, s.data_ptr(), 8, 256, wq.data_ptr(), ws.data_ptr(), 64,
                              out.data_ptr(), 64, 0, None, 0, None, side.cuda_stream)
    assert rc == _lib.ERR_LAUNCH, rc
    try:
        graph.capture_end()
    except RuntimeError:
        pass
stream = torch.cuda.current_stream().cuda_stream
seeds, u = torch.arange(4, device="cuda"), torch.empty(4, 2, device="cuda")
for rc in (lib.aiosb_stateless_uniforms(seeds.data_ptr(), 4, 2, u.data_ptr(), stream),
           lib.aiosb_quantize_fp8(x.data_ptr(), 8, 256, 256, q.data_ptr(), s.data_ptr(), stream),
           lib.aiosb_linear_fp8(q.data_ptr(), 256, s.data_ptr(), 8, 256, wq.data_ptr(), ws.data_ptr(), 64,
                                out.data_ptr(), 64, 0, None, 0, None, stream)):
    assert rc == _lib.OK, _lib.last_error()
torch.cuda.synchronize()
assert torch.equal(out, want)
print("FINE")
"""


def test_a_refused_launch_is_not_reported_by_the_next_call(cuda_device) -> None:
    proc = subprocess.run([sys.executable, "-c", CODE], cwd=REPO, capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0 and "FINE" in proc.stdout, proc.stderr[-2000:]
