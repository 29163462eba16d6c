"""GPU test that a CUDA failure is reported once, by the call that met it."""

import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

pytest.importorskip("torch")

# A validation loss waits for its stream, which CUDA refuses while the stream is captured;
# the lookup behind it is a good call with memory of its own. In a process of its own:
# torch's allocator does not come back from a capture that was broken off.
_CODE = """
import torch
from modern_fm_b200.embedding import embedding_lookup
from modern_fm_b200.evaluate import fm_eval_device

one = lambda *s: torch.ones(s, device="cuda", dtype=torch.float64)
ip, ix = torch.arange(9, device="cuda"), torch.arange(8, device="cuda", dtype=torch.int32)
args = (ip, ix, one(8), 0.0, one(8), one(8, 4), one(8))
table, out = torch.randn(8, 4, device="cuda"), torch.empty(8, 4, device="cuda")
side, home = torch.cuda.Stream(), torch.cuda.current_stream()
side.wait_stream(home)
want = fm_eval_device(*args, stream=side)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
failed = False
try:
    with torch.cuda.stream(side):
        graph.capture_begin()
        try:
            fm_eval_device(*args, stream=side)
        except RuntimeError:
            failed = True
        graph.capture_end()
except RuntimeError:
    pass
assert failed
embedding_lookup(table, ix, out=out, stream=home)
home.synchronize()
assert torch.equal(out, table)
assert fm_eval_device(*args, stream=home) == want
print("good calls behind a failed one")
"""


def test_a_failed_call_leaves_no_error_behind():
    r = subprocess.run([sys.executable, "-c", "import sys; sys.path[:0] = " + repr(sys.path) + "\n" + _CODE],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "good calls" in r.stdout, r.stderr[-2000:]
