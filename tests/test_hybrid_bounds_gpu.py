"""The bounds-check build of the hybrid extension: an index on the device that is out of range is reported through the status word and its access goes into the
allocation.  In a child process, as in test_bounds_check_gpu.py."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

CHILD = r'''
import torch
from llaminar_b200 import ops
from llaminar_b200.ops import hybrid
dev, FAR = "cuda", 1_000_000
it = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
def told(call, want):
    call()
    torch.cuda.synchronize()
    assert hybrid.bounds_status() == (3 if want else 0), (call.__name__, want)
    assert hybrid.bounds_status() == 0

d, T = 128, 40
C, width = 3 * d, 4 * d + 2
rows = torch.randn(T, width, device=dev).to(torch.bfloat16)
state = lambda: (torch.zeros(2, C, 3, device=dev), torch.zeros(2, 1, d, d, device=dev))
args = (C, C, C + d, torch.randn(C, 4, device=dev), -torch.ones(1, device=dev), torch.ones(1, device=dev), torch.ones(d, device=dev))
pos = torch.arange(T, dtype=torch.int32, device=dev) + 5
out = torch.zeros(T, d, dtype=torch.bfloat16, device=dev)
for n in (T, 3):                                                   # in chunks, row by row
    prefill = lambda slot: ops.gdn_prefill(rows[:n], *args, *state(), pos[:n], it([0, n]), it([slot]), out[:n], 1, 0, 1e-6)
    told(lambda: prefill(1), False)
    told(lambda: prefill(FAR), True)
    told(lambda: prefill(-1), True)
kept = []
told(lambda: kept.append(ops.gdn_verify(rows[:3], *args, *state(), it([1]), out[:3], 1, 0, 1e-6)), False)
told(lambda: ops.gdn_verify(rows[:3], *args, *state(), it([2]), out[:3], 1, 0, 1e-6), True)
told(lambda: ops.gdn_commit(kept[0], it([2]), *state()), False)
kept[0].slots = it([FAR])
told(lambda: ops.gdn_commit(kept[0], it([2]), *state()), True)

H, Hk, D = 4, 2, 128
qkv = torch.randn(2, (H + 2 * Hk) * D, device=dev).to(torch.bfloat16)
q = torch.zeros(2, H, D, dtype=torch.bfloat16, device=dev)
kv = torch.zeros(9, 2, Hk, 64, D, dtype=torch.bfloat16, device=dev)
freqs = torch.ones(8, dtype=torch.float64, device=dev)
table = it([[1, 2, 0, 0], [3, 4, 0, 0]])
def rope(pos, sid, table):
    return lambda: ops.rope_part_kv(qkv, q, kv, None, None, freqs, 1.0, it(pos), it(sid), table, H, Hk, D, 1e-6)
told(rope([70, 71], [0, 1], table), False)
far = table.clone(); far[1, 1] = FAR
told(rope([70, 71], [0, 1], far), True)
told(rope([70, 71], [0, 2], table), True)
told(rope([70, 256], [0, 1], table), True)
kv.zero_()
told(rope([70, -1], [0, 1], it([[1, 2, 0, 0], [5, 6, 0, 0]])), True)
assert (kv[4] == 0).all()                                          # nothing lands in front of the sequence's first page

def shared(table, lens=(100, 100)):
    return lambda: ops.attn_decode_shared(q, kv, torch.empty_like(q), table, it(list(lens)), it([64]), H, Hk, D, 1, 0.1, ops.scratch_for(dev), max_shared=64)
told(shared(it([[1, 2, 0, 0], [1, 4, 0, 0]])), False)
told(shared(it([[FAR, 2, 0, 0], [FAR, 4, 0, 0]])), True)
told(shared(it([[1, 2, 0, 0], [1, -5, 0, 0]])), True)
assert int(ops.scratch_for(dev).status[0]) == 0
print("BOUNDS_CHECK_OK")
'''


def test_bounds_check_build_reports_bad_slots_pages_and_positions():
    env = dict(os.environ, LLAMINAR_BOUNDS_CHECK="1")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", CHILD], cwd=root, env=env, capture_output=True, text=True, timeout=1500)
    assert "BOUNDS_CHECK_OK" in r.stdout, r.stdout[-2000:] + r.stderr[-4000:]
