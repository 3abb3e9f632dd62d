"""A backward captured into a graph beside an eager graph of the same leaves: refused before torch's engine brings the default stream into the capture.  In a process
of its own, which has to go on: eager gradients, and a capture with leaves of its own."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = '''
import sys
import torch
import wav2sleep_amd as W
name = sys.argv[1]
R = lambda *s: torch.randn(*s, device='cuda')
x, gy = R(2, 40, 16), R(2, 40, 16)
if name == 'short_conv':
    leaves = [x, R(16, 4), R(16)]
    op = lambda v: W.short_conv(*v)
elif name == 'ssm_scan':
    leaves = [x, R(2, 40, 16), -torch.rand(16, 8, device='cuda'), R(2, 40, 8), R(2, 40, 8), R(16), R(2, 40, 16), R(16)]
    op = lambda v: W.ssm_scan(*v)
else:
    leaves = [x, R(16), R(2, 40, 16)]
    op = lambda v: W.add_rms_norm(*v)[0]
fresh = lambda: [t.detach().requires_grad_(True) for t in leaves]
grads = lambda v: torch.autograd.grad(op(v), v, gy)
side = torch.cuda.Stream()
with torch.cuda.stream(side):
    grads(fresh())
torch.cuda.synchronize()
old = fresh()
alive = op(old)                      # an eager graph of these leaves, on the default stream
g = torch.cuda.CUDAGraph()
try:
    with torch.cuda.graph(g):
        grads(old)
except RuntimeError as e:
    assert 'captured while an eager graph' in str(e), e
    print('refused', flush=True)
else:
    raise SystemExit('not refused')
torch.cuda.synchronize()
want = torch.autograd.grad(alive, old, gy)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):            # beside the living graph: leaves of its own
    got = grads(fresh())
for _ in range(3):
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
fixed = old[1].detach().requires_grad_(True)
keep = op([t.detach() if i != 1 else fixed for i, t in enumerate(old)])   # an eager graph of one leaf, whose gradient the capture does not ask for
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    v = [t if i != 1 else fixed for i, t in enumerate(fresh())]
    got = torch.autograd.grad(op(v), v[0], gy)
g.replay()
torch.cuda.synchronize()
assert torch.equal(got[0], want[0])
print('went on', flush=True)
'''


@pytest.mark.parametrize('name', ['short_conv', 'ssm_scan', 'add_rms_norm'])
def test_a_captured_backward_beside_an_eager_graph(name):
    r = subprocess.run([sys.executable, '-c', CHILD, name], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.split('\n')[-3:-1] == ['refused', 'went on'], (r.returncode, r.stdout[-2000:], r.stderr[-2000:])
