"""Vocabulary-row operators whose waits for a copy run out: the call ends, the
status says so, nothing beside the results is written, the GPU goes on.  Each
in a process of its own, with a time limit that a copy cannot or may not meet."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CODE = """
import torch
from tinylm_c_b200 import _lib, ops
ops.init(0)
status = _lib.lib().tl_device_status
seen = {_lib.TL_OK: 0, _lib.TL_ETIMEOUT: 0}

def guarded(*shape, dtype=torch.float32):
    n = 1
    for d in shape:
        n *= d
    flat = torch.full((n + 64,), 77, dtype=dtype, device="cuda")
    return flat[:n].view(*shape), flat[n:]

def done(guards, check):
    rc = status()
    assert rc in seen, rc
    seen[rc] += 1
    assert all((g == 77).all().item() for g in guards)
    if rc == _lib.TL_OK:
        check()

# a cluster, one computing warp, one piece, several pieces, the first two with fewer rows than blocks
for N, V, dtype in ((3, 40000, torch.bfloat16), (40, 300, torch.float32), (3000, 300, torch.float32),
                    (700, 4100, torch.float32), (700, 40001, torch.bfloat16), (200, 140000, torch.bfloat16)):
    gen = torch.Generator(device="cuda").manual_seed(V)
    z = torch.randn(N, V, generator=gen, device="cuda").to(dtype)
    z[::3] = 1.0                                     # rows whose candidates overflow their list
    want = torch.log_softmax(z.double(), 1)
    ids = torch.zeros(N, dtype=torch.int32, device="cuda")
    for K in (0, 7, 128):
        (lp, g0), (H, g1) = guarded(N), guarded(N)
        (ti, g2), (tl, g3) = guarded(N, max(K, 1), dtype=torch.int32), guarded(N, max(K, 1))
        ops.token_logprobs(z, ids, N, V, lp, entropy=H, K=K, top_ids=ti if K else None, top_logp=tl if K else None)
        done((g0, g1, g2, g3), lambda: torch.testing.assert_close(lp.double(), want[:, 0], rtol=1e-4, atol=1e-4))
    for K, tail, weighted, grad in ((5, False, True, True), (100, True, False, True), (33, True, True, False)):
        v, t = torch.topk(z.float() + torch.randn(N, V, generator=gen, device="cuda"), K, dim=1)
        v = v - torch.logsumexp(z.float(), 1, keepdim=True) - 1.0
        w = (torch.arange(N, device="cuda") % 4 != 1).float() if weighted else None
        (L, g0), (dz, g1) = guarded(N), guarded(N, V, dtype=dtype)
        ops.distill_topk(z, t.int(), v.contiguous(), N, V, K, L, dz if grad else None, weight=w, tail=tail)
        done((g0, g1), lambda: None)
a = torch.randn(512, 512, device="cuda", generator=gen)
torch.testing.assert_close((a @ a).double(), a.double() @ a.double(), rtol=1e-2, atol=1e-1)
assert status() == _lib.TL_OK
print("ended", seen[_lib.TL_OK], seen[_lib.TL_ETIMEOUT])
"""


TOKEN = """
import torch
from tinylm_c_b200 import _lib, ops
ops.init(0)
N, V, K = 3000, 300, 4
z = torch.randn(N, V, device="cuda")
v, t = torch.topk(z, K, dim=1)
v, t, L = v.contiguous(), t.int().contiguous(), torch.empty(N, device="cuda")
ids, a, stats = torch.full((N,), V, dtype=torch.int32, device="cuda"), torch.ones(N, device="cuda"), torch.ones(N, 2, device="cuda")
for _ in range(20):
    ops.distill_topk(z, t, v, N, V, K, L, torch.empty_like(z))
torch.cuda.synchronize()
for call in (lambda: ops.token_logprobs_bwd(torch.empty_like(z), z, ids, N, V, stats, a),
             lambda: ops.token_logprobs(z, ids, N, V, a), lambda: ops.distill_topk(z, t + V, v, N, V, K, L)):
    call()
status = _lib.lib().tl_device_status
print("status", status(), status())
ops.token_logprobs_bwd(torch.empty_like(z), z, ids, N, V, stats, a)
print(status())
"""


def test_a_bad_token_does_not_hide_an_expired_wait(cuda):
    """The status after a wait that ran out is that, whatever a later call found in its ids."""
    from tinylm_c_b200 import _lib
    env = dict(os.environ, TL_COPY_TIMEOUT_NS="0")
    r = subprocess.run([sys.executable, "-c", TOKEN], cwd=ROOT, capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0, r.stderr[-2000:]
    got = [int(x) for x in r.stdout.split("status")[1].split()]
    assert got == [_lib.TL_ETIMEOUT, _lib.TL_OK, _lib.TL_EINVAL]


@pytest.mark.parametrize("limit_ns", [2000000000, 100000, 10000, 3000, 1000, 300, 0])
def test_waits_that_run_out(cuda, limit_ns):
    env = dict(os.environ, TL_COPY_TIMEOUT_NS=str(limit_ns))
    r = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0, r.stderr[-2000:]
    ok, out = map(int, r.stdout.split("ended")[1].split())
    print(limit_ns, "ns:", ok, "calls ended in time,", out, "did not")
    assert ok + out == 36
    if limit_ns == 2000000000:
        assert out == 0
    if limit_ns <= 300:              # the barrier itself waits for a microsecond or two before it is looked at again
        assert out > 0


@pytest.mark.parametrize("text", ["", "soon", "-5"])
def test_a_limit_that_is_none_is_not_taken(cuda, text):
    env = dict(os.environ, TL_COPY_TIMEOUT_NS=text)
    r = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.split("ended")[1].split() == ["36", "0"]
