"""Vocabulary-row operators at the limits of what they accept: large upstream
gradients, the longest rows, refused and unusual arguments."""
import numpy as np
import pytest
import torch

import logits_ref as ref
from tinylm_c_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def f64(t):
    return t.detach().double().cpu().numpy()


def logits(seed, N, V, dtype):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(N, V, generator=gen, device="cuda") * 3).to(DT[dtype])


def scored(z, tau):
    N, V = z.shape
    H, stats = torch.empty(N, device="cuda"), torch.empty(N, 2, device="cuda")
    ops.token_logprobs(z, None, N, V, None, entropy=H, stats=stats, temperature=tau)
    return H, stats


@pytest.mark.parametrize("tau,b", [(1e-6, 500.0), (1e-6, -3e4), (1e-4, 65536.0), (0.03, 1e9), (1.0, 1e12), (1.0, -1e30),
                                   (50.0, 1.0), (1e6, 1e6)])
def test_entropy_gradient_of_large_upstream_values(cuda, tau, b):
    """Tokens without probability have no gradient however large dentropy / temperature is: rows with
    tokens masked by -inf and by the type's lowest value, and tokens far below the largest logit."""
    for N, V, dtype in ((4, 3000, "f32"), (4, 40000, "bf16"), (4, 300, "bf16")):
        z = logits(V, N, V, dtype)
        some = torch.arange(V, device="cuda") % 7 == 0
        z[0, some] = float("-inf")
        z[1, some] = torch.finfo(z.dtype).min
        z[2, 1:] = float("-inf")
        H, stats = scored(z, tau)
        up = np.full(N, b, np.float32) * np.float32([1, -1, 1, 0.5])
        want, tol = ref.score_grad(f64(z), np.full(N, -1), tau, None, up, dtype)
        dz = torch.empty_like(z)
        ops.token_logprobs_bwd(dz, z, None, N, V, stats, None, entropy=H, dentropy=torch.from_numpy(up).cuda(),
                               temperature=tau)
        # a p below 2^-126 may be taken as 0 (logits_ref allows it for factors up to 2^26 only): its
        # |log p + H| is under 128 where the gradient can be told from 0
        tol = tol + 2.0 ** -126 * 128 * np.abs(up.astype(np.float64))[:, None] / tau
        ref.close(f64(dz), want, tol, f"dlogits {N} x {V} {dtype}")
    assert _lib.lib().tl_device_status() == _lib.TL_OK


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_sums_of_the_longest_rows(cuda, dtype):
    """Rows of equal logits behind 2048 larger ones, 2^18 in all, more rows than SMs: every thread's terms
    round the same way, so a sum shows how many it adds one after another.  The logarithm of a row's sum
    is off by the sum's bound and its own rounding, the entropy by its bound."""
    N, V, first = 300, 1 << 18, 2048
    below = torch.linspace(0.01, 3.0, N, device="cuda").to(DT[dtype])
    z = (-below)[:, None].expand(N, V).contiguous()
    z[:, :first] = 0.0
    logp, H, stats = torch.empty(N, device="cuda"), torch.empty(N, device="cuda"), torch.empty(N, 2, device="cuda")
    ids = torch.arange(N, device="cuda", dtype=torch.int32) * 811 + first
    ops.token_logprobs(z, ids, N, V, logp, entropy=H, stats=stats)
    d = f64(below)
    total = first + (V - first) * np.exp(-d)
    ls = np.log(total)
    ref.close(f64(stats[:, 1]), ls, ref.a_bound(V) + 2 * ref.U * ls, "log of the sum")
    ref.close(f64(logp), -d - ls, ref.logp_bound(-d - ls, V), "logp")
    ref.close(f64(H), ls + (V - first) * np.exp(-d) * d / total, ref.entropy_bound(V), "entropy")
    # a loss is -log p of one named token
    K, one = 1, torch.zeros(N, 1, device="cuda")
    loss, dz = torch.empty(N, device="cuda"), torch.empty_like(z)
    ops.distill_topk(z, ids[:, None].contiguous(), one, N, V, K, loss, dz)
    ref.close(f64(loss), d + ls, ref.a_bound(V) + 2 * ref.U * (d + ls), "loss")
    assert _lib.lib().tl_device_status() == _lib.TL_OK
