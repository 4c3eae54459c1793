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
