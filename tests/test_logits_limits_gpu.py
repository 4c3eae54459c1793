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


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,V,gap", [(5, 100, 0), (4, 1001, 3), (400, 3001, 0), (200, 20011, 1)])
def test_gradient_between_the_rows(cuda, dtype, N, V, gap):
    """Logits and their gradient as the halves of one buffer's rows, in both orders: the same bits as
    with the gradient in other memory (sums go by where in 16 bytes a row starts, so in the same places
    there), the logits and what lies between left as they were."""
    z = logits(V, N, V, dtype)
    ids = torch.arange(N, device="cuda", dtype=torch.int32) % V
    v, t = torch.topk(z.float(), 7, dim=1)
    v, t = v.contiguous(), t.int().contiguous()
    H, stats = scored(z, 1.0)
    a, loss = torch.ones(N, device="cuda"), torch.empty(N, device="cuda")
    for flip in (False, True):
        both, other = (torch.full((N, 2 * V + gap), 77.0, dtype=DT[dtype], device="cuda") for _ in range(2))
        at = [slice(0, V), slice(V + gap, 2 * V + gap)]
        zi, di, own = both[:, at[flip]], both[:, at[not flip]], other[:, at[not flip]]
        zi.copy_(z)
        keep = both.clone()
        for run in (lambda d: ops.token_logprobs_bwd(d, zi, ids, N, V, stats, a, entropy=H, dentropy=a),
                    lambda d: ops.distill_topk(zi, t, v, N, V, 7, loss, d)):
            run(own)
            run(di)
            assert torch.equal(di, own) and torch.equal(zi, z)
        di.fill_(77.0)
        assert torch.equal(both, keep)
    assert _lib.lib().tl_device_status() == _lib.TL_OK


def test_gradient_rows_that_share_elements(cuda):
    """Refused: one element shared with the next row on either side, rows apart at another stride."""
    V = 64
    flat = torch.zeros(4000, device="cuda")
    ids, out, stats = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.empty(4, device="cuda"), torch.zeros(4, 2, device="cuda")

    def rows(start, ld):
        return torch.as_strided(flat, (4, V), (ld, 1), start)

    for z, d in ((rows(0, 2 * V), rows(V - 1, 2 * V)), (rows(0, 2 * V), rows(V + 1, 2 * V)), (rows(V + 1, 2 * V), rows(0, 2 * V)),
                 (rows(0, 2 * V), rows(V, 2 * V + 1)), (rows(0, 2 * V - 1), rows(V, 2 * V - 1))):
        with pytest.raises(_lib.TLError) as e:
            ops.token_logprobs_bwd(d, z, ids, 4, V, stats, out)
        assert e.value.code == _lib.TL_EINVAL
        with pytest.raises(_lib.TLError):
            ops.distill_topk(z, ids, out, 4, V, 1, out, d)
    ops.token_logprobs_bwd(rows(V, 2 * V), rows(0, 2 * V), ids, 4, V, stats, out)
