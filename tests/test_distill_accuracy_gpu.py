"""Distillation of rows whose loss is small against the terms that make it up
(a confident student, a student close to its teacher), against 64 bits with
bounds relative to the result.

Apart from the tokens not named, whose exponentials are summed in fp32, a row's
K entries are worked out in double.  So one error is left: with p_n and p_r the
student's mass of the named tokens and of the others, q_n and q_r the
teacher's, p_r's sum is off by a factor 1 + delta,

  delta <= A + (4 D + 8) u     (A: the bound of an fp32 sum, logits_ref; D: the
                                distance of the two parts' largest logits over
                                the temperature; u = 2^-24)

which moves p_r by delta p_r p_n only, p_n by as much the other way, and

  the loss by                         delta |q_n p_r - q_r p_n|,
  Q p_v - q_v of a named token by     delta Q p_v p_r,
  another token's p_v (Q - q_r/p_r),  delta (p_v/p_r) (q_r + 2 Q p_r) at most,
                                      and (4 |y_v - y_max| + 12) u of itself.

What is worked out in double is off by a few 2^-53 of the terms: under ten
roundings on q and on p each.
"""
import numpy as np
import pytest
import torch

import logits_ref as ref
from tinylm_c_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def exact(z, ids, vals, tau, tail, scale, dtype):
    """Losses and gradient of scale * their sum in 64 bits, with their bounds."""
    N, V = z.shape
    L, Lt, G, Gt = np.zeros(N), np.zeros(N), np.zeros((N, V)), np.zeros((N, V))
    rel, least = ref.half_step(dtype)
    k = scale / tau
    for n in range(N):
        on = ids[n] >= 0
        v, t = ids[n][on], vals[n][on].astype(np.float64)
        q = np.exp(t) if tail else np.exp((t - t.max()) / tau)
        q = q if tail else q / q.sum()
        qn = q.sum()
        qr = 1.0 - qn if tail and 1.0 - qn >= ref.TAIL_MIN else 0.0
        y = z[n] / tau
        named = np.zeros(V, bool)
        named[v] = True
        e = np.exp(y - y.max())
        en, er = e[named].sum(), e[~named].sum()
        all_, pn, pr = en + er, en / (en + er), er / (en + er)
        D = abs(y[named].max() - y[~named].max())
        delta = ref.a_bound(V) + (4 * D + 8) * ref.U
        logp = y - y.max() - np.log(all_)
        L[n] = (q * (np.log(q) - logp[v])).sum()
        if qr > 0:
            L[n] += qr * (np.log(qr) - np.log(er) + np.log(all_))
        Lt[n] = delta * abs(qn * pr - qr * pn) + 4 * ref.U * abs(L[n]) + 1e-14
        p, Q = e / all_, qn + qr
        dense = np.zeros(V)
        dense[v] = q
        g = np.where(named, Q * p - dense, p * (Q - qr / pr))
        mine = np.where(named, delta * Q * p * pr, delta * p / pr * (qr + 2 * Q * pr))
        own = np.where(named, 4.0, 4 * np.abs(y - y[~named].max()) + 12) * ref.U * np.abs(g)
        own += 10 * 2.0 ** -53 * np.where(named, Q * p + dense, 0.0)
        G[n], Gt[n] = k * g, k * (mine + own) * (1 + rel) + rel * k * np.abs(g) + least
    return L, Lt, G, Gt


def rows(seed, N, V, dtype):
    """A trained model's logits: a wide body and a few likely tokens a row."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    z = torch.randn(N, V, generator=gen, device="cuda") * 2
    likely = torch.randint(0, V, (N, 4), generator=gen, device="cuda")
    z.scatter_add_(1, likely, torch.rand(N, 4, generator=gen, device="cuda") * 12)
    return z.to(DT[dtype]), gen


def teacher(z, gen, K, tau, tail, noise):
    t = z.float() + noise * torch.randn(z.shape, generator=gen, device="cuda")
    vals, ids = torch.topk(t.double(), K, dim=1)
    if tail:
        vals = vals / tau - torch.logsumexp(t.double() / tau, 1, keepdim=True)
    return ids.int(), vals.float()


def check(z, ids, vals, tau, tail, dtype, pick=None):
    N, V = z.shape
    K, scale = ids.shape[1], 4096.0 if dtype == "f16" else 0.25
    loss, dz = torch.empty(N, device="cuda"), torch.empty_like(z)
    ops.distill_topk(z, ids, vals, N, V, K, loss, dz, scale=scale, temperature=tau, tail=tail)
    at = torch.arange(N, device="cuda") if pick is None else pick
    f64 = lambda t: t[at].double().cpu().numpy()  # noqa: E731
    L, Lt, G, Gt = exact(f64(z), ids[at].cpu().numpy(), vals[at].cpu().numpy(), tau, tail, scale, dtype)
    ref.close(f64(loss), L, Lt, "loss")
    ref.close(f64(dz), G, Gt, "dlogits")
    assert _lib.lib().tl_device_status() == _lib.TL_OK
    return L


# every layout of the rows: one computing warp, one piece, several pieces, a cluster
SHAPES = [(5, 231, "f32"), (1, 619, "f16"), (3, 5000, "f32"), (2, 8192, "bf16"), (2, 20010, "bf16"), (1, 20000, "f32")]


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("tau", [0.5, 1.0, 2.0])
@pytest.mark.parametrize("K", [1, 3, 30, 100])
@pytest.mark.parametrize("N,V,dtype", SHAPES)
def test_student_near_its_teacher(cuda, N, V, dtype, K, tau, tail):
    for seed in range(4):
        z, gen = rows(seed * 1000 + V + K, N, V, dtype)
        check(z, *teacher(z, gen, K, tau, tail, 1.0), tau, tail, dtype)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("gap", [4.0, 9.0, 14.0, 30.0])
def test_confident_student(cuda, gap, tail):
    """Nearly all of the mass on the one or the few tokens that the teacher names."""
    for N, V, dtype, K in ((4, 300, "f32", 1), (4, 4096, "f32", 2), (3, 9000, "bf16", 1), (2, 30000, "f32", 5)):
        z, gen = rows(V + int(gap), N, V, dtype)
        ids, vals = teacher(z, gen, K, 1.0, tail, 0.5)
        z.scatter_(1, ids.long(), (z.float().amax(1, keepdim=True) + gap).to(z.dtype).expand(N, K).contiguous())
        L = check(z, ids, vals, 1.0, tail, dtype)
        assert np.isfinite(L).all()


@pytest.mark.parametrize("tail", [False, True])
def test_close_student_of_many_rows(cuda, tail):
    """More rows than SMs, in one piece and in several: a teacher's noise of a tenth, losses near 1e-3."""
    pick = torch.tensor([0, 1, 7, 80, 150, 151, 152, 299], device="cuda")
    for V, dtype, K in ((700, "f32", 20), (8192, "f32", 64), (50001, "f16", 100), (100003, "bf16", 32)):
        z, gen = rows(V, 300, V, dtype)
        check(z, *teacher(z, gen, K, 2.0, tail, 0.1), 2.0, tail, dtype, pick)
