"""Distillation of the device model: its gradient against differences along it
whose step error is taken out, and what a refused step leaves as it was."""
import numpy as np
import pytest
import torch

from tinylm_c_b200 import _lib, model

pytestmark = pytest.mark.gpu


def setting(cuda, B=2, K=16, tau=2.0):
    """The nano preset with weights large enough that its distributions are not flat, and the most
    likely tokens of a teacher of other weights; seeded throughout."""
    cfg = model.cfg8("nano")
    m = model.Model(cfg, 2)
    n = B * m.T
    rng = np.random.default_rng(41)
    tok = torch.from_numpy(rng.integers(0, cfg[0], n).astype(np.int32)).to(cuda)
    w = torch.from_numpy(((rng.random(n) + 0.5) * (rng.random(n) > 0.2)).astype(np.float32)).to(cuda)
    Pt, P = (model.init_params(cfg, seed).to(cuda) * 3.0 for seed in (43, 45))     # odd: 42 gives 43's
    ids, lp = torch.empty(n, K, dtype=torch.int32, device=cuda), torch.empty(n, K, device=cuda)
    m.score(Pt, tok, None, B, None, K=K, top_ids=ids, top_logp=lp, temperature=tau)
    return m, P, tok, ids, lp, w, dict(K=K, B=B, weight=w, temperature=tau)


@pytest.mark.parametrize("tail", [False, True])
def test_gradient_against_differences(cuda, tail):
    """f(P + h g) - f(P - h g) over 2 h |g|^2 is 1 + c h^2 + O(h^4) for the gradient g.  A step that
    changes the loss by 1 % has c h^2 of 2 % at such weights, which the quotients of h and h / 2 take
    out: (4 q(h/2) - q(h)) / 3 is off by O(h^4), a fourth of a percent of that 2 % or less where the
    quotients' own distance from 1 falls by about 4; and by the losses' rounding, 2^-24 of a loss over
    a change of 1 % of it, 2^-24 / 0.01 each, taken 16 / 3 and 4 / 3 times."""
    m, P, tok, ids, lp, w, kw = setting(cuda)
    G, loss = torch.zeros_like(P), torch.zeros(1, device=cuda)
    m.distill(P, G, tok, ids, lp, tail=tail, loss_out=loss, **kw)
    g2 = float(G.double().square().sum())

    def quotient(h):
        out = []
        for x in (P + h * G, P - h * G):
            m.distill(x, None, tok, ids, lp, tail=tail, loss_out=loss, **kw)
            out.append(loss.item())
        return (out[0] - out[1]) / (2 * h * g2)

    h = 0.01 * loss.item() / g2
    a, b = quotient(h), quotient(h / 2)
    assert abs(a - 1) < 0.05                      # the step is small enough for the two terms to say it
    # the model's products carry its gradients to 1e-4, the losses' rounding 8 * 2^-24 / 0.01, the step's
    # fourth power a twentieth of its square's effect at most
    tol = 1e-4 + 8 * 2.0 ** -24 / 0.01 + abs(a - 1) / 20
    assert abs((4 * b - a) / 3 - 1) <= tol, (a, b)
    m.close()


def test_refused_steps_leave_the_gradient(cuda):
    m, P, tok, ids, lp, w, kw = setting(cuda)
    G, M, V = (torch.full_like(P, v) for v in (3.0, 1.0, 2.0))
    before = P.clone()
    L, n = _lib.lib(), P.numel()
    host = torch.zeros(8)

    def step(tok_=tok.data_ptr(), ids_=ids.data_ptr(), K=16, weight=None, B=2, tau=2.0, tail=0, t=1, loss=None, norm=None,
             M_=M.data_ptr()):
        return L.tl_model_distill_step(m.h, P.data_ptr(), G.data_ptr(), M_, V.data_ptr(), tok_, ids_, lp.data_ptr(), K,
                                       weight, B, tau, tail, 1e-3, t, 1.0, loss, norm)

    assert L.tl_sync() == 0
    for bad in (dict(K=0), dict(K=-1), dict(K=200), dict(B=3), dict(B=0), dict(tau=0.0), dict(tau=float("nan")), dict(tail=2),
                dict(t=0), dict(tok_=None), dict(ids_=None), dict(M_=None)):
        assert step(**bad) == _lib.TL_EINVAL, bad
    for bad in (dict(tok_=host.data_ptr()), dict(weight=host.data_ptr()), dict(loss=host.data_ptr()),
                dict(norm=host.data_ptr())):
        assert step(**bad) == _lib.TL_EPTR, bad
    assert step(ids_=ids.data_ptr() + 2) == _lib.TL_EALIGN
    torch.cuda.synchronize()
    assert L.tl_sync() == 0
    assert (G == 3.0).all() and (M == 1.0).all() and (V == 2.0).all() and torch.equal(P, before) and n == G.numel()
    m.close()
