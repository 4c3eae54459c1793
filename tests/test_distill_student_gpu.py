"""Distillation of the device model: what a refused step leaves as it was."""
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
