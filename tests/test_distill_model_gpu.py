"""The device model scored and distilled (tl_model_score, tl_model_distill,
tl_model_distill_step): against its own cross-entropy paths, against
differences, and teacher to student as a user runs them."""
import numpy as np
import pytest
import torch

import logits_ref as ref
from tinylm_c_b200 import _lib, model, ops

pytestmark = pytest.mark.gpu


def batch(cfg, B, seed, dev):
    V, T = cfg[0], cfg[6]
    rng = np.random.default_rng(seed)
    tok = torch.from_numpy(rng.integers(0, V, B * T).astype(np.int32)).to(dev)
    tgt = torch.from_numpy(rng.integers(0, V, B * T).astype(np.int32)).to(dev)
    return tok, tgt


def params(cfg, seed, dev):
    """Initial parameters with larger weights, so that the model's distributions are not flat."""
    P = model.init_params(cfg, seed).to(dev)
    return P * 3.0


def scored(m, P, tok, tgt, B, K, tau=1.0):
    n, dev = B * m.T, P.device
    logp, H = torch.empty(n, device=dev), torch.empty(n, device=dev)
    ids, lp = torch.empty(n, K, dtype=torch.int32, device=dev), torch.empty(n, K, device=dev)
    m.score(P, tok, tgt, B, logp, entropy=H, K=K, top_ids=ids, top_logp=lp, temperature=tau)
    torch.cuda.synchronize()
    return logp, H, ids, lp


@pytest.mark.parametrize("preset,B,micro", [("nano", 4, 4), ("nano", 4, 1), ("m1", 2, 2), ("m8", 2, 1)])
def test_score_agrees_with_the_loss(cuda, preset, B, micro):
    """The mean of -log p over a batch is the forward pass's loss: the same logits, sums in another
    order (the row's bound), the loss's 1e-12 under its logarithm and its float result."""
    cfg = model.cfg8(preset)
    m = model.Model(cfg, micro)
    P = params(cfg, 1, cuda)
    tok, tgt = batch(cfg, B, 2, cuda)
    loss = torch.zeros(1, device=cuda)
    m.forward(P, tok, tgt, B, loss)
    logp, H, ids, lp = scored(m, P, tok, tgt, B, 8)
    want = -logp.double().mean().item()
    tol = 2 * float(ref.logp_bound(np.float64(logp.abs().max().item()), cfg[0])) + 1e-12 * np.exp(
        float(logp.abs().max())) + 2 * 2.0 ** -24 * abs(want)
    assert abs(loss.item() - want) <= tol, (loss.item(), want, tol)
    assert (lp[:, 0] >= logp - 1e-5).all() and (lp[:, :-1] >= lp[:, 1:]).all()
    assert (H > 0).all() and (H <= np.log(cfg[0]) + 1e-3).all()
    m.close()


@pytest.mark.parametrize("preset,B,micro", [("nano", 2, 2), ("nano", 4, 2), ("m1", 2, 2)])
def test_one_token_teacher_is_cross_entropy(cuda, preset, B, micro):
    """A teacher that names the target alone gives the cross-entropy's loss and gradient: the same
    backward pass from logits' gradients that agree to fp32 rounding (1e-4 as for the model's own
    gradients, relative in L2)."""
    cfg = model.cfg8(preset)
    m = model.Model(cfg, micro)
    P = params(cfg, 3, cuda)
    tok, tgt = batch(cfg, B, 4, cuda)
    Ga, Gb = torch.zeros_like(P), torch.zeros_like(P)
    la, lb = torch.zeros(1, device=cuda), torch.zeros(1, device=cuda)
    m.forward_backward(P, Ga, tok, tgt, None, B, la)
    vals = torch.zeros(B * m.T, 1, device=cuda)
    m.distill(P, Gb, tok, tgt.view(-1, 1), vals, 1, B, loss_out=lb)
    alone = torch.zeros(1, device=cuda)
    m.distill(P, None, tok, tgt.view(-1, 1), vals, 1, B, loss_out=alone)
    torch.cuda.synchronize()
    assert abs(la.item() - lb.item()) <= 1e-5 * abs(la.item())
    assert alone.item() == lb.item()
    rel = (Ga - Gb).double().norm() / Ga.double().norm()
    assert rel <= 1e-4, rel
    # gradients accumulate
    m.distill(P, Gb, tok, tgt.view(-1, 1), vals, 1, B)
    assert (Gb - 2 * Ga).double().norm() / Ga.double().norm() <= 2e-4
    m.close()


@pytest.mark.parametrize("tail", [False, True])
def test_teacher_to_student(cuda, tail):
    """A teacher's most likely tokens train a student: the loss's gradient against differences along
    it, steps equal to their parts, a student equal to its teacher has nothing to learn."""
    cfg, B, K, tau = model.cfg8("nano"), 2, 16, 2.0
    m = model.Model(cfg, 2)
    Pt, P = params(cfg, 5, cuda), params(cfg, 6, cuda)
    tok, tgt = batch(cfg, B, 7, cuda)
    _, _, ids, lp = scored(m, Pt, tok, tgt, B, K, tau)
    w = (torch.rand(B * m.T, device=cuda) + 0.5) * (torch.rand(B * m.T, device=cuda) > 0.2)
    G, loss = torch.zeros_like(P), torch.zeros(1, device=cuda)
    m.distill(P, G, tok, ids, lp, K, B, weight=w, temperature=tau, tail=tail, loss_out=loss)

    def at(x):
        out = torch.zeros(1, device=cuda)
        m.distill(x, None, tok, ids, lp, K, B, weight=w, temperature=tau, tail=tail, loss_out=out)
        return out.item()

    assert at(P) == loss.item() and loss.item() > 0
    # along the gradient: f(P + h g) - f(P - h g) = 2 h |g|^2 up to the third derivative; the step
    # moves the loss by about 2 %, and losses are floats (2^-24 each, sums of 1e-6)
    g2 = float(G.double().square().sum())
    h = 0.01 * loss.item() / g2
    diff = (at(P + h * G) - at(P - h * G)) / (2 * h)
    assert abs(diff - g2) <= 0.02 * g2, (diff, g2)
    # one step is distill + clip + AdamW, bit for bit
    n = P.numel()
    Pa, Ma, Va = P.clone(), torch.zeros_like(P), torch.zeros_like(P)
    Pb, Mb, Vb = P.clone(), torch.zeros_like(P), torch.zeros_like(P)
    Ga, norm, l2 = torch.full_like(P, 9.0), torch.zeros(1, device=cuda), torch.zeros(1, device=cuda)
    m.distill_step(Pa, Ga, Ma, Va, tok, ids, lp, K, B, 1e-3, 1, weight=w, temperature=tau, tail=tail, loss_out=l2,
                   norm_out=norm)
    Gb, nb = torch.zeros_like(P), torch.zeros(1, device=cuda)
    m.distill(Pb, Gb, tok, ids, lp, K, B, weight=w, temperature=tau, tail=tail)
    ops.clip_adamw(Pb, Gb, Mb, Vb, n, 1e-3, 0.9, 0.95, 0.1, 1, 1.0, nb)
    torch.cuda.synchronize()
    assert l2.item() == loss.item() and norm.item() == nb.item()
    assert torch.equal(Ga, Gb) and torch.equal(Pa, Pb) and torch.equal(Ma, Mb) and torch.equal(Va, Vb)
    # the teacher itself: with a tail its loss is 0 up to the rounding of log probabilities
    if tail:
        G0, l0 = torch.zeros_like(P), torch.zeros(1, device=cuda)
        m.distill(Pt, G0, tok, ids, lp, K, B, temperature=tau, tail=True, loss_out=l0)
        assert abs(l0.item()) <= 2e-5
        assert G0.double().norm() <= 1e-3 * G.double().norm()
    assert _lib.lib().tl_device_status() == _lib.TL_OK
    m.close()


def test_mtp_heads_get_no_gradient(cuda):
    cfg, B, K = model.cfg8("m1", 2), 2, 4
    m = model.Model(cfg, 2)
    P = params(cfg, 8, cuda)
    tok, tgt = batch(cfg, B, 9, cuda)
    _, _, ids, lp = scored(m, P * 0.5, tok, tgt, B, K)
    G = torch.zeros_like(P)
    m.distill(P, G, tok, ids, lp, K, B, tail=True)
    heads = 2 * cfg[1] * cfg[1]
    assert (G[-heads:] == 0).all() and (G[:-heads] != 0).any()
    m.close()


def test_training_steps_are_unchanged_beside_scoring(cuda):
    """Scoring and distilling between a model's ordinary steps, graph replays among them, leaves those
    steps' results as they are."""
    cfg, B = model.cfg8("nano"), 2
    tok, tgt = batch(cfg, B, 10, cuda)

    def run(between):
        m = model.Model(cfg, 2)
        P = params(cfg, 11, cuda)
        G, M, V = torch.zeros_like(P), torch.zeros_like(P), torch.zeros_like(P)
        loss, out = torch.zeros(1, device=cuda), []
        for t in range(1, 5):
            m.step(P, G, M, V, tok, tgt, None, B, 1e-3, t, 1.0, loss, graph=t % 2 == 0)
            out.append(loss.item())
            if between:
                _, _, ids, lp = scored(m, P, tok, tgt, B, 5)
                m.distill(P, torch.zeros_like(P), tok, ids, lp, 5, B)
        torch.cuda.synchronize()
        m.close()
        return out, P

    (a, Pa), (b, Pb) = run(False), run(True)
    assert a == b and torch.equal(Pa, Pb)


def test_refusals(cuda):
    cfg = model.cfg8("nano")
    m = model.Model(cfg, 2)
    P = params(cfg, 1, cuda)
    tok, tgt = batch(cfg, 2, 1, cuda)
    n = 2 * m.T
    logp = torch.empty(n, device=cuda)
    ids, vals = torch.zeros(n, 4, dtype=torch.int32, device=cuda), torch.zeros(n, 4, device=cuda)

    def refused(f, code=_lib.TL_EINVAL):
        with pytest.raises(_lib.TLError) as e:
            f()
        assert e.value.code == code

    big = torch.zeros(3 * m.T, dtype=torch.int32, device=cuda)
    refused(lambda: m.score(P, big, big, 3, torch.empty(3 * m.T, device=cuda)))          # no multiple of the micro-batch
    refused(lambda: m.score(P, tok, tgt, 2, logp, temperature=0.0))
    refused(lambda: m.score(P, tok, None, 2, logp))
    refused(lambda: m.score(P, tok, None, 2, None))
    refused(lambda: m.distill(P, None, tok, ids, vals, 4, 2))
    refused(lambda: m.distill(P, torch.zeros_like(P), tok, ids, vals, 4, 2, temperature=-1.0))
    refused(lambda: m.distill_step(P, P.clone(), P.clone(), P.clone(), tok, ids, vals, 4, 2, 1e-3, 0))
    with pytest.raises(ValueError):
        m.distill(P, torch.zeros_like(P), tok, ids, vals, 5, 2)                            # entries of 4 given
    with pytest.raises(ValueError):
        m.score(P, tok, tgt, 2, logp[:-1])
    L = _lib.lib()
    host = torch.zeros(n)
    assert L.tl_model_score(m.h, P.data_ptr(), tok.data_ptr(), tgt.data_ptr(), 2, 1.0, host.data_ptr(), None, 0, None,
                            None) == _lib.TL_EPTR
    assert L.tl_model_score(None, None, None, None, 2, 1.0, None, None, 0, None, None) == _lib.TL_EINVAL
    m.close()
