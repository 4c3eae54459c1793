"""Refusals of the vocabulary-row operators: argument checks that need no GPU,
and the binding's own checks of tensors."""
import pytest
import torch

from tinylm_c_b200 import _lib, ops

P = 4096          # a pointer that is never followed: every call below is refused first


def score(dtype=0, ld=100, N=2, V=100, tau=1.0, ids=P, logp=P, entropy=None, stats=None, K=0, ti=None, tl=None):
    return _lib.lib().tl_token_logprobs(P, dtype, ld, ids, N, V, tau, logp, entropy, stats, K, ti, tl)


def grad(dtype=0, ld=100, ldd=100, N=2, V=100, tau=1.0, ids=P, stats=P, entropy=None, dlogp=P, dentropy=None):
    return _lib.lib().tl_token_logprobs_bwd(P, ldd, P, dtype, ld, ids, N, V, tau, stats, entropy, dlogp, dentropy)


def distill(dtype=0, ld=100, K=4, N=2, V=100, tau=1.0, tail=0, scale=1.0, loss=P, dz=P, ldd=100):
    return _lib.lib().tl_distill_topk(P, dtype, ld, P, P, K, N, V, tau, tail, None, scale, loss, dz, ldd)


ROWS = [dict(dtype=3), dict(dtype=-1), dict(N=-1), dict(N=(1 << 30) + 1), dict(V=0), dict(V=-5), dict(V=_lib.TL_VOCAB_MAX + 1, ld=1 << 20),
        dict(ld=99), dict(ld=-1), dict(ld=1 << 41), dict(tau=0.0), dict(tau=-1.0), dict(tau=float("nan")),
        dict(tau=float("inf")), dict(tau=1e-7), dict(tau=1e7)]


@pytest.mark.parametrize("fn", [score, grad, distill])
@pytest.mark.parametrize("bad", ROWS, ids=str)
def test_bad_rows_and_temperatures(fn, bad):
    assert fn(**bad) == _lib.TL_EINVAL
    assert _lib.lib().tl_last_error()


@pytest.mark.parametrize("bad", [dict(K=-1), dict(K=_lib.TL_TOPK_MAX + 1, V=1000, ld=1000), dict(K=101),
                                 dict(ids=None), dict(logp=None), dict(logp=None, ids=None), dict(K=0, ti=P),
                                 dict(K=0, tl=P)], ids=str)
def test_bad_score_arguments(bad):
    assert score(**bad) == _lib.TL_EINVAL


@pytest.mark.parametrize("bad", [dict(dlogp=None), dict(ids=None), dict(dlogp=None, dentropy=P), dict(ldd=99)], ids=str)
def test_bad_gradient_arguments(bad):
    assert grad(**bad) == _lib.TL_EINVAL


@pytest.mark.parametrize("bad", [dict(K=0), dict(K=-3), dict(K=_lib.TL_TOPK_MAX + 1, V=1000, ld=1000, ldd=1000),
                                 dict(K=101), dict(tail=2), dict(tail=-1), dict(scale=float("nan")),
                                 dict(scale=float("inf")), dict(loss=None, dz=None), dict(ldd=99)], ids=str)
def test_bad_distill_arguments(bad):
    assert distill(**bad) == _lib.TL_EINVAL


def test_largest_k_is_taken_up_to_the_context_check():
    """Arguments at their limits pass every check before the device's."""
    if torch.cuda.is_available():
        pytest.skip("the context check ends the call only without a GPU")
    big = dict(V=_lib.TL_VOCAB_MAX, ld=_lib.TL_VOCAB_MAX)
    assert score(K=_lib.TL_TOPK_MAX, ti=P, tl=P, **big) == _lib.TL_ENOINIT
    assert grad(ldd=_lib.TL_VOCAB_MAX, **big) == _lib.TL_ENOINIT
    assert distill(K=_lib.TL_TOPK_MAX, ldd=_lib.TL_VOCAB_MAX, **big) == _lib.TL_ENOINIT
    assert score(tau=1e-6) == _lib.TL_ENOINIT and score(tau=1e6) == _lib.TL_ENOINIT


def test_constants_match_header():
    import os
    import re
    src = open(os.path.join(os.path.dirname(_lib.LIB_PATH), "..", "include", "tinylm_cuda.h")).read()
    for name in ("TL_F32", "TL_BF16", "TL_F16", "TL_TOPK_MAX", "TL_VOCAB_MAX"):
        assert int(re.search(rf"#define {name}\s+(\d+)", src).group(1)) == getattr(_lib, name)


def test_binding_refuses_tensors_it_cannot_take():
    z, e, i = torch.zeros(2, 8), torch.zeros(2), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CPU tensor"):
        ops.token_logprobs(z, i, 2, 8, e)
    with pytest.raises(ValueError, match="CPU tensor"):
        ops.token_logprobs_bwd(z, z, i, 2, 8, torch.zeros(2, 2), e)
    with pytest.raises(ValueError, match="CPU tensor"):
        ops.distill_topk(z, i, e, 2, 8, 1, e, z)
    with pytest.raises(TypeError):
        ops.token_logprobs(1234, i, 2, 8, e)
    with pytest.raises(ValueError, match="bad sizes"):
        ops.token_logprobs(z, i, -1, 8, e)
    with pytest.raises(ValueError, match="bad sizes"):
        ops.distill_topk(z, i, e, 2, 0, 1, e, z)


def test_calls_run_on_the_tensor_s_device(monkeypatch):
    """Tensors of another device than the current one: the call is made with theirs current."""
    seen, current = [], [0]

    class On:
        def __init__(self, d):
            self.d = d

        def __enter__(self):
            self.before, current[0] = current[0], self.d

        def __exit__(self, *a):
            current[0] = self.before

    class Lib:
        def tl_token_logprobs(self, *a):
            seen.append(current[0])
            return 0

    t = type("T", (), {"device": type("D", (), {"index": 1})()})()
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", lambda d: On(d.index))
    monkeypatch.setattr(ops, "_prep", lambda t: seen.append(("prep", current[0])))
    monkeypatch.setattr(ops, "lib", Lib)
    ops._call_on(t, "tl_token_logprobs")
    current[0] = 1
    ops._call_on(t, "tl_token_logprobs")
    assert seen == [("prep", 1), 1, ("prep", 1), 1] and current[0] == 1


class Fake(torch.Tensor):
    """A CPU tensor that says it is on the GPU: the binding's shape and type checks come before any call."""
    is_cuda = True


def fake(t):
    return t.as_subclass(Fake)


@pytest.mark.parametrize("bad,error", [
    (dict(logits=torch.zeros(2, 8, dtype=torch.float64)), TypeError),
    (dict(logits=torch.zeros(2, 7)), ValueError),
    (dict(logits=torch.zeros(1, 8)), ValueError),
    (dict(logits=torch.zeros(2, 16)[:, ::2]), ValueError),
    (dict(logits=torch.zeros(8, 2).t()), ValueError),
    (dict(logits=torch.zeros(1, 8).expand(2, 8)), ValueError),
    (dict(logits=torch.zeros(15)), ValueError),
    (dict(ids=torch.zeros(2, dtype=torch.int64)), TypeError),
    (dict(ids=torch.zeros(1, dtype=torch.int32)), ValueError),
    (dict(logp=torch.zeros(2, dtype=torch.float64)), TypeError),
    (dict(logp=torch.zeros(4)[::2]), ValueError),
    (dict(entropy=torch.zeros(1)), ValueError),
    (dict(stats=torch.zeros(3)), ValueError),
    (dict(K=3, top_ids=torch.zeros(5, dtype=torch.int32), top_logp=torch.zeros(6)), ValueError),
    (dict(K=3, top_ids=torch.zeros(6), top_logp=torch.zeros(6)), TypeError),
])
def test_binding_checks_shapes_and_types(bad, error):
    args = dict(logits=torch.zeros(2, 8), ids=torch.zeros(2, dtype=torch.int32), logp=torch.zeros(2))
    args.update(bad)
    args = {k: fake(v) if isinstance(v, torch.Tensor) else v for k, v in args.items()}
    with pytest.raises(error):
        ops.token_logprobs(args.pop("logits"), args.pop("ids"), 2, 8, args.pop("logp"), **args)


def test_stream_without_torch_s_private_call(monkeypatch):
    """A torch that lacks the one-call form of the current stream: the public one is taken."""
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda idx: type("S", (), {"cuda_stream": 1234 + idx})())
    seen = []
    monkeypatch.setattr(ops, "_stream_set", {})
    monkeypatch.setattr(ops, "lib", lambda: type("L", (), {"tl_set_stream": lambda self, s: seen.append(s) or 0})())
    ops._bind_stream(1)
    ops._bind_stream(1)
    assert seen == [1235]
