"""Host-side mirror of the reference's hot-path primitives, on CUDA tensors.

Same names, argument order and meaning as tinylm.c's static functions, so a
test or a driver reads like the reference's own code:

    mm(Y, X, W, M, K, N)                          tinylm.c:439-478
    mm_bt(dX, dY, W, M, K, N)                     tinylm.c:480-508
    mm_atb(dW, X, dY, M, K, N)                    tinylm.c:510-537
    global_gradnorm(G, n) -> float                tinylm.c:1171-1176
    adamw(P, G, M, V, n, lr, b1, b2, wd, t, gscale)   tinylm.c:1159-1170

Buffers are torch CUDA float32 tensors (torch supplies device memory and the
stream; every byte of arithmetic runs in libtinylm_cuda).  A CPU tensor raises:
there is no CPU fallback.  Errors raise TLError instead of the reference's
exit(1).
"""
import ctypes

import torch

from ._lib import check, lib

_inited = set()
_stream_set = {}


def init(device=0):
    """tl_init for `device` and bind the library to torch's current stream there."""
    device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
    idx = device.index if device.index is not None else torch.cuda.current_device()
    with torch.cuda.device(idx):
        if idx not in _inited:
            check(lib().tl_init(idx))
            _inited.add(idx)
        _bind_stream(idx)
    return idx


def _raw_stream(idx):
    """torch's current stream of a device as a cudaStream_t: in one call where this torch has it (a call of a
    few rows is as long as its way through Python), else by the public way."""
    try:
        return torch._C._cuda_getCurrentRawStream(idx)
    except AttributeError:
        return torch.cuda.current_stream(idx).cuda_stream


def _bind_stream(idx):
    s = _raw_stream(idx)
    if _stream_set.get(idx) != s:
        check(lib().tl_set_stream(s))
        _stream_set[idx] = s


def _ptr(t, name, numel=None):
    if isinstance(t, int):
        return t
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a CUDA tensor or a device pointer")
    if not t.is_cuda:
        raise ValueError(f"{name}: CPU tensor given; libtinylm_cuda computes on the GPU only")
    if t.dtype != torch.float32:
        raise TypeError(f"{name}: expected float32, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")
    if numel is not None and t.numel() < numel:
        raise ValueError(f"{name}: has {t.numel()} elements, call needs {numel}")
    return t.data_ptr()


def _prep(t):
    if isinstance(t, torch.Tensor) and not t.is_cuda:
        raise ValueError("CPU tensor given; libtinylm_cuda computes on the GPU only")
    idx = t.device.index if isinstance(t, torch.Tensor) else torch.cuda.current_device()
    if idx not in _inited:
        init(idx)
    else:
        _bind_stream(idx)


def mm(Y, X, W, M, K, N):
    """Y[M,N] = X[M,K] @ W[K,N] (overwrite)."""
    _prep(Y)
    check(lib().tl_matmul(_ptr(Y, "Y", M * N), _ptr(X, "X", M * K), _ptr(W, "W", K * N), M, K, N))


def mm_bt(dX, dY, W, M, K, N):
    """dX[M,K] += dY[M,N] @ W[K,N]^T (accumulate)."""
    _prep(dX)
    check(lib().tl_matmul_bt(_ptr(dX, "dX", M * K), _ptr(dY, "dY", M * N), _ptr(W, "W", K * N), M, K, N))


def mm_bt_sum(dX, dYs, Ws, Ns, M, K):
    """dX[M,K] = sum_t dYs[t][M,Ns[t]] @ Ws[t][K,Ns[t]]^T (overwrite), 1 to 3 products."""
    _prep(dX)
    n = len(Ns)
    if not (len(dYs) == len(Ws) == n):
        raise ValueError("dYs, Ws and Ns must have the same length")
    arr = ctypes.c_void_p * max(n, 1)
    a = arr(*[_ptr(x, "dY", M * nt) for x, nt in zip(dYs, Ns)])
    b = arr(*[_ptr(w, "W", K * nt) for w, nt in zip(Ws, Ns)])
    nn = (ctypes.c_int * max(n, 1))(*Ns)
    check(lib().tl_matmul_bt_sum(_ptr(dX, "dX", M * K), n, a, b, nn, M, K))


def mm_atb(dW, X, dY, M, K, N):
    """dW[K,N] += X[M,K]^T @ dY[M,N] (accumulate)."""
    _prep(dW)
    check(lib().tl_matmul_at(_ptr(dW, "dW", K * N), _ptr(X, "X", M * K), _ptr(dY, "dY", M * N), M, K, N))


def set_gemm_engine(engine):
    """0 automatic, 1 CUDA-core fp32, 2 tensor-core 3xTF32 (one CTA per
    128 x 128 tile), 3 tensor-core 3xTF32 (CTA pair per 256 x 256 tile),
    4 tensor-core CTA pair with scaled fp16 hi/lo operands (3 fp16 MMAs),
    5 tensor-core CTA pair with the hybrid split (tf32 hi*hi + bf16 cross
    terms)."""
    check(lib().tl_set_gemm_engine(int(engine)))


def set_attn_engine(engine):
    """Attention forward and backward: 0 automatic, 1 CUDA cores, 2 tensor
    cores (T=256, hd=64)."""
    check(lib().tl_set_attn_engine(int(engine)))


def last_gemm_engine():
    return lib().tl_last_gemm_engine()


def global_gradnorm(G, n):
    """sqrt(sum (double)G^2) as float; waits for the result like the reference."""
    _prep(G)
    out = ctypes.c_float(0.0)
    check(lib().tl_grad_norm(_ptr(G, "G", n), n, ctypes.addressof(out)))
    return out.value


def grad_norm_dev(G, n, out):
    """Device-side norm into out[0] (float32 CUDA tensor); no host sync."""
    _prep(G)
    check(lib().tl_grad_norm(_ptr(G, "G", n), n, _ptr(out, "out", 1)))


def adamw(P, G, M, V, n, lr, b1, b2, wd, t, gscale):
    """AdamW with the clip scale folded in (host scalar gscale)."""
    _prep(P)
    check(lib().tl_adamw_step(_ptr(P, "P", n), _ptr(G, "G", n), _ptr(M, "M", n), _ptr(V, "V", n), n,
                              lr, b1, b2, wd, int(t), gscale))


def adamw_dev(P, G, M, V, n, lr, b1, b2, wd, t, gscale_dev=None):
    """AdamW reading the clip scale from device memory (None = 1.0)."""
    _prep(P)
    gp = None if gscale_dev is None else _ptr(gscale_dev, "gscale_dev", 1)
    check(lib().tl_adamw_step_dev(_ptr(P, "P", n), _ptr(G, "G", n), _ptr(M, "M", n), _ptr(V, "V", n),
                                  n, lr, b1, b2, wd, int(t), gp))


def clip_adamw(P, G, M, V, n, lr, b1, b2, wd, t, max_norm=1.0, norm_out=None):
    """norm -> clip scale -> AdamW, all on the device (train_loop tinylm.c:2630-2633)."""
    _prep(P)
    no = None if norm_out is None else _ptr(norm_out, "norm_out", 1)
    check(lib().tl_clip_adamw_step(_ptr(P, "P", n), _ptr(G, "G", n), _ptr(M, "M", n), _ptr(V, "V", n),
                                   n, lr, b1, b2, wd, int(t), max_norm, no))


_ROW_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # TL_F32, TL_BF16, TL_F16


def _rows(t, name, N, V):
    """(pointer, row stride) of N rows of V logits: a tensor [>= N, >= V] whose rows are dense, or a
    contiguous one of at least N*V elements."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a CUDA tensor")
    if not t.is_cuda:
        raise ValueError(f"{name}: CPU tensor given; libtinylm_cuda computes on the GPU only")
    if t.dtype not in _ROW_DTYPES:
        raise TypeError(f"{name}: expected float32, bfloat16 or float16, got {t.dtype}")
    if t.dim() == 2:
        if t.shape[0] < N or t.shape[1] < V:
            raise ValueError(f"{name}: shape {tuple(t.shape)}, call needs [{N}, {V}]")
        if V > 1 and t.stride(1) != 1:
            raise ValueError(f"{name}: rows must be dense (stride {t.stride(1)} along them)")
        ld = t.stride(0) if N > 1 else V
        if ld < V:
            raise ValueError(f"{name}: row stride {ld} below V = {V}")
        return t.data_ptr(), ld
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be two-dimensional or contiguous")
    if t.numel() < N * V:
        raise ValueError(f"{name}: has {t.numel()} elements, call needs {N * V}")
    return t.data_ptr(), V


def _vec(t, name, numel, dtype=torch.float32):
    """Pointer of a contiguous CUDA tensor of at least numel elements; None passes through."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a CUDA tensor")
    if not t.is_cuda:
        raise ValueError(f"{name}: CPU tensor given; libtinylm_cuda computes on the GPU only")
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")
    if t.numel() < numel:
        raise ValueError(f"{name}: has {t.numel()} elements, call needs {numel}")
    return t.data_ptr()


def _call_on(t, name, *args):
    """Entry point `name` on t's device and torch's current stream there."""
    if t.device.index == torch.cuda.current_device():
        _prep(t)
        check(getattr(lib(), name)(*args))
        return
    with torch.cuda.device(t.device):
        _prep(t)
        check(getattr(lib(), name)(*args))


def _sizes(N, V, K):
    if N < 0 or V < 1 or K < 0:
        raise ValueError(f"bad sizes N = {N}, V = {V}, K = {K}")


def token_logprobs(logits, ids, N, V, logp, entropy=None, stats=None, K=0, top_ids=None, top_logp=None,
                   temperature=1.0):
    """Scores N rows of V logits (fp32, bf16 or fp16, any row stride).

    logp[n] = log p(ids[n]) (0 where ids[n] is -1; ids and logp may both be
    None), entropy[n], stats[n][2] (what token_logprobs_bwd needs) and the K
    most likely tokens top_ids[n][K] / top_logp[n][K].  ids and top_ids are
    int32, every other output float32; outputs left None are not computed.
    See tl_token_logprobs in tinylm_cuda.h for masked, empty and NaN rows.
    """
    _sizes(N, V, K)
    z, ld = _rows(logits, "logits", N, V)
    _call_on(logits, "tl_token_logprobs", z, _ROW_DTYPES[logits.dtype], ld, _vec(ids, "ids", N, torch.int32), N, V,
             temperature, _vec(logp, "logp", N), _vec(entropy, "entropy", N), _vec(stats, "stats", 2 * N), K,
             _vec(top_ids, "top_ids", N * K, torch.int32), _vec(top_logp, "top_logp", N * K))


def token_logprobs_bwd(dlogits, logits, ids, N, V, stats, dlogp, entropy=None, dentropy=None, temperature=1.0):
    """dlogits = gradient of sum dlogp*logp + dentropy*entropy in the logits.

    stats and entropy are those of token_logprobs at the same temperature;
    dlogp (with ids) or dentropy (with entropy) may be None.  dlogits has the
    logits' type and may be the logits tensor itself.
    """
    _sizes(N, V, 0)
    z, ld = _rows(logits, "logits", N, V)
    dz, ldd = _rows(dlogits, "dlogits", N, V)
    if dlogits.dtype != logits.dtype:
        raise TypeError(f"dlogits: expected {logits.dtype}, got {dlogits.dtype}")
    _call_on(logits, "tl_token_logprobs_bwd", dz, ldd, z, _ROW_DTYPES[logits.dtype], ld,
             _vec(ids, "ids", N, torch.int32), N, V, temperature, _vec(stats, "stats", 2 * N),
             _vec(entropy, "entropy", N), _vec(dlogp, "dlogp", N), _vec(dentropy, "dentropy", N))


def distill_topk(logits, t_ids, t_vals, N, V, K, loss, dlogits=None, weight=None, scale=1.0, temperature=1.0,
                 tail=False):
    """KL divergence of N student rows from a teacher's K most likely tokens.

    loss[n] = weight[n] * sum q log(q / p); dlogits, if given, receives the
    gradient of scale * sum(loss) and may be the logits tensor itself.  q is
    the softmax of t_vals / temperature over the row's tokens, or, with
    tail=True, exp(t_vals) (log probabilities at this temperature) and the
    mass they leave as one more class.  t_ids is int32 [N][K] with -1 as
    padding, t_vals float32 [N][K]; either of loss and dlogits may be None.
    See tl_distill_topk in tinylm_cuda.h.
    """
    _sizes(N, V, K)
    z, ld = _rows(logits, "logits", N, V)
    dz, ldd = (None, 0) if dlogits is None else _rows(dlogits, "dlogits", N, V)
    if dlogits is not None and dlogits.dtype != logits.dtype:
        raise TypeError(f"dlogits: expected {logits.dtype}, got {dlogits.dtype}")
    _call_on(logits, "tl_distill_topk", z, _ROW_DTYPES[logits.dtype], ld,
             _vec(t_ids, "t_ids", N * K, torch.int32), _vec(t_vals, "t_vals", N * K), K, N, V, temperature, int(tail),
             _vec(weight, "weight", N), scale, _vec(loss, "loss", N), dz, ldd)


def sync():
    check(lib().tl_sync())
