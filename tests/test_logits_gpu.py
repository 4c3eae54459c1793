"""Vocabulary-row operators on the GPU (token log probabilities, their
gradient, top-K distillation) against the 64-bit formulas of logits_ref.py, at
the sizes, strides and masks where they can go wrong."""
import numpy as np
import pytest
import torch

import logits_ref as ref
from tinylm_c_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def make(rng, N, V, dtype, pad=0, offset=0, std=3.0, dev="cuda"):
    """Logits [N, V] with row stride V+pad, starting `offset` elements into a buffer whose other
    elements hold a canary."""
    flat = torch.full((offset + N * (V + pad) + 9,), 77.0, dtype=DT[dtype], device=dev)
    z = flat[offset:offset + N * (V + pad)].view(N, V + pad)[:, :V]
    x = rng.standard_normal((N, V)) * std
    x[np.arange(N), rng.integers(0, V, N)] += 6.0
    z.copy_(torch.from_numpy(x))
    return z, flat


def f64(t):
    return t.detach().double().cpu().numpy()


def run_score(z, ids, K, tau, want_entropy=True):
    N, V = z.shape
    dev = z.device
    logp = torch.full((N + 1,), -5.0, device=dev)
    H = torch.full((N + 1,), -5.0, device=dev) if want_entropy else None
    stats = torch.full((N + 1, 2), -5.0, device=dev)
    ti = torch.full((N + 1, K), -7, dtype=torch.int32, device=dev) if K else None
    tl = torch.full((N + 1, K), -5.0, device=dev) if K else None
    ops.token_logprobs(z, ids, N, V, logp, entropy=H, stats=stats, K=K, top_ids=ti, top_logp=tl, temperature=tau)
    torch.cuda.synchronize()
    # rows behind the last are left as they were
    assert logp[N] == -5.0 and (stats[N] == -5.0).all() and (H is None or H[N] == -5.0)
    assert ti is None or ((ti[N] == -7).all() and (tl[N] == -5.0).all())
    cut = lambda t: None if t is None else t[:N]  # noqa: E731
    return cut(logp), cut(H), cut(stats), cut(ti), cut(tl)


def check_score(z, ids, K, tau):
    zz, ii = f64(z), ids.cpu().numpy()
    want = ref.score(zz, ii, tau, K)
    for ent in (True, False):
        logp, H, stats, ti, tl = run_score(z, ids, K, tau, ent)
        ref.close(logp.cpu(), want["logp"], want["logp_tol"], "logp")
        if ent:
            ref.close(H.cpu(), want["entropy"], want["entropy_tol"], "entropy")
        if K:
            assert np.array_equal(ti.cpu().numpy(), want["top_ids"]), "top_ids"
            ref.close(tl.cpu(), want["top_logp"], want["top_logp_tol"], "top_logp")


def random_ids(rng, N, V, dev="cuda"):
    ids = rng.integers(0, V, N).astype(np.int32)
    ids[rng.random(N) < 0.2] = -1
    return torch.from_numpy(ids).to(dev)


SIZES = [  # N, V, pad, offset, K
    (1, 1, 0, 0, 1), (3, 2, 0, 1, 2), (2, 7, 3, 0, 7), (5, 31, 0, 3, 4), (4, 64, 0, 0, 64), (3, 127, 1, 0, 33),
    (5, 128, 0, 0, 128), (2, 129, 0, 5, 128), (7, 511, 0, 0, 16), (9, 512, 0, 0, 8), (3, 1000, 24, 0, 100),
    (2, 1024, 0, 0, 17), (3, 1025, 0, 0, 32), (2, 2047, 1, 0, 64), (4, 2048, 0, 0, 5), (3, 4095, 0, 2, 128),
    (2, 4097, 0, 0, 1), (2, 8192, 0, 0, 64), (3, 8193, 0, 1, 20), (2, 16384, 0, 0, 128), (1, 16391, 0, 0, 7),
    (2, 32768, 8, 0, 50), (2, 50001, 0, 0, 32), (1, 65537, 0, 3, 128), (1, 131072, 0, 0, 20), (2, 131073, 5, 0, 64),
    (1, 262144, 0, 0, 128), (1, 262143, 0, 1, 3),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,V,pad,offset,K", SIZES)
def test_score_matches_formula(cuda, dtype, N, V, pad, offset, K):
    rng = np.random.default_rng(V * 7 + N)
    z, flat = make(rng, N, V, dtype, pad, offset)
    before = flat.clone()
    check_score(z, random_ids(rng, N, V), K, [1.0, 0.5, 2.0][V % 3])
    assert torch.equal(flat, before)
    assert _lib.lib().tl_device_status() == _lib.TL_OK


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("N", [1, 2, 5, 17, 64, 149, 300, 1200])
def test_score_row_counts(cuda, dtype, N):
    """Few rows (split over several blocks) and many."""
    rng = np.random.default_rng(N)
    z, _ = make(rng, N, 4100, dtype)
    check_score(z, random_ids(rng, N, 4100), 9, 1.0)


PATTERNS = ["constant", "ascending", "descending", "two_values", "lowest_mask", "all_lowest", "inf_mask", "empty",
            "one_allowed", "zeros_signed", "huge", "spike", "block_high", "mass_ties"]


def pattern(name, rng, V, dtype):
    lowest = float(torch.finfo(DT[dtype]).min)
    x = rng.standard_normal(V) * 2
    some = rng.choice(V, max(1, min(V // 3, 11)), replace=False)
    if name == "constant":
        x[:] = 1.5
    elif name == "ascending":
        x = np.linspace(-8, 8, V)
    elif name == "descending":
        x = np.linspace(8, -8, V)
    elif name == "two_values":
        x = np.where(rng.random(V) < 0.5, 1.0, 1.5)
    elif name == "lowest_mask":            # a mask by the type's lowest value, a few tokens allowed
        y = np.full(V, lowest)
        y[some] = x[some]
        x = y
    elif name == "all_lowest":             # nothing allowed: uniform
        x[:] = lowest
    elif name == "inf_mask":
        y = np.full(V, -np.inf)
        y[some] = x[some]
        x = y
    elif name == "empty":
        x[:] = -np.inf
    elif name == "one_allowed":
        x[:] = -np.inf
        x[V - 1] = -3.0
    elif name == "zeros_signed":           # -0 and +0 are equal: the lower index wins
        x = np.where(rng.random(V) < 0.5, 0.0, -0.0)
    elif name == "huge":
        x = x * 1000 + 20000
    elif name == "spike":
        x[V // 2] = 60.0
    elif name == "block_high":             # all large values side by side
        x[V // 3:V // 3 + max(1, V // 4)] += 20
    elif name == "mass_ties":              # many values equal to the K-th largest
        x = np.floor(x * 2) / 2
    return x


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [5, 200, 1030, 5000, 40000, 131080])
def test_score_masks_ties_and_extremes(cuda, dtype, V):
    rng = np.random.default_rng(V)
    z, _ = make(rng, len(PATTERNS), V, dtype)
    for i, name in enumerate(PATTERNS):
        z[i].copy_(torch.from_numpy(pattern(name, rng, V, dtype)))
    ids = torch.from_numpy(rng.integers(0, V, len(PATTERNS)).astype(np.int32)).cuda()
    ids[PATTERNS.index("one_allowed")] = V - 1
    for K in sorted({min(k, V) for k in (1, 20, 128)}):
        check_score(z, ids, K, 1.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [3, 700, 9000, 140000])
def test_nan_and_inf_rows(cuda, dtype, V):
    """A NaN or +inf anywhere makes the row's results NaN and its alternatives -1, other rows are untouched."""
    rng = np.random.default_rng(V)
    z, _ = make(rng, 6, V, dtype)
    z[0, V - 1] = float("nan")
    z[1, 0] = float("inf")
    z[2, :] = float("nan")
    z[3, :] = float("-inf")
    z[3, V // 2] = float("nan")
    z[4, 0], z[4, V - 1] = float("inf"), float("inf")
    ids = torch.tensor([0, V - 1, 1, 0, -1, 2], dtype=torch.int32, device="cuda")
    check_score(z, ids, min(V, 12), 1.0)


def test_ids_outside_are_reported(cuda):
    z, _ = make(np.random.default_rng(0), 3, 100, "f32")
    ids = torch.tensor([4, 100, -2], dtype=torch.int32, device="cuda")
    logp, *_ = run_score(z, ids, 0, 1.0)
    assert logp[1] == 0.0 and logp[2] == 0.0 and logp[0] < 0.0
    assert _lib.lib().tl_device_status() == _lib.TL_EINVAL
    assert _lib.lib().tl_device_status() == _lib.TL_OK
    t_ids = torch.tensor([[4, 100], [-5, 3], [1, 2]], dtype=torch.int32, device="cuda")
    t_vals = torch.zeros(3, 2, device="cuda")
    loss, dz = torch.empty(3, device="cuda"), torch.empty_like(z)
    ops.distill_topk(z, t_ids, t_vals, 3, 100, 2, loss, dz)
    assert _lib.lib().tl_device_status() == _lib.TL_EINVAL
    L, lt, d, dt = ref.distill(f64(z), t_ids.cpu().numpy(), t_vals.cpu().numpy(), 1.0, False, None, 1.0, "f32")
    ref.close(loss.cpu(), L, lt, "loss")
    ref.close(dz.cpu(), d, dt, "dlogits")


# ------------------------------------------------------------------ gradient
def scored(z, ids, tau):
    N, V = z.shape
    logp, H, stats = torch.empty(N, device="cuda"), torch.empty(N, device="cuda"), torch.empty(N, 2, device="cuda")
    ops.token_logprobs(z, ids, N, V, logp, entropy=H, stats=stats, temperature=tau)
    return H, stats


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,V,pad,offset,K", SIZES)
@pytest.mark.parametrize("which", ["both", "logp", "entropy"])
def test_score_grad_matches_formula(cuda, dtype, N, V, pad, offset, K, which):
    rng = np.random.default_rng(V * 3 + N)
    z, flat = make(rng, N, V, dtype, pad, offset)
    ids = random_ids(rng, N, V)
    tau = [1.0, 0.5, 2.0][V % 3]
    H, stats = scored(z, ids, tau)
    a = torch.from_numpy(rng.standard_normal(N).astype(np.float32)).cuda() if which != "entropy" else None
    b = torch.from_numpy(rng.standard_normal(N).astype(np.float32)).cuda() if which != "logp" else None
    want, tol = ref.score_grad(f64(z), ids.cpu().numpy(), tau, None if a is None else f64(a),
                               None if b is None else f64(b), dtype)
    for opad, ooff in ((pad, offset), (0, 0), (3, 1)):        # the same alignment as the logits, and others
        dz, dflat = make(rng, N, V, dtype, opad, ooff)
        keep = dflat.clone()
        ops.token_logprobs_bwd(dz, z, ids if a is not None else None, N, V, stats, a,
                               entropy=H if b is not None else None, dentropy=b, temperature=tau)
        torch.cuda.synchronize()
        ref.close(dz.cpu().double(), want, tol, f"dlogits {opad} {ooff}")
        keep[ooff:ooff + N * (V + opad)].view(N, V + opad)[:, :V] = dz
        assert torch.equal(dflat, keep)                        # nothing beside the rows was written
    ops.token_logprobs_bwd(z, z, ids if a is not None else None, N, V, stats, a,
                           entropy=H if b is not None else None, dentropy=b, temperature=tau)
    ref.close(z.cpu().double(), want, tol, "dlogits in place")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [5, 200, 5000, 131080])
def test_score_grad_masks_and_extremes(cuda, dtype, V):
    rng = np.random.default_rng(V + 1)
    rows = PATTERNS + ["nan", "unread"]
    N = len(rows)
    z, _ = make(rng, N, V, dtype)
    for i, name in enumerate(PATTERNS):
        z[i].copy_(torch.from_numpy(pattern(name, rng, V, dtype)))
    z[N - 2:, V // 2] = float("nan")
    ids = torch.from_numpy(rng.integers(0, V, N).astype(np.int32)).cuda()
    H, stats = scored(z, ids, 1.0)
    a = rng.standard_normal(N).astype(np.float32)
    b = rng.standard_normal(N).astype(np.float32)
    a[N - 1] = b[N - 1] = 0.0                                  # nothing comes back: zeros despite the NaN
    want, tol = ref.score_grad(f64(z), ids.cpu().numpy(), 1.0, a, b, dtype)
    dz = torch.empty_like(z)
    ops.token_logprobs_bwd(dz, z, ids, N, V, stats, torch.from_numpy(a).cuda(), entropy=H,
                           dentropy=torch.from_numpy(b).cuda())
    ref.close(dz.cpu().double(), want, tol, "dlogits")


def test_score_grad_matches_differences(cuda):
    """Central differences of the operator's own sums along random directions.  With step h the
    difference quotient is off by h^2/6 times a third derivative (at most 6 per unit of sum |a|+|b|
    (1+H) for |direction| <= 1) and by the results' rounding over h."""
    rng = np.random.default_rng(11)
    N, V, h = 6, 777, 2.0 ** -5
    z, _ = make(rng, N, V, "f32")
    ids = random_ids(rng, N, V)
    a, b = (torch.from_numpy(rng.standard_normal(N).astype(np.float32)).cuda() for _ in range(2))
    H, stats = scored(z, ids, 1.0)
    dz = torch.empty_like(z)
    ops.token_logprobs_bwd(dz, z, ids, N, V, stats, a, entropy=H, dentropy=b)

    def total(x):
        logp, ent = torch.empty(N, device="cuda"), torch.empty(N, device="cuda")
        ops.token_logprobs(x, ids, N, V, logp, entropy=ent)
        return float((a.double() * logp.double() + b.double() * ent.double()).sum())

    size = float((a.abs() + b.abs() * (1 + H)).sum())
    tol = size * (6 * h * h / 6 + 2 * ref.entropy_bound(V) / (2 * h))
    for _ in range(4):
        u = torch.from_numpy(rng.uniform(-1, 1, (N, V)).astype(np.float32)).cuda()
        got = float((dz.double() * u.double()).sum())
        diff = (total(z + h * u) - total(z - h * u)) / (2 * h)
        assert abs(got - diff) <= tol, (got, diff, tol)


# -------------------------------------------------------------- distillation
def teacher(rng, z, K, tau, tail):
    """A teacher near the student: its K largest logits or log probabilities, some rows padded."""
    N, V = z.shape
    t = f64(z) + rng.standard_normal((N, V))
    ids = np.argsort(-t, axis=1, kind="stable")[:, :K].astype(np.int32)
    vals = np.take_along_axis(t, ids, 1)
    if tail:
        m = t.max(1, keepdims=True)
        vals = (vals - m) / tau - np.log(np.exp((t - m) / tau).sum(1, keepdims=True))
    if N > 2 and K > 1:
        ids[1, K // 2:] = -1
        ids[2, ::2] = -1
    return ids, vals.astype(np.float32)


def run_distill(z, ids, vals, tau, tail, w, scale, dz):
    N, V = z.shape
    K = ids.shape[1]
    loss = torch.full((N + 1,), -5.0, device="cuda")
    ops.distill_topk(z, torch.from_numpy(ids).cuda(), torch.from_numpy(vals).cuda(), N, V, K, loss, dz,
                     weight=None if w is None else torch.from_numpy(w).cuda(), scale=scale, temperature=tau,
                     tail=tail)
    torch.cuda.synchronize()
    assert loss[N] == -5.0
    return loss[:N]


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,V,pad,offset,K", SIZES)
def test_distill_matches_formula(cuda, dtype, N, V, pad, offset, K, tail):
    rng = np.random.default_rng(V * 5 + N)
    z, flat = make(rng, N, V, dtype, pad, offset)
    tau = [1.0, 0.5, 2.0][V % 3]
    ids, vals = teacher(rng, z, K, tau, tail)
    w = None
    if N > 3:
        w = rng.uniform(0.5, 1.5, N).astype(np.float32)
        w[3] = 0.0
    scale = 0.25
    L, lt, d, dt = ref.distill(f64(z), ids, vals, tau, tail, w, scale, dtype)
    for opad, ooff in ((pad, offset), (0, 0), (3, 1)):
        dz, dflat = make(rng, N, V, dtype, opad, ooff)
        keep = dflat.clone()
        loss = run_distill(z, ids, vals, tau, tail, w, scale, dz)
        ref.close(loss.cpu(), L, lt, "loss")
        ref.close(dz.cpu().double(), d, dt, f"dlogits {opad} {ooff}")
        keep[ooff:ooff + N * (V + opad)].view(N, V + opad)[:, :V] = dz
        assert torch.equal(dflat, keep)
    alone = run_distill(z, ids, vals, tau, tail, w, scale, None)
    assert torch.equal(alone, loss)                            # the loss alone: the same bits
    loss = run_distill(z, ids, vals, tau, tail, w, scale, z)
    ref.close(loss.cpu(), L, lt, "loss in place")
    ref.close(z.cpu().double(), d, dt, "dlogits in place")


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [40, 3000, 70000])
def test_distill_odd_teachers_and_students(cuda, dtype, V, tail):
    """Repeated tokens, rows of padding, tokens of probability 0 on either side, a confident
    student, masked students, a NaN."""
    rng = np.random.default_rng(V)
    K, N = 12, 15
    z, _ = make(rng, N, V, dtype)
    ids, vals = teacher(rng, z, K, 1.0, tail)
    ids[0, 5] = ids[0, 2]                  # one token named three times
    ids[0, 9] = ids[0, 2]
    if tail:
        vals[0] -= np.float32(np.log(3.0))
    ids[3] = -1                            # no teacher tokens
    vals[4, 1:] = -np.inf                  # one token only
    vals[5] = -np.inf
    z[6, int(ids[6, 0])] = float("-inf")   # the student rules out what the teacher names: loss +inf
    z[7, :] = float("-inf")                # a student that allows nothing
    z[8, :] = float(torch.finfo(DT[dtype]).min)
    z[9, int(ids[9, 0])] = 80.0            # almost no mass left for the rest
    z[10, V - 1] = float("nan")
    vals[11, 0] = np.nan
    ids[11, 0] = 0
    keep = set(ids[12].tolist())           # the student allows exactly what the teacher names
    for v in range(V):
        if v not in keep:
            z[12, v] = float("-inf")
    ids[13, :] = np.arange(K)              # in index order, at the row's start
    vals[14, K - 1] = np.inf
    w = np.ones(N, np.float32)
    L, lt, d, dt = ref.distill(f64(z), ids, vals, 1.0, tail, w, 1.0, dtype)
    dz = torch.empty_like(z)
    loss = run_distill(z, ids, vals, 1.0, tail, w, 1.0, dz)
    ref.close(loss.cpu(), L, lt, "loss")
    ref.close(dz.cpu().double(), d, dt, "dlogits")
    w[6:12] = 0.0                          # rows that do not count are not read
    L, lt, d, dt = ref.distill(f64(z), ids, vals, 1.0, tail, w, 1.0, dtype)
    loss = run_distill(z, ids, vals, 1.0, tail, w, 1.0, dz)
    ref.close(loss.cpu(), L, lt, "loss")
    ref.close(dz.cpu().double(), d, dt, "dlogits")
    assert (dz[6:12] == 0).all() and (loss[6:12] == 0).all()


@pytest.mark.parametrize("dtype,N,V,K", [("bf16", 4, 20010, 88), ("f16", 3, 963, 113), ("f32", 200, 9000, 60)])
def test_distill_close_student(cuda, dtype, N, V, K):
    """A loss of a few hundredths, a difference of terms of log V = 7 to 10 whose fp32 rounding alone is
    2^-21 to 2^-22 each.  From fp32 sums whose terms' errors have independent signs (a few u of 2^-24
    on sums of up to V terms) 16 u = 1e-6 is left for a row's loss."""
    rng = np.random.default_rng(V)
    z, _ = make(rng, N, V, dtype)
    ids, vals = teacher(rng, z, K, 2.0, True)
    L, _, _, _ = ref.distill(f64(z), ids, vals, 2.0, True, None, 1.0, dtype)
    loss = run_distill(z, ids, vals, 2.0, True, None, 1.0, torch.empty_like(z))
    assert 1e-3 < np.median(L) < 0.2
    ref.close(loss.cpu(), L, 16 * ref.U, "loss")


@pytest.mark.parametrize("tail", [False, True])
def test_distill_whole_vocabulary(cuda, tail):
    """A teacher that names every token leaves no tail."""
    rng = np.random.default_rng(3)
    N, V = 5, 100
    z, _ = make(rng, N, V, "f32")
    t = rng.standard_normal((N, V)) * 2
    vals = (t - np.log(np.exp(t).sum(1, keepdims=True))).astype(np.float32)
    ids = np.stack([rng.permutation(V) for _ in range(N)]).astype(np.int32)
    L, lt, d, dt = ref.distill(f64(z), ids, vals, 1.0, tail, None, 1.0, "f32")
    dz = torch.empty_like(z)
    loss = run_distill(z, ids, vals, 1.0, tail, None, 1.0, dz)
    assert torch.isfinite(loss).all()
    ref.close(loss.cpu(), L, lt, "loss")
    ref.close(dz.cpu().double(), d, dt, "dlogits")


@pytest.mark.parametrize("tail", [False, True])
def test_distill_gradient_matches_differences(cuda, tail):
    """Central differences of the operator's own loss, as above: the loss is sum q (-log p) and
    log-sum-exp terms, third derivatives at most 6 a row for |direction| <= 1."""
    rng = np.random.default_rng(12)
    N, V, K, h = 5, 900, 10, 2.0 ** -5
    z, _ = make(rng, N, V, "f32")
    ids, vals = teacher(rng, z, K, 1.0, tail)
    dz = torch.empty_like(z)
    run_distill(z, ids, vals, 1.0, tail, None, 1.0, dz)
    tol = N * (6 * h * h / 6) * 2 + N * 2 * (ref.entropy_bound(V) + 1e-5) / (2 * h)
    for _ in range(4):
        u = torch.from_numpy(rng.uniform(-1, 1, (N, V)).astype(np.float32)).cuda()
        got = float((dz.double() * u.double()).sum())
        up = run_distill(z + h * u, ids, vals, 1.0, tail, None, 1.0, None).double().sum()
        down = run_distill(z - h * u, ids, vals, 1.0, tail, None, 1.0, None).double().sum()
        assert abs(got - float(up - down) / (2 * h)) <= tol


# ----------------------------------------------------------- used together
@pytest.mark.parametrize("dtype,V", [("f32", 2048), ("bf16", 50001)])
def test_teacher_scores_then_student_distils(cuda, dtype, V):
    """A teacher's alternatives go straight into the student's loss; a student equal to its teacher
    has none, and no gradient."""
    rng = np.random.default_rng(5)
    N, K, tau = 40, 24, 2.0
    z, _ = make(rng, N, V, dtype)
    zt, _ = make(rng, N, V, dtype)
    ids = random_ids(rng, N, V)
    logp, ti, tl = torch.empty(N, device="cuda"), torch.empty(N, K, dtype=torch.int32, device="cuda"), \
        torch.empty(N, K, device="cuda")
    ops.token_logprobs(zt, ids, N, V, logp, K=K, top_ids=ti, top_logp=tl, temperature=tau)
    loss, dz = torch.empty(N, device="cuda"), torch.empty_like(z)
    ops.distill_topk(z, ti, tl, N, V, K, loss, dz, scale=1.0 / N, temperature=tau, tail=True)
    L, lt, d, dt = ref.distill(f64(z), ti.cpu().numpy(), tl.cpu().numpy(), tau, True, None, 1.0 / N, dtype)
    ref.close(loss.cpu(), L, lt, "loss")
    ref.close(dz.cpu().double(), d, dt, "dlogits")
    ops.distill_topk(zt, ti, tl, N, V, K, loss, dz, temperature=tau, tail=True)
    L, lt, d, dt = ref.distill(f64(zt), ti.cpu().numpy(), tl.cpu().numpy(), tau, True, None, 1.0, dtype)
    ref.close(loss.cpu(), L, lt, "loss of the teacher itself")
    ref.close(dz.cpu().double(), d, dt, "gradient of the teacher itself")
    assert float(np.abs(L).max()) < 1e-6   # the formula's own value: rounding of fp32 log probabilities


def everything(z, ids, t_ids, t_vals, out):
    N, V = z.shape
    ops.token_logprobs(z, ids, N, V, out["logp"], entropy=out["H"], stats=out["stats"], K=7, top_ids=out["ti"],
                       top_logp=out["tl"])
    ops.token_logprobs_bwd(out["d1"], z, ids, N, V, out["stats"], out["logp"], entropy=out["H"], dentropy=out["H"])
    ops.distill_topk(z, t_ids, t_vals, N, V, t_ids.shape[1], out["loss"], out["d2"], tail=True)


def outputs(z):
    N = z.shape[0]
    new = lambda *s, **k: torch.zeros(*s, device="cuda", **k)  # noqa: E731
    return {"logp": new(N), "H": new(N), "stats": new(N, 2), "ti": new(N, 7, dtype=torch.int32), "tl": new(N, 7),
            "d1": torch.zeros_like(z), "loss": new(N), "d2": torch.zeros_like(z)}


@pytest.mark.parametrize("N,V", [(3, 1000), (2, 100000), (500, 8192)])
def test_same_bits_twice_captured_and_on_two_streams(cuda, N, V):
    """Eager twice, replayed from two CUDA graphs over new inputs, and on two streams at once: the
    same bits every time."""
    rng = np.random.default_rng(N)
    zs = [make(rng, N, V, "f32")[0].clone() for _ in range(2)]
    ids = random_ids(rng, N, V)
    tch = [teacher(rng, z, 9, 1.0, True) for z in zs]
    tch = [(torch.from_numpy(i).cuda(), torch.from_numpy(v).cuda()) for i, v in tch]
    want = []
    for z, (ti, tv) in zip(zs, tch):
        a, b = outputs(z), outputs(z)
        everything(z, ids, ti, tv, a)
        everything(z, ids, ti, tv, b)
        torch.cuda.synchronize()
        assert all(torch.equal(a[k], b[k]) for k in a)
        want.append(a)
    # two streams
    streams = [torch.cuda.Stream() for _ in zs]
    got = [outputs(z) for z in zs]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, z, (ti, tv), o in zip(streams, zs, tch, got):
            with torch.cuda.stream(s):
                everything(z, ids, ti, tv, o)
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w[k], g[k]) for k in w)
    # captured
    buf_z, buf_i, buf_v = zs[0].clone(), tch[0][0].clone(), tch[0][1].clone()
    outs, graphs = [outputs(buf_z), outputs(buf_z)], []
    for o in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            everything(buf_z, ids, buf_i, buf_v, o)
        graphs.append(g)
    for w, z, (ti, tv) in zip(want, zs, tch):
        buf_z.copy_(z)
        buf_i.copy_(ti)
        buf_v.copy_(tv)
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(w[k], o[k]) for k in w)


@pytest.mark.parametrize("tau", [1e-6, 0.03, 50.0, 1e6])
def test_extreme_temperatures(cuda, tau):
    """Close to the largest logit alone, and close to uniform."""
    rng = np.random.default_rng(6)
    for N, V, dtype in ((4, 3000, "f32"), (2, 40000, "bf16")):
        z, _ = make(rng, N, V, dtype)
        ids = random_ids(rng, N, V)
        check_score(z, ids, 10, tau)
        H, stats = scored(z, ids, tau)
        a = torch.ones(N, device="cuda")
        want, tol = ref.score_grad(f64(z), ids.cpu().numpy(), tau, f64(a), None, dtype)
        dz = torch.empty_like(z)
        ops.token_logprobs_bwd(dz, z, ids, N, V, stats, a, temperature=tau)
        ref.close(dz.cpu().double(), want, tol, "dlogits")
        t_ids, t_vals = teacher(rng, z, 6, tau, False)
        L, lt, d, dt = ref.distill(f64(z), t_ids, t_vals, tau, False, None, tau, dtype)
        loss = run_distill(z, t_ids, t_vals, tau, False, None, tau, dz)
        ref.close(loss.cpu(), L, lt, "loss")
        ref.close(dz.cpu().double(), d, dt, "dlogits")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_rows_of_hard_patterns(cuda, dtype):
    """Rows that overflow the list of candidates beside rows that do not, many to a block, for every
    way the rows are laid out: short, one piece, several pieces."""
    rng = np.random.default_rng(8)
    for N, V, K in ((1500, 300, 12), (1300, 6000, 40), (700, 20000, 128), (400, 70000, 5)):
        z, _ = make(rng, N, V, dtype)
        names = ["constant", "ascending", "lowest_mask", "inf_mask", "empty", "mass_ties", "two_values"]
        rows = {name: torch.from_numpy(pattern(name, rng, V, dtype)).to(z) for name in names}
        some = rng.choice(N, 70, replace=False)
        for i, n in enumerate(some):
            z[n] = rows[names[i % len(names)]]
        ids = random_ids(rng, N, V)
        logp, H, stats, ti, tl = run_score(z, ids, K, 1.0)
        pick = np.concatenate([some, rng.choice(N, 40, replace=False)])
        at = torch.from_numpy(pick).cuda()
        want = ref.score(f64(z[at]), ids[at].cpu().numpy(), 1.0, K)
        ref.close(logp[at].cpu(), want["logp"], want["logp_tol"], "logp")
        ref.close(H[at].cpu(), want["entropy"], want["entropy_tol"], "entropy")
        assert np.array_equal(ti[at].cpu().numpy(), want["top_ids"])
        ref.close(tl[at].cpu(), want["top_logp"], want["top_logp_tol"], "top_logp")


@pytest.mark.parametrize("tail", [False, True])
def test_distill_many_rows(cuda, tail):
    """Many rows to a block, every third without weight, in one piece and in several, in place."""
    rng = np.random.default_rng(13)
    for N, V, K, dtype, pad in ((1400, 700, 5, "f32", 1), (1200, 8192, 20, "f32", 0), (500, 50001, 9, "bf16", 0),
                                (460, 120000, 6, "bf16", 8)):
        z, flat = make(rng, N, V, dtype, pad)
        pick = np.sort(rng.choice(N, 30, replace=False))
        at = torch.from_numpy(pick).cuda()
        t = z.float() + torch.randn(N, V, device="cuda")
        vals, ids = torch.topk(t, K, dim=1)
        if tail:
            vals = torch.log_softmax(t, 1).gather(1, ids)
        ids, vals = ids.int().contiguous(), vals.contiguous()
        w = torch.rand(N, device="cuda") + 0.5
        w[::3] = 0.0
        L, lt, d, dt = ref.distill(f64(z[at]), ids[at].cpu().numpy(), vals[at].cpu().numpy(), 1.0, tail, f64(w[at]), 2.0,
                                   dtype)
        loss = torch.empty(N, device="cuda")
        dz = torch.full_like(z, 5.0)
        ops.distill_topk(z, ids, vals, N, V, K, loss, dz, weight=w, scale=2.0, tail=tail)
        ref.close(loss[at].cpu(), L, lt, "loss")
        ref.close(dz[at].cpu().double(), d, dt, "dlogits")
        assert (dz[::3] == 0).all() and (loss[::3] == 0).all()
        again = torch.empty(N, device="cuda")
        keep = flat.clone()
        ops.distill_topk(z, ids, vals, N, V, K, again, z, weight=w, scale=2.0, tail=tail)
        assert torch.equal(again, loss) and torch.equal(z, dz)
        keep[:N * (V + pad)].view(N, V + pad)[:, :V] = z
        assert torch.equal(flat, keep)


def test_first_call_inside_a_capture():
    """In a fresh process, after ops.init, the first call of each operator is captured."""
    import subprocess
    import sys
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device visible")
    code = """
import torch
from tinylm_c_b200 import ops
ops.init(0)
for N, V in ((3, 900), (2, 70000), (300, 9000)):
    z = torch.randn(N, V, device="cuda"); ids = torch.zeros(N, dtype=torch.int32, device="cuda")
    lp, H, st = torch.zeros(N, device="cuda"), torch.zeros(N, device="cuda"), torch.zeros(N, 2, device="cuda")
    ti, tl = torch.zeros(N, 4, dtype=torch.int32, device="cuda"), torch.zeros(N, 4, device="cuda")
    dz, L = torch.zeros_like(z), torch.zeros(N, device="cuda")
    def go():
        ops.token_logprobs(z, ids, N, V, lp, entropy=H, stats=st, K=4, top_ids=ti, top_logp=tl)
        ops.distill_topk(z, ti, tl, N, V, 4, L, dz, tail=True)
        ops.token_logprobs_bwd(dz, z, ids, N, V, st, lp, entropy=H, dentropy=H)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        go()
    g.replay(); torch.cuda.synchronize()
    got = [t.clone() for t in (lp, H, ti, tl, L, dz)]
    for t in (lp, H, ti, tl, L, dz): t.zero_()
    go(); torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, (lp, H, ti, tl, L, dz)))
    assert torch.allclose(lp, torch.log_softmax(z, 1)[:, 0], atol=1e-4)
print("captured")
"""
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_offsets_past_32_bits(cuda):
    """Rows that start more than 2^32 bytes and 2^31 elements into the logits."""
    N, V, pad = 3, 5000, (1 << 30) + 1001
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free device memory")
    rng = np.random.default_rng(9)
    flat = torch.empty(2 * (V + pad) + V, dtype=torch.bfloat16, device="cuda")
    z = torch.as_strided(flat, (N, V), (V + pad, 1))
    z.copy_(torch.from_numpy(rng.standard_normal((N, V)) * 3))
    ids = torch.tensor([1, 2, 4999], dtype=torch.int32, device="cuda")
    check_score(z, ids, 20, 1.0)
    dflat = torch.empty_like(flat)
    dz = torch.as_strided(dflat, (N, V), (V + pad, 1))
    H, stats = scored(z, ids, 1.0)
    a = torch.ones(N, device="cuda")
    want, tol = ref.score_grad(f64(z), ids.cpu().numpy(), 1.0, f64(a), None, "bf16")
    ops.token_logprobs_bwd(dz, z, ids, N, V, stats, a)
    ref.close(dz.cpu().double(), want, tol, "dlogits")
    t_ids, t_vals = teacher(rng, z, 6, 1.0, True)
    L, lt, d, dt = ref.distill(f64(z), t_ids, t_vals, 1.0, True, None, 1.0, "bf16")
    loss = run_distill(z, t_ids, t_vals, 1.0, True, None, 1.0, dz)
    ref.close(loss.cpu(), L, lt, "loss")
    ref.close(dz.cpu().double(), d, dt, "dlogits")


def test_no_rows(cuda):
    z = torch.empty(0, 50, device="cuda")
    e = torch.empty(0, device="cuda")
    i = torch.empty(0, dtype=torch.int32, device="cuda")
    ops.token_logprobs(z, i, 0, 50, e, entropy=e, K=3, top_ids=i, top_logp=e)
    ops.token_logprobs_bwd(z, z, i, 0, 50, e, e, entropy=e, dentropy=e)
    ops.distill_topk(z, i, e, 0, 50, 3, e, z)
    torch.cuda.synchronize()


def test_refusals_on_the_device(cuda):
    """Host memory, overlap and misalignment are refused before any launch (the argument checks that
    need no device are in test_logits_cpu.py)."""
    L = _lib.lib()
    z = torch.randn(4, 64, device="cuda")
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    out, stats = torch.empty(4, device="cuda"), torch.zeros(4, 2, device="cuda")
    host = torch.randn(4, 64)
    ops.init(0)
    def score(zp, ip, op):
        return L.tl_token_logprobs(zp, 0, 64, ip, 4, 64, 1.0, op, None, None, 0, None, None)

    assert score(host.data_ptr(), ids.data_ptr(), out.data_ptr()) == _lib.TL_EPTR
    assert score(z.data_ptr(), host.data_ptr(), out.data_ptr()) == _lib.TL_EPTR
    assert score(z.data_ptr(), ids.data_ptr(), host.data_ptr()) == _lib.TL_EPTR
    assert score(z.data_ptr() + 2, ids.data_ptr(), out.data_ptr()) == _lib.TL_EALIGN
    assert score(None, ids.data_ptr(), out.data_ptr()) == _lib.TL_EINVAL
    # dlogits shifted into the logits' rows
    flat = torch.randn(4 * 64 + 64, device="cuda")
    z1, z2 = flat[:256].view(4, 64), flat[16:272].view(4, 64)
    with pytest.raises(_lib.TLError) as e:
        ops.token_logprobs_bwd(z2, z1, ids, 4, 64, stats, out)
    assert e.value.code == _lib.TL_EINVAL
    with pytest.raises(_lib.TLError):
        ops.distill_topk(z1, ids, out, 4, 64, 1, out, z2)
    with pytest.raises(_lib.TLError):                          # half of each row, another stride
        ops.distill_topk(flat[:256].view(2, 128)[:, :64], ids, out, 2, 64, 1, out, flat[:128].view(2, 64))
