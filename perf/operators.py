"""Workloads of the vocabulary-row operators: scoring given tokens and distilling a teacher.

Three operators over rows of logits [N, V] (fp32, bf16 or fp16, any row stride):

    score         log probability of one given token a row, the row's entropy and its K most
                  likely tokens                                            ops.token_logprobs
    score_grad    gradient of those log probabilities and entropies         ops.token_logprobs_bwd
    distill       KL divergence from a teacher's K most likely tokens, and its gradient in the
                  student's logits                                          ops.distill_topk

Each case runs in a plain form of elementary torch operations in 32 bits, or through the library
when `own` is true.  Definitions, shared by every form here:

    y = z / temperature, log p_v = y_v - log sum_u exp(y_u), H = -sum_v p_v log p_v
    a given token of -1 has no log probability: 0, and no gradient
    a row of -inf only has log p = -inf and H = 0, and no gradient
    the K most likely tokens: larger logit first, the lower index first among equal ones; a token
    of logit -inf is none: index -1, log probability -inf in its place
    distill: entries of index -1 are padding.  q is the softmax of the teacher's values over
    temperature (tail false), or exp of its log probabilities with the mass they leave as one
    more class, the tail (tail true; a tail below 2^-20 is 0).  A row's loss is its weight times
    sum q log(q / p), the tail's p being that of all tokens the teacher did not name; gradients
    are those of scale times the sum of the rows' losses.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TAIL_MIN = 2.0 ** -20


def listed():
    return [
        # one generated token with its 5 alternatives: the answer of a single request, all latency
        {"name": "score_one_token", "op": "score", "dtype": "f32", "N": 1, "V": 8192, "K": 5, "entropy": True,
         "temperature": 1.0, "pad": 0, "masked": 0.0},
        # one step of 16 sequences over a large vocabulary, half of them held to an allowed list of tokens
        {"name": "score_step_131k_bf16", "op": "score", "dtype": "bf16", "N": 16, "V": 131072, "K": 20,
         "entropy": True, "temperature": 0.7, "pad": 0, "masked": 0.5},
        # validation log-likelihoods and entropies of two windows of the nano preset
        {"name": "score_nano", "op": "score", "dtype": "f32", "N": 512, "V": 512, "K": 0, "entropy": True,
         "temperature": 1.0, "pad": 0, "masked": 0.0},
        # the same for one micro-batch of 64 windows of the scaled preset
        {"name": "score_scaled", "op": "score", "dtype": "f32", "N": 16384, "V": 8192, "K": 0, "entropy": True,
         "temperature": 1.0, "pad": 0, "masked": 0.0},
        # a teacher of the scaled preset writing down its 64 most likely tokens for a student
        {"name": "teacher_scaled_k64", "op": "score", "dtype": "f32", "N": 16384, "V": 8192, "K": 64,
         "entropy": False, "temperature": 1.0, "pad": 0, "masked": 0.0},
        # a bf16 teacher with an odd vocabulary: every row starts at another alignment
        {"name": "teacher_50k_bf16", "op": "score", "dtype": "bf16", "N": 4095, "V": 50001, "K": 32,
         "entropy": True, "temperature": 2.0, "pad": 0, "masked": 0.05},
        # policy gradient with an entropy bonus on one micro-batch of the scaled preset
        {"name": "grad_scaled", "op": "score_grad", "dtype": "f32", "N": 16384, "V": 8192, "entropy": True,
         "temperature": 1.0, "pad": 0, "masked": 0.0},
        # the gradient of a likelihood alone over a large vocabulary in padded bf16 rows, an odd number of them
        {"name": "grad_131k_bf16", "op": "score_grad", "dtype": "bf16", "N": 1021, "V": 131072, "entropy": False,
         "temperature": 1.0, "pad": 64, "masked": 0.05},
        # distilling the nano preset on two windows, a softened teacher's 8 tokens
        {"name": "distill_nano_k8", "op": "distill", "dtype": "f32", "N": 512, "V": 512, "K": 8, "tail": False,
         "temperature": 2.0, "pad": 0, "weights": False},
        # distilling the scaled preset on one micro-batch, all of the teacher's mass kept
        {"name": "distill_scaled_k64", "op": "distill", "dtype": "f32", "N": 16384, "V": 8192, "K": 64, "tail": True,
         "temperature": 1.0, "pad": 0, "weights": False},
        # fp16 student, odd vocabulary and stride, padding tokens weighted 0
        {"name": "distill_50k_f16", "op": "distill", "dtype": "f16", "N": 2047, "V": 50001, "K": 100, "tail": False,
         "temperature": 2.0, "pad": 6, "weights": True},
        # bf16 student with a large vocabulary
        {"name": "distill_131k_bf16", "op": "distill", "dtype": "bf16", "N": 2048, "V": 131072, "K": 32, "tail": True,
         "temperature": 1.0, "pad": 0, "weights": True},
    ]


def draw(rng):
    op = rng.choice(["score", "score_grad", "distill"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    size = 4 if dtype == "f32" else 2
    V = int(round(math.exp(rng.uniform(math.log(130), math.log(131072)))))
    most = 1_000_000_000 // (V * size * (1 if op == "score" else 2))    # bytes of the largest listed case
    N = int(round(math.exp(rng.uniform(0.0, math.log(min(16384, most))))))
    case = {"op": op, "dtype": dtype, "N": N, "V": V, "temperature": rng.choice([0.5, 1.0, 1.0, 2.0]),
            "pad": rng.choice([0, 0, 1, 8, 37])}
    if op == "distill":
        case.update(K=int(round(math.exp(rng.uniform(0.0, math.log(128))))), tail=rng.random() < 0.5,
                    weights=rng.random() < 0.5)
    else:
        case.update(entropy=rng.random() < 0.6, masked=rng.choice([0.0, 0.0, 0.1, 0.5]))
    if op == "score":
        case["K"] = rng.choice([0, int(round(math.exp(rng.uniform(0.0, math.log(128)))))])
    return case


# ---------------------------------------------------------------- inputs
def _rows(gen, case):
    """Logits of a trained model's shape: a wide body and a few likely tokens a row."""
    N, V, dev = case["N"], case["V"], torch.device("cuda", 0)
    z = torch.empty(N, V + case["pad"], dtype=DTYPES[case["dtype"]], device=dev)
    for lo in range(0, N, 2048):                               # bounded temporaries
        hi = min(N, lo + 2048)
        x = torch.randn(hi - lo, V + case["pad"], generator=gen, device=dev).mul_(2.0)
        likely = torch.randint(0, V, (hi - lo, 4), generator=gen, device=dev)
        x.scatter_add_(1, likely, torch.rand(hi - lo, 4, generator=gen, device=dev).mul_(12.0))
        z[lo:hi] = x
    return z[:, :V]


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev).manual_seed(seed)
    N, V, tau = case["N"], case["V"], case["temperature"]
    s = {"case": case, "logits": _rows(gen, case)}
    unit = 4096.0 if case["dtype"] == "f16" else 1.0           # fp16 gradients are scaled up, as such training does
    new = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device=dev)  # noqa: E731
    if case["op"] == "distill":
        K = case["K"]
        t_ids, t_vals = [], []
        for lo in range(0, N, 2048):                           # a teacher near the student
            z = s["logits"][lo:lo + 2048].float()
            z = z + torch.randn(z.shape, generator=gen, device=dev)
            v, i = torch.topk(z, K, dim=1)
            if case["tail"]:
                v = v / tau - torch.logsumexp(z / tau, 1, keepdim=True)
            t_ids.append(i.int())
            t_vals.append(v)
        s["t_ids"], s["t_vals"] = torch.cat(t_ids), torch.cat(t_vals)
        if K > 1:                                              # some rows came with fewer tokens
            few = torch.rand(N, generator=gen, device=dev) < 0.05
            s["t_ids"][few, K // 2:] = -1
        s["weight"] = None
        if case["weights"]:
            s["weight"] = torch.rand(N, generator=gen, device=dev) + 0.5
            s["weight"][torch.rand(N, generator=gen, device=dev) < 0.1] = 0.0
        s["scale"] = unit / N
        s["loss"], s["dlogits"] = new(N), new(N, V + case["pad"], dtype=DTYPES[case["dtype"]])[:, :V]
        return s
    if case["masked"]:                                         # rows held to about 1 token in 50
        held = torch.rand(N, generator=gen, device=dev) < case["masked"]
        z = s["logits"][held]
        s["logits"][held] = z.masked_fill_(torch.rand(z.shape, generator=gen, device=dev) < 0.98, float("-inf"))
        s["logits"][held, V // 2] = 1.0
    s["ids"] = torch.randint(0, V, (N,), generator=gen, device=dev, dtype=torch.int32)
    if case["masked"]:
        s["ids"][held] = V // 2
    s["ids"][torch.rand(N, generator=gen, device=dev) < 0.05] = -1
    s["logp"], s["entropy"] = new(N), new(N) if case["entropy"] else None
    s["stats"] = new(N, 2)
    if case["op"] == "score":
        s["top_ids"] = new(N, case["K"], dtype=torch.int32) if case["K"] else None
        s["top_logp"] = new(N, case["K"]) if case["K"] else None
        return s
    s["dlogp"] = torch.randn(N, generator=gen, device=dev) * (unit / N)
    s["dentropy"] = torch.randn(N, generator=gen, device=dev) * (unit / N) if case["entropy"] else None
    s["dlogits"] = new(N, V + case["pad"], dtype=DTYPES[case["dtype"]])[:, :V]
    # what the forward pass left: each row's largest logit, the logarithm of its sum, its entropy
    z = s["logits"]
    for lo in range(0, N, 2048):
        zf = z[lo:lo + 2048].float()
        m = zf.amax(1, keepdim=True)
        y = (zf - m) / tau
        e = torch.exp(y)
        total = e.sum(1, keepdim=True)
        s["stats"][lo:lo + 2048, 0:1], s["stats"][lo:lo + 2048, 1:2] = m, total.log()
        if case["entropy"]:
            s["entropy"][lo:lo + 2048] = total.log()[:, 0] - (e * y.clamp(min=-1e30)).sum(1) / total[:, 0]
    return s


# ---------------------------------------------------------------- the plain form
def _log_softmax(z, tau):
    """log p of rows of 32-bit logits; a row of -inf only gives -inf."""
    m = z.amax(1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    y = (z - m) / tau
    return y - torch.exp(y).sum(1, keepdim=True).log()


def _top(z, logp, K):
    """The K largest logits a row, the lower index first among equal ones: one key a token, its
    logit's order above its index counted down."""
    V = z.shape[1]
    bits = (z + 0.0).view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()
    down = torch.arange(V - 1, -1, -1, device=z.device)
    ids = V - 1 - (torch.topk((order << 32) | down, K, dim=1).values & 0xFFFFFFFF)
    found = torch.gather(logp, 1, ids)
    none = torch.isinf(torch.gather(z, 1, ids))
    return torch.where(none, -1, ids).int(), torch.where(none, float("-inf"), found)


def _score(s):
    case, z = s["case"], s["logits"].float()
    logp = _log_softmax(z, case["temperature"])
    ids = s["ids"].long()
    of_ids = torch.gather(logp, 1, ids.clamp(min=0)[:, None])[:, 0]
    out = {"logp": torch.where(ids < 0, torch.zeros_like(of_ids), of_ids)}
    if case["entropy"]:
        out["entropy"] = -torch.where(torch.isinf(logp), torch.zeros_like(logp), torch.exp(logp) * logp).sum(1)
    if case["K"]:
        out["top_ids"], out["top_logp"] = _top(z, logp, case["K"])
    return out


def _score_grad(s):
    case, z = s["case"], s["logits"].float()
    logp = _log_softmax(z, case["temperature"])
    p = torch.exp(logp)
    ids = s["ids"].long()
    up = torch.where(ids < 0, torch.zeros_like(s["dlogp"]), s["dlogp"])[:, None]
    d = -p * up
    if case["entropy"]:
        plogp = torch.where(torch.isinf(logp), torch.zeros_like(logp), p * logp)
        d = d + s["dentropy"][:, None] * (p * plogp.sum(1, keepdim=True) - plogp)
    d.scatter_add_(1, ids.clamp(min=0)[:, None], up)
    return {"dlogits": (d / case["temperature"]).to(s["logits"].dtype)}


def _distill(s):
    case, z, tau = s["case"], s["logits"].float(), s["case"]["temperature"]
    logp = _log_softmax(z, tau)
    ids = s["t_ids"].long()
    named = ids >= 0
    t = torch.where(named, s["t_vals"], float("-inf"))
    if case["tail"]:
        q = torch.exp(t)
    else:
        q = torch.exp((t - t.amax(1, keepdim=True)) / tau)
        q = q / q.sum(1, keepdim=True)
    dense = torch.zeros_like(z).scatter_add_(1, ids.clamp(min=0), q)
    loss = torch.where(dense > 0, dense * (torch.log(dense) - logp), torch.zeros_like(z)).sum(1)
    total, p = q.sum(1), torch.exp(logp)
    d = -dense
    if case["tail"]:
        of_set = torch.zeros_like(z).scatter_add_(1, ids.clamp(min=0), named.float()) > 0
        rest = torch.where(of_set, torch.zeros_like(p), p)
        p_rest, q_rest = rest.sum(1), (1.0 - total).clamp(min=0)
        q_rest = torch.where(q_rest < TAIL_MIN, torch.zeros_like(q_rest), q_rest)
        has = q_rest > 0
        loss = loss + torch.where(has, q_rest * (torch.log(q_rest) - torch.log(p_rest)), torch.zeros_like(loss))
        total = total + q_rest
        d = d - rest * torch.where(has, q_rest / p_rest, torch.zeros_like(q_rest))[:, None]
    d = d + p * total[:, None]
    w = torch.ones_like(loss) if s["weight"] is None else s["weight"]
    return {"loss": w * loss, "dlogits": (d * (w * (s["scale"] / tau))[:, None]).to(s["logits"].dtype)}


def run(state):
    s, case = state, state["case"]
    N, V, tau = case["N"], case["V"], case["temperature"]
    if not own:
        return {"score": _score, "score_grad": _score_grad, "distill": _distill}[case["op"]](s)
    from tinylm_c_b200 import ops
    if case["op"] == "score":
        ops.token_logprobs(s["logits"], s["ids"], N, V, s["logp"], entropy=s["entropy"], K=case["K"],
                           top_ids=s["top_ids"], top_logp=s["top_logp"], temperature=tau)
        return {k: s[k] for k in ("logp", "entropy", "top_ids", "top_logp") if s[k] is not None}
    if case["op"] == "score_grad":
        ops.token_logprobs_bwd(s["dlogits"], s["logits"], s["ids"], N, V, s["stats"], s["dlogp"],
                               entropy=s["entropy"], dentropy=s["dentropy"], temperature=tau)
        return {"dlogits": s["dlogits"]}
    ops.distill_topk(s["logits"], s["t_ids"], s["t_vals"], N, V, case["K"], s["loss"], s["dlogits"],
                     weight=s["weight"], scale=s["scale"], temperature=tau, tail=case["tail"])
    return {"loss": s["loss"], "dlogits": s["dlogits"]}


# ---------------------------------------------------------------- sizes and the definition in 64 bits
def work(case):
    """Logits read once, results written once; an exponential, a logarithm or a comparison is one operation."""
    N, V, size = case["N"], case["V"], 4 if case["dtype"] == "f32" else 2
    if case["op"] == "score":
        per_row = 4 + 4 + (4 if case["entropy"] else 0) + 8 * case["K"]
        each = 5 + (2 if case["entropy"] else 0) + (1 if case["K"] else 0)
        return {"bytes": N * (V * size + per_row), "flops": N * V * each}
    if case["op"] == "score_grad":
        per_row = 4 + 8 + 4 + (8 if case["entropy"] else 0)
        return {"bytes": N * (2 * V * size + per_row), "flops": N * V * (5 + (3 if case["entropy"] else 0))}
    per_row = 8 * case["K"] + 4 + (4 if case["weights"] else 0)
    return {"bytes": N * (2 * V * size + per_row), "flops": N * V * 7 + N * case["K"] * 12}


def exact(case, seed):
    s = prepare(case, seed)
    parts = []
    step = max(1, (1 << 27) // case["V"])
    for lo in range(0, case["N"], step):
        rows = slice(lo, min(case["N"], lo + step))
        z = s["logits"][rows].double()
        y = z / case["temperature"]
        lse = torch.logsumexp(y, 1)
        lse = torch.where(torch.isinf(lse), torch.full_like(lse, float("inf")), lse)
        parts.append({"score": _exact_score, "score_grad": _exact_grad, "distill": _exact_distill}[case["op"]](
            case, s, rows, z, y, lse))
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}


def _exact_score(case, s, rows, z, y, lse):
    ids = s["ids"][rows].long()
    n = torch.arange(len(ids), device=z.device)
    out = {"logp": torch.where(ids == -1, 0.0, y[n, ids.clamp(min=0)] - lse)}
    if case["entropy"]:
        out["entropy"] = torch.special.entr(torch.exp(y - lse[:, None])).sum(1)
    if case["K"]:
        v, i = torch.sort(z, dim=1, descending=True, stable=True)
        v, i = v[:, :case["K"]], i[:, :case["K"]]
        out["top_ids"] = torch.where(v == float("-inf"), -1, i).int()
        out["top_logp"] = v / case["temperature"] - lse[:, None]
    return out


def _exact_grad(case, s, rows, z, y, lse):
    ids = s["ids"][rows].long()
    g = s["dlogp"][rows].double() * (ids != -1)
    logp = y - lse[:, None]
    p = torch.exp(logp)
    each = g[:, None].expand_as(p)
    if case["entropy"]:
        h = torch.special.entr(p).sum(1, keepdim=True)
        each = each + s["dentropy"][rows].double()[:, None] * (logp.clamp(min=-1e300) + h)
    d = -p * each
    n = torch.arange(len(ids), device=z.device)
    d[n, ids.clamp(min=0)] += g
    return {"dlogits": d / case["temperature"]}


def _exact_distill(case, s, rows, z, y, lse):
    tau, ids = case["temperature"], s["t_ids"][rows].long()
    t = s["t_vals"][rows].double().masked_fill(ids == -1, float("-inf"))
    q = torch.exp(t) if case["tail"] else torch.softmax(t / tau, 1)
    w = s["weight"][rows].double() if s["weight"] is not None else torch.ones_like(lse)
    logp = y - lse[:, None]
    at = torch.gather(logp, 1, ids.clamp(min=0))
    loss = (torch.special.xlogy(q, q) - torch.where(q > 0, q * at, 0.0)).sum(1)
    d = torch.exp(logp)
    total = q.sum(1)
    if case["tail"]:
        named = torch.zeros_like(z, dtype=torch.bool)
        n = torch.arange(len(ids), device=z.device)[:, None].expand_as(ids)
        named[n[ids != -1], ids[ids != -1]] = True
        log_rest = torch.logsumexp(y.masked_fill(named, float("-inf")), 1) - lse
        r = 1.0 - total
        r = torch.where(r < TAIL_MIN, 0.0, r)
        loss = loss + torch.where(r > 0, r * (torch.log(r) - log_rest), 0.0)
        share = torch.where(r > 0, r * torch.exp(-log_rest), 0.0)
        d = d * torch.where(named, (total + r)[:, None], (total + r - share)[:, None])
    else:
        d = d * total[:, None]
    d.scatter_add_(1, ids.clamp(min=0), -q)
    return {"loss": w * loss, "dlogits": d * (w * s["scale"] / tau)[:, None]}
