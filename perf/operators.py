"""The vocabulary's discrete operators on real work: calls a program makes through the package's public
entry points, beside each operator's plain form in elementary torch operations.

* ``distill``: a training step of ``softmax_distill``, the head trained on a teacher's top logits: the loss
  and the gradients of every parameter, or of h alone through a frozen head;
* ``lookup`` / ``lookup_train``: ``embedding_lookup``, token ids to scaled rows of the table, without or with
  the table's gradient;
* ``sample``: ``sample_tokens``, one token per row of logits from a given uniform number, under a
  temperature, top-k, top-p and min-p.

A case is a dict of plain values; ``draw`` gives more of the same ranges.  ``own`` selects what ``run``
computes: the package's operators, or the plain forms.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
RAGGED_TAIL = 0.25   # share of the last tokens of a padded batch that carry no loss, at most


def _distill(name, dtype, tokens, K, V, T, *, bias=True, temperature=1.0, weight="none", z=0.0, spread=1.0, wrt="all"):
    c = dict(op="distill", dtype=dtype, tokens=tokens, K=K, V=V, T=T, bias=bias, temperature=temperature,
             weight=weight, z=z, spread=spread, wrt=wrt)
    return {"name": name, **c} if name else c


def _lookup(name, op, dtype, tokens, V, D, *, scale=1.0, pad=0.0):
    c = dict(op=op, dtype=dtype, tokens=tokens, V=V, D=D, scale=scale, pad=pad)
    return {"name": name, **c} if name else c


def _sample(name, dtype, rows, V, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=False, spread=3.0):
    c = dict(op="sample", dtype=dtype, rows=rows, V=V, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p,
             mixed=mixed, spread=spread)
    return {"name": name, **c} if name else c


def listed():
    return [
        # a plumbing-size step in fp32: a call of a few launches
        _distill("distill_small_fp32", "fp32", 512, 256, 4096, 8, spread=1.0),
        # a microbatch of a model with a mid-size vocabulary, padded sequences, soft targets at temperature 2
        _distill("distill_microbatch", "bf16", 500, 1024, 32000, 16, temperature=2.0, weight="ragged", z=1e-4),
        # a frozen head: gradients of h alone, fp16 under a loss scale, a wide teacher list
        _distill("distill_frozen_fp16", "fp16", 2048, 1024, 151936, 64, bias=False, spread=3.0, wrt="h"),
        # the large step: half the headline's tokens on a wider model
        _distill("distill_large", "bf16", 8192, 4096, 128256, 32, weight="bernoulli", temperature=1.5),
        # one decoding step of 48 sequences: the sampled ids become the next inputs
        _lookup("lookup_decode", "lookup", "bf16", 48, 128256, 4096),
        # a prompt of odd length, fp16, scaled by sqrt(D)
        _lookup("lookup_prompt_fp16", "lookup", "fp16", 8191, 151936, 1000, scale=math.sqrt(1000)),
        # the plumbing-size step in fp32
        _lookup("lookup_train_small", "lookup_train", "fp32", 512, 4096, 256),
        # a batch of 8 padded sequences onto a mid-width table
        _lookup("lookup_train_padded", "lookup_train", "bf16", 32768, 256000, 300, pad=0.2),
        # a training step's inputs on a table tied to the headline head
        _lookup("lookup_train_tied", "lookup_train", "bf16", 16384, 151936, 2560, scale=math.sqrt(2560)),
        # one token of one sequence, the usual filters
        _sample("sample_one", "bf16", 1, 151936, temperature=0.7, top_k=50, top_p=0.9),
        # one decoding step of a batch, nucleus sampling over the whole vocabulary
        _sample("sample_batch", "fp32", 48, 128256, top_p=0.95, min_p=0.001),
        # rollouts: many rows, every request with settings of its own
        _sample("sample_rollouts", "bf16", 512, 151936, mixed=True),
    ]


# what a drawn case may cost at most
DRAW_FLOPS = {"bf16": 2e13, "fp16": 2e13, "fp32": 1e12}
DRAW_TABLE, DRAW_ROWS, DRAW_LOGITS = 151936 * 2560, 16384 * 2560, 512 * 151936


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["distill", "distill", "distill", "lookup", "lookup_train", "lookup_train", "sample", "sample", "sample"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    while True:
        V = _log(rng, 1000, 256000)
        if op == "distill":
            K = _log(rng, 64, 4096)
            if rng.random() < 0.75:
                K = max(64, K // 64 * 64)   # hidden sizes are mostly multiples of 64; others are padded by the call
            c = _distill(None, dtype, _log(rng, 1, 8192), K, V, _log(rng, 1, 128), bias=rng.random() < 0.7,
                         temperature=rng.choice([1.0, 1.5, 2.0]), weight=rng.choice(["none", "bernoulli", "ragged"]),
                         z=rng.choice([0.0, 1e-4]), spread=rng.choice([1.0, 3.0]), wrt=rng.choice(["all", "all", "h"]))
            if work(c)["flops"] <= DRAW_FLOPS[dtype]:
                return c
        elif op == "sample":
            c = _sample(None, dtype, _log(rng, 1, 512), V, temperature=rng.choice([0.0, 0.7, 1.0, 1.3]),
                        top_k=rng.choice([0, 0, _log(rng, 1, 2000)]), top_p=rng.choice([1.0, 0.5, 0.9, 0.99]),
                        min_p=rng.choice([0.0, 0.0, 0.02]), mixed=rng.random() < 0.3, spread=rng.choice([1.0, 3.0, 6.0]))
            if c["rows"] * V <= DRAW_LOGITS:
                return c
        else:
            D = _log(rng, 16, 4096)
            tokens = _log(rng, 1 if op == "lookup" else 64, 65536)
            c = _lookup(None, op, dtype, tokens, V, D, scale=rng.choice([1.0, math.sqrt(D)]),
                        pad=rng.choice([0.0, 0.0, 0.3]))
            if V * D * BYTES[dtype] <= 2 * DRAW_TABLE and tokens * D * BYTES[dtype] <= 2 * DRAW_ROWS:
                return c


def _zipf(g, shape, V):
    """Token ids as text has them: the r-th most frequent with probability near 1 / (r ln V), at scattered ids."""
    r = torch.exp(torch.rand(shape, device=DEVICE, generator=g, dtype=torch.float64) * math.log(V)).long().clamp_(1, V) - 1
    return (r * 7919 + 13) % V if V % 7919 else r


def _inputs(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    V = case["V"]

    def r(*s, sc=1.0):
        return torch.randn(*s, device=DEVICE, generator=g).mul_(sc)

    if case["op"] == "sample":
        R = case["rows"]
        x = r(R, V, sc=case["spread"])
        x[:, (torch.rand(V, device=DEVICE, generator=g) < 0.02)] = -math.inf   # masked ids: unused slots, control tokens
        t = {"logits": x.to(dt), "u": torch.rand(R, device=DEVICE, generator=g)}
        for name in ("temperature", "top_k", "top_p", "min_p"):
            t[name] = case[name]
        if case["mixed"]:   # every request with settings of its own, some without any filter, some greedy

            def pick(values, dtype):
                at = torch.randint(0, len(values), (R,), device=DEVICE, generator=g)
                return torch.tensor(values, device=DEVICE, dtype=dtype)[at]

            t["temperature"] = pick([0.0, 0.6, 0.8, 1.0, 1.2], torch.float32)
            t["top_k"] = pick([0, 0, 20, 50, 1000], torch.int32)
            t["top_p"] = pick([1.0, 0.8, 0.9, 0.95], torch.float32)
            t["min_p"] = pick([0.0, 0.0, 0.05], torch.float32)
        return t
    if case["op"] == "distill":
        N, K, T = case["tokens"], case["K"], case["T"]
        t = {"h": r(N, K).to(dt), "W": r(V, K, sc=case["spread"] * K ** -0.5).to(dt)}
        t["bias"] = r(V, sc=0.5 if case["spread"] > 1 else 0.02).to(dt) if case["bias"] else None
        ids = _zipf(g, (N, T), V)
        # a teacher's list holds an id once: later repeats are absent entries (id -1), so lists are of uneven length
        s, at = ids.sort(dim=1, stable=True)
        again = torch.zeros_like(s, dtype=torch.bool)
        again[:, 1:] = s[:, 1:] == s[:, :-1]
        ids = torch.where(torch.zeros_like(again).scatter_(1, at, again), -1, ids)
        t["teacher_ids"] = ids
        t["teacher_logits"] = (12 - torch.rand(N, T, device=DEVICE, generator=g).add_(1e-3).log_().neg_().cumsum(1)).to(dt)
        t["weight"] = None
        if case["weight"] == "bernoulli":
            t["weight"] = (torch.rand(N, device=DEVICE, generator=g) >= 0.1).float()
        elif case["weight"] == "ragged":
            n = torch.randint(0, max(1, int(RAGGED_TAIL * N)) + 1, (1,), device=DEVICE, generator=g)
            t["weight"] = (torch.arange(N, device=DEVICE) < N - n).float()
        # the loss's cotangent: fp16 trains under a loss scale
        t["g"] = torch.tensor(float(N) if case["dtype"] == "fp16" else 1.0, device=DEVICE)
        return t
    N, D = case["tokens"], case["D"]
    ids = _zipf(g, (N,), V)
    if case["pad"]:
        ids = torch.where(torch.rand(N, device=DEVICE, generator=g) < case["pad"], -1, ids)
    t = {"ids": ids, "E": r(V, D, sc=0.02).to(dt)}
    if case["op"] == "lookup_train":
        t["g"] = r(N, D).to(dt)
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    state = {"case": case, **t}
    if case["op"] == "distill":
        state["params"] = [t["h"]] if case["wrt"] == "h" else [x for x in (t["h"], t["W"], t["bias"]) if x is not None]
        for x in state["params"]:
            x.requires_grad_(True)
    elif case["op"] == "lookup_train":
        t["E"].requires_grad_(True)
    return state


# ---------------------------------------------------------------- the plain forms
def _plain_distill(s):
    """loss = sum_n w_n (sum_k p_nk (log p_nk - z_nk + lse_n) + zw lse_n^2) / sum_n w_n over the tokens with a
    teacher, with z = h W^T / temperature + bias / temperature and p = softmax(teacher / temperature)."""
    case = s["case"]
    tau, zw = case["temperature"], case["z"]
    h, W = s["h"].detach().float(), s["W"].detach().float()
    ids = s["teacher_ids"]
    there = ids >= 0
    at = ids.clamp(min=0)
    t = torch.where(there, s["teacher_logits"].float() / tau, -math.inf)
    top = t.amax(dim=1, keepdim=True)
    any_there = there.any(dim=1)
    p = torch.where(there, (t - torch.where(any_there[:, None], top, 0.0)).exp(), 0.0)
    p = p / p.sum(dim=1, keepdim=True).clamp_min(1e-30)
    S = (h @ W.t()).mul_(1 / tau)
    if s["bias"] is not None:
        S += s["bias"].detach().float() / tau
    m = S.amax(dim=1)
    z = S.gather(1, at)
    P = S.sub_(m[:, None]).exp_()
    total = P.sum(dim=1)
    lse = m + total.log()
    w = s["weight"] if s["weight"] is not None else torch.ones_like(lse)
    w = torch.where(any_there, w, 0.0)
    kl = torch.where(p > 0, p * (p.clamp_min(1e-38).log() - z + lse[:, None]), 0.0).sum(dim=1)
    denom = torch.where(w.sum() != 0, w.sum(), 1.0)   # a batch without a token to learn from: 0
    loss = (w * (kl + zw * lse.square())).sum() / denom
    g = s["g"] * w / denom
    dS = P.mul_(((g * (1 + 2 * zw * lse)) / total)[:, None])
    dS.scatter_add_(1, at, -g[:, None] * p)
    out = [loss, ((dS @ W) / tau).to(s["h"].dtype)]
    if case["wrt"] == "all":
        out.append(((dS.t() @ h) / tau).to(s["W"].dtype))
        if s["bias"] is not None:
            out.append((dS.sum(dim=0) / tau).to(s["bias"].dtype))
    return out


def _plain_lookup(s):
    case, ids, E = s["case"], s["ids"], s["E"].detach()
    there = (ids >= 0)[:, None]
    at = ids.clamp(min=0)
    out = torch.where(there, E[at].float() * case["scale"], 0.0).to(E.dtype)
    if case["op"] == "lookup":
        return out
    gE = torch.zeros(E.shape, device=E.device).index_add_(0, at, torch.where(there, s["g"].float(), 0.0))
    return out, gE.mul_(case["scale"]).to(E.dtype)


def _column(x, dtype):
    return x.to(dtype)[:, None] if isinstance(x, torch.Tensor) else torch.full((1, 1), x, dtype=dtype, device=DEVICE)


def _plain_sample(s):
    """In 64 bits: the drawn token lies next to the borders of the cumulative sums."""
    x = s["logits"].double()
    V = x.shape[1]
    tau, k = _column(s["temperature"], torch.float64), _column(s["top_k"], torch.int64)
    p, mp = _column(s["top_p"], torch.float64), _column(s["min_p"], torch.float64)
    k = torch.where((k <= 0) | (k > V), V, k)
    k = torch.where(tau == 0, 1, k)
    tau = torch.where(tau == 0, 1.0, tau)
    xs, order = x.sort(dim=1, descending=True, stable=True)
    ws = ((xs - xs[:, :1]) / tau).exp()
    keep = (torch.arange(V, device=x.device)[None, :] < k).expand(x.shape)
    wk = torch.where(keep, ws, 0.0)
    cum = wk.cumsum(dim=1)
    keep = keep & ((p >= 1) | (cum - wk < p * cum[:, -1:]))
    keep = keep & (ws >= mp)
    keep[:, 0] = True
    w = torch.zeros_like(ws).scatter_(1, order, torch.where(keep, ws, 0.0))
    cum = w.cumsum(dim=1)
    total = cum[:, -1:]
    token = (cum <= s["u"].double()[:, None] * total).sum(dim=1, keepdim=True)
    return token[:, 0], (w.gather(1, token) / total).log()[:, 0].float()


def run(state):
    case = state["case"]
    if not own:
        return {"distill": _plain_distill, "lookup": _plain_lookup, "lookup_train": _plain_lookup,
                "sample": _plain_sample}[case["op"]](state)
    import swvr_amd
    if case["op"] == "sample":
        return swvr_amd.sample_tokens(state["logits"], state["u"], temperature=state["temperature"],
                                      top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"])
    if case["op"] == "distill":
        loss = swvr_amd.softmax_distill(state["h"], state["W"], state["teacher_logits"], state["teacher_ids"],
                                        state["bias"], temperature=case["temperature"], weight=state["weight"],
                                        z_loss_weight=case["z"])
        return [loss.detach(), *torch.autograd.grad(loss, state["params"], state["g"])]
    if case["op"] == "lookup":
        with torch.no_grad():
            return swvr_amd.embedding_lookup(state["ids"], state["E"], scale=case["scale"])
    out = swvr_amd.embedding_lookup(state["ids"], state["E"], scale=case["scale"])
    return (out.detach(), *torch.autograd.grad(out, [state["E"]], state["g"]))


def work(case):
    """Each input read and each output written once.  Distillation: the scores once, and one product for each
    matrix gradient, over the tokens of non-zero weight (``bernoulli``: nine of ten).  Lookups: the rows named
    by the ids; their gradient: the cotangent's rows and the whole table's gradient.  Sampling: the logits."""
    e = BYTES[case["dtype"]]
    V = case["V"]
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (e * V + 16.0), "flops": 3.0 * case["rows"] * V}
    if case["op"] == "distill":
        N, K, T = case["tokens"], case["K"], case["T"]
        active = N * {"none": 1.0, "bernoulli": 0.9, "ragged": 1.0 - RAGGED_TAIL / 2}[case["weight"]]
        nb = V if case["bias"] else 0
        params, every = e * (N * K + V * K + nb), case["wrt"] == "all"
        written = params if every else e * N * K
        return {"bytes": params + written + N * T * (8.0 + e) + 4 * N, "flops": 2.0 * active * V * K * (3 if every else 2)}
    N, D = case["tokens"], case["D"]
    live = N * (1 - case["pad"])
    forward = live * D * e + N * D * e + 8.0 * N
    if case["op"] == "lookup":
        return {"bytes": forward, "flops": 1.0 * live * D}
    return {"bytes": forward + live * D * e + V * D * e, "flops": 2.0 * live * D}


# ---------------------------------------------------------------- the definitions in 64 bits
EXACT_FLOPS = 4e14
EXACT_BLOCK = 4 << 30   # bytes of one block of 64-bit scores


def _exact_distill(case, t):
    tau, zw, T, V = case["temperature"], case["z"], case["T"], case["V"]
    h, W = t["h"].double(), t["W"].double()
    b = t["bias"].double() if t["bias"] is not None else None
    ids = t["teacher_ids"]
    N = h.shape[0]
    w = t["weight"].double() if t["weight"] is not None else torch.ones(N, dtype=torch.float64, device=DEVICE)
    w = w * (ids >= 0).any(dim=1)
    denom = torch.where(w.sum() != 0, w.sum(), 1.0)
    loss = torch.zeros((), dtype=torch.float64, device=DEVICE)
    gh, gW = torch.empty_like(h), torch.zeros_like(W)
    gb = torch.zeros(V, dtype=torch.float64, device=DEVICE)
    step = max(1, EXACT_BLOCK // (8 * V))
    for n0 in range(0, N, step):
        r = slice(n0, min(N, n0 + step))
        n = torch.arange(r.stop - n0, device=DEVICE)
        logq = torch.addmm(b, h[r], W.t()) if b is not None else h[r] @ W.t()
        logq /= tau
        lse = torch.logsumexp(logq, dim=1)
        logq -= lse[:, None]
        teacher = t["teacher_logits"][r].double() / tau
        teacher = teacher.masked_fill(ids[r] < 0, -math.inf)
        logp = (teacher - torch.logsumexp(teacher, dim=1, keepdim=True)).nan_to_num_(nan=-math.inf, neginf=-math.inf)
        wn = w[r] / denom
        terms = zw * lse.square()
        dS = logq.exp()
        dS *= (wn * t["g"] * (1 + 2 * zw * lse))[:, None]
        for k in range(T):
            at = ids[r][:, k].clamp(min=0)
            p = logp[:, k].exp()
            terms = terms + torch.where(p > 0, p * (logp[:, k] - logq[n, at]), 0.0)
            dS[n, at] -= wn * t["g"] * p
        loss += (wn * terms).sum()
        gh[r] = dS @ W / tau
        if case["wrt"] == "all":
            gW += dS.t() @ h[r]
            gb += dS.sum(dim=0)
    if case["wrt"] == "h":
        return [loss, gh]
    return [loss, gh, gW / tau] + ([gb / tau] if b is not None else [])


def _exact_sample(case, t):
    """Row by row, the kept set as a prefix of the order by logit."""
    R, V = t["logits"].shape

    def of(name, i):
        return t[name][i].item() if isinstance(t[name], torch.Tensor) else t[name]

    tokens, logprobs = [], []
    for i in range(R):
        x = t["logits"][i].double()
        tau, k, p, mp = (of(name, i) for name in ("temperature", "top_k", "top_p", "min_p"))
        order = torch.argsort(-x, stable=True)
        if tau == 0:
            tokens.append(order[0])
            logprobs.append(torch.zeros((), dtype=torch.float64, device=DEVICE))
            continue
        w = torch.exp((x[order] - x[order[0]]) / tau)
        if 0 < k < V:
            w = w[:k]
        if p < 1:
            before = torch.cat([w.new_zeros(1), w.cumsum(0)[:-1]])
            w = w[:max(1, int((before < p * w.sum()).sum()))]
        w = w[:max(1, int((w >= mp).sum()))]
        kept, back = order[:w.numel()].sort()
        w = w[back]
        j = int(torch.searchsorted(w.cumsum(0), t["u"][i].double() * w.sum(), right=True))
        tokens.append(kept[j])
        logprobs.append(torch.log(w[j] / w.sum()))
    return torch.stack(tokens), torch.stack(logprobs)


def exact(case, seed):
    if case["op"] == "distill" and work(case)["flops"] > EXACT_FLOPS:
        return None
    t = _inputs(case, seed)
    if case["op"] == "distill":
        return _exact_distill(case, t)
    if case["op"] == "sample":
        return _exact_sample(case, t)
    there = t["ids"] >= 0
    out = torch.zeros(case["tokens"], case["D"], dtype=torch.float64, device=DEVICE)
    out[there] = t["E"][t["ids"][there]].double() * case["scale"]
    if case["op"] == "lookup":
        return out
    gE = torch.zeros(case["V"], case["D"], dtype=torch.float64, device=DEVICE)
    gE.index_put_((t["ids"][there],), t["g"][there].double() * case["scale"], accumulate=True)
    return out, gE
