"""The operators behind several continuations of one prompt, as cases that can be timed and compared.

Two operators, each one pass through its public entry point:

  sample   drawing a token per row of logits with temperature, top-k, top-p and min-p from given random numbers
           (ops.sample_rows)
  prefix   attention of a batch whose sequences share a prompt's keys and values and go on in caches of their own
           (ops.shared_prefix_attention): one new token a sequence, a few, or whole prompts behind the prefix

Sizes are those of the configurations that the tests and the benchmark run, and ragged ones around them.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # interactive: one sequence of the 8B-shaped model, temperature alone; launches and host time count
        dict(name="sample_b1", kind="sample", dtype="bf16", rows=1, vocab=128256, pad=0, how="plain"),
        # the generation benchmark's batch, the usual pair of filters
        dict(name="sample_b16_topk_topp", kind="sample", dtype="bf16", rows=16, vocab=128256, pad=0, how="topk_topp"),
        # serving: nucleus sampling alone, whose border lies anywhere in the row
        dict(name="sample_b64_topp", kind="sample", dtype="bf16", rows=64, vocab=128256, pad=0, how="topp"),
        # the reference's precision and vocabulary with one more token, rows cut from a padded product
        dict(name="sample_f32_odd_minp", kind="sample", dtype="f32", rows=24, vocab=32001, pad=63, how="minp"),
        # the largest batch: every row with settings of its own, greedy ones among them
        dict(name="sample_b512_mixed", kind="sample", dtype="bf16", rows=512, vocab=128256, pad=0, how="mixed"),
        # the smallest attention call: the reference's fp32 precision and head size
        dict(name="prefix_f32_small", kind="prefix", dtype="f32", B=4, Hq=4, Hkv=4, D=64, S=1, prefix=61, past=8,
             ragged=False),
        # sixteen samples of one 2k prompt, at the generation benchmark's heads
        dict(name="prefix_b16_2k", kind="prefix", dtype="bf16", B=16, Hq=32, Hkv=8, D=128, S=1, prefix=2048,
             past=100, ragged=False),
        # serving: 64 conversations behind one long system prompt, each at its own length
        dict(name="prefix_b64_8k", kind="prefix", dtype="bf16", B=64, Hq=32, Hkv=8, D=128, S=1, prefix=8191,
             past=700, ragged=True),
        # few samples of a very long document
        dict(name="prefix_b4_32k", kind="prefix", dtype="bf16", B=4, Hq=32, Hkv=8, D=128, S=1, prefix=32000,
             past=257, ragged=True),
        # a model without grouped heads, heads of 64
        dict(name="prefix_mha_d64", kind="prefix", dtype="bf16", B=32, Hq=16, Hkv=16, D=64, S=1, prefix=1021,
             past=300, ragged=True),
        # five drafted tokens a sequence checked in one pass
        dict(name="prefix_draft5", kind="prefix", dtype="bf16", B=8, Hq=32, Hkv=8, D=128, S=5, prefix=3001,
             past=90, ragged=True),
        # questions of a padded batch behind one document: the prompt pass
        dict(name="prefix_prompts", kind="prefix", dtype="bf16", B=8, Hq=32, Hkv=8, D=128, S=257, prefix=4096,
             past=0, ragged=False),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_MOST_BYTES = 131e6  # of the largest listed sampling case
_MOST_FLOPS = 1.4e11  # of the largest listed attention case (bf16)


def draw(rng):
    dtype = "f32" if rng.random() < 0.25 else "bf16"
    if rng.random() < 0.45:
        vocab = rng.choice([32000, 128256, _log(rng, 500, 160000), _log(rng, 500, 160000)])
        rows = _log(rng, 1, 512)
        rows = max(1, min(rows, int(_MOST_BYTES / (vocab * (4 if dtype == "f32" else 2)))))
        return dict(kind="sample", dtype=dtype, rows=rows, vocab=vocab, pad=rng.choice([0, 0, rng.randint(1, 130)]),
                    how=rng.choice(["plain", "topk", "topk_topp", "topp", "minp", "mixed"]))
    D = rng.choice([32, 64, 128] if dtype == "f32" else [64, 128])
    Hkv = rng.choice([1, 2, 4, 8, 16])
    Hq = min(64, Hkv * rng.choice([1, 2, 4, 8]))
    S = rng.choice([1, 1, 1, rng.randint(2, 9), _log(rng, 10, 512)])
    B = _log(rng, 1, 64)
    c = dict(kind="prefix", dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, D=D, S=S, prefix=_log(rng, 1, 32768),
             past=rng.choice([0, _log(rng, 1, 2000)]), ragged=rng.random() < 0.6)
    most = _MOST_FLOPS / (16 if dtype == "f32" else 1)
    while work(c)["flops"] > most or B * Hq * S * (c["prefix"] + c["past"] + S) > 3e8:
        c["B"] = B = max(1, B // 2)
        c["prefix"] = max(1, c["prefix"] * 2 // 3)
        c["S"] = S = max(1, S * 3 // 4)
    return c


def _past(case):
    """Cache rows that each sequence holds before the call."""
    B, n = case["B"], case["past"]
    return [n * ((5 * b + 3) % B + 1) // B for b in range(B)] if case["ragged"] else [n] * B


def work(case):
    """Each input read once and each output written once; a product's term counts two."""
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    if c["kind"] == "sample":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * size + c["rows"] * 28, "flops": 4 * n}
    B, Hq, Hkv, D, S = (c[x] for x in ("B", "Hq", "Hkv", "D", "S"))
    past = _past(c)
    rows = 2 * Hkv * D * (c["prefix"] + sum(past) + B * S) + 2 * B * Hq * S * D
    pairs = sum(S * (c["prefix"] + n) + S * (S + 1) // 2 for n in past)
    return {"bytes": rows * size, "flops": 4.0 * D * Hq * pairs}


# ---------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------
def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DT[c["dtype"]]

    def rnd(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dt)

    def uni(n, lo=0.0, hi=1.0):
        return lo + (hi - lo) * torch.rand(n, generator=g, device="cuda")

    if c["kind"] == "sample":
        rows, V = c["rows"], c["vocab"]
        # logits as a language model gives them: falling with the logarithm of a token's rank, ranks scattered over
        # the vocabulary, noise on top
        rank = torch.rand((rows, V), generator=g, device="cuda").argsort(1)
        x = (-1.3 * torch.log(rank + 1.0) + torch.randn((rows, V), generator=g, device="cuda") + 8.0).to(dt)
        logits = torch.empty((rows, V + c["pad"]), dtype=dt, device="cuda")
        logits.fill_(1e4)  # what lies in the padding is nobody's token
        logits = logits[:, :V]
        logits.copy_(x)
        s = dict(kind="sample", logits=logits, u=uni(rows), temperature=0.8, top_k=0, top_p=1.0, min_p=0.0)
        how = c["how"]
        if how in ("topk", "topk_topp"):
            s["top_k"] = 50
        if how in ("topp", "topk_topp"):
            s["top_p"] = 0.95
        if how == "minp":
            s["min_p"] = 0.05
        if how == "mixed":  # settings of the requests that the batch happens to hold
            pick = uni(rows)
            s["temperature"] = torch.where(pick < 0.2, 0.0, uni(rows, 0.5, 1.3))
            s["top_k"] = torch.where(uni(rows) < 0.5, 0.0, uni(rows, 5.0, 200.0)).to(torch.int32)
            s["top_p"] = torch.where(uni(rows) < 0.5, 1.0, uni(rows, 0.5, 0.99))
            s["min_p"] = torch.where(uni(rows) < 0.7, 0.0, uni(rows, 0.01, 0.2))
        return s
    B, Hq, Hkv, D, S = (c[x] for x in ("B", "Hq", "Hkv", "D", "S"))
    past = _past(c)
    L = (max(past) + S + 63) // 64 * 64
    return dict(kind="prefix", q=rnd(B, Hq, S, D, std=1.5), kp=rnd(Hkv, c["prefix"], D), vp=rnd(Hkv, c["prefix"], D),
                k=rnd(B, Hkv, L, D), v=rnd(B, Hkv, L, D), n_prefix=c["prefix"], scale=1.0 / math.sqrt(D),
                n_past=torch.tensor(past, dtype=torch.int32, device="cuda") if c["ragged"] else past[0])


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _plain_sample(logits, u, temperature, top_k, top_p, min_p):
    """The filters on the sorted row, the draw in token order; in 64 bits: a token's border among 1e5 others is
    narrower than 32 bits resolve."""
    V = logits.shape[1]
    col = lambda t, d: torch.as_tensor(t, dtype=d, device=logits.device).reshape(-1, 1)  # noqa: E731
    t, k, p, m = col(temperature, torch.float64), col(top_k, torch.int64), col(top_p, torch.float64), \
        col(min_p, torch.float64)
    greedy = t <= 0
    k = torch.where(greedy, 1, torch.where(k > 0, k, V))
    t = torch.where(greedy, 1.0, t)
    x = logits.double()
    x, order = torch.sort(x, dim=1, descending=True, stable=True)  # equal logits: the lowest index first
    w = torch.exp((x - x[:, :1]) / t) * (torch.arange(V, device=x.device) < k)
    before = torch.cumsum(w, 1) - w
    keep = ((before < p * w.sum(1, keepdim=True)) | (p >= 1)) & (w >= m)
    kept = torch.zeros_like(w).scatter_(1, order, w * keep)
    run = torch.cumsum(kept, 1)
    return (run <= u.double().reshape(-1, 1) * run[:, -1:]).sum(1)


def _plain_prefix(q, kp, vp, k, v, n_prefix, n_past, scale):
    """One softmax over the prefix's keys and the sequence's own, in 32 bits; the prefix's products for the whole
    batch at once."""
    B, Hq, S, D = q.shape
    Hkv, L = k.shape[1], k.shape[2]
    G = Hq // Hkv
    qf = q.float().view(B, Hkv, G * S, D)
    qh = qf.transpose(0, 1).reshape(Hkv, B * G * S, D)
    sp = torch.bmm(qh, kp[:, :n_prefix].float().transpose(1, 2).contiguous()).view(Hkv, B, G * S, n_prefix)
    so = torch.matmul(qf, k.float().transpose(2, 3).contiguous())
    past = torch.as_tensor(n_past, device=q.device).reshape(-1, 1, 1, 1, 1)
    last = past + torch.arange(S, device=q.device).view(1, 1, 1, S, 1)
    seen = torch.arange(L, device=q.device) <= last
    so = so.view(B, Hkv, G, S, L).masked_fill(~seen, float("-inf")).view(B, Hkv, G * S, L)
    s = torch.cat([sp.transpose(0, 1), so], 3) * scale
    p = torch.exp(s - s.amax(3, keepdim=True))
    p = p / p.sum(3, keepdim=True)
    pp = p[..., :n_prefix].transpose(0, 1).reshape(Hkv, B * G * S, n_prefix)
    op = torch.bmm(pp, vp[:, :n_prefix].float()).view(Hkv, B, G * S, D).transpose(0, 1)
    o = op + torch.matmul(p[..., n_prefix:].contiguous(), v.float())
    return o.reshape(B, Hq, S, D).to(q.dtype)


def run(state):
    s = state
    if s["kind"] == "sample":
        a = (s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
        if own:
            from teenyformers_amd import ops
            return ops.sample_rows(*a)
        return _plain_sample(*a)
    a = (s["q"], s["kp"], s["vp"], s["k"], s["v"], s["n_prefix"], s["n_past"], s["scale"])
    if own:
        from teenyformers_amd import ops
        return ops.shared_prefix_attention(*a)
    return _plain_prefix(*a)


# ---------------------------------------------------------------------------
# from the definition, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "sample":
        x = s["logits"].double().cpu().numpy()
        rows, V = x.shape
        full = lambda t: np.broadcast_to(t.cpu().numpy() if torch.is_tensor(t) else t, rows)  # noqa: E731
        T, K, P, M, U = (full(s[n]) for n in ("temperature", "top_k", "top_p", "min_p", "u"))
        out = np.empty(rows, dtype=np.int64)
        for r in range(rows):
            if T[r] <= 0:
                out[r] = np.argmax(x[r])  # the first of equal ones
                continue
            w = np.exp((x[r] - x[r].max()) / float(T[r]))
            order = np.argsort(-x[r], kind="stable")
            n = V if K[r] <= 0 else min(V, int(K[r]))
            run_ = np.cumsum(w[order[:n]])
            if P[r] < 1:  # the shortest part that holds the share
                n = min(n, int(np.searchsorted(run_, float(P[r]) * run_[-1], side="left")) + 1)
            kept = order[:n]
            kept = np.sort(kept[w[kept] >= float(M[r])])
            c = np.cumsum(w[kept])
            out[r] = kept[np.searchsorted(c, float(U[r]) * c[-1], side="right")]
        return torch.from_numpy(out)
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    kp, vp = s["kp"].double(), s["vp"].double()
    B, Hq, S, D = q.shape
    Hkv, P = k.shape[1], s["n_prefix"]
    out = torch.empty_like(q)
    for b, n in enumerate(_past(case)):
        for h in range(Hq):
            j = h // (Hq // Hkv)
            keys = torch.cat([kp[j, :P], k[b, j, :n + S]])
            values = torch.cat([vp[j, :P], v[b, j, :n + S]])
            score = q[b, h].mm(keys.t()) * s["scale"]
            at = torch.arange(P + n + S, device=q.device)
            score[at[None, :] > P + n + torch.arange(S, device=q.device)[:, None]] = -math.inf
            out[b, h] = torch.softmax(score, 1).mm(values)
    return out
