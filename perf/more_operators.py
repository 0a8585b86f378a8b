"""The operators behind a paged cache and drafted tokens, as cases that can be timed and compared.

Four operators, each one pass through its public entry point:

  append   the QKV projection's rows split, rotated and written to the pages of their sequences
           (ops.paged_qkv_rope_split)
  attn     attention of each sequence's new tokens over its pages: one token, a few drafted ones, a chunk of a prompt,
           or a batch that mixes them (ops.paged_attention)
  copy     pages copied within the pool, of all layers at once: a forked sequence's last page, a compacted pool
           (ops.copy_pages)
  verify   drafted tokens checked against the target's probabilities from given random numbers, and the token after
           the accepted ones (ops.verify_drafts)

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
        # the smallest step: the reference's fp32 precision and head size, three drafted tokens a sequence
        dict(name="attn_f32_small", kind="attn", dtype="f32", B=4, Hq=4, Hkv=4, D=64, page=16, S=3, past=61,
             ragged=True, chunk=0),
        # interactive: one sequence of the 8B-shaped model; launches and host time count
        dict(name="attn_b1", kind="attn", dtype="bf16", B=1, Hq=32, Hkv=8, D=128, page=16, S=1, past=700,
             ragged=False, chunk=0),
        # five tokens a sequence checked in one pass, heads of 64 without groups
        dict(name="attn_draft5_d64", kind="attn", dtype="bf16", B=8, Hq=16, Hkv=16, D=64, page=32, S=5, past=3001,
             ragged=True, chunk=0),
        # serving: 64 conversations, each at its own length
        dict(name="attn_b64", kind="attn", dtype="bf16", B=64, Hq=32, Hkv=8, D=128, page=64, S=1, past=8191,
             ragged=True, chunk=0),
        # a serving step: 2048 tokens of a long prompt among the next tokens of 32 conversations
        dict(name="attn_mixed", kind="attn", dtype="bf16", B=33, Hq=32, Hkv=8, D=128, page=16, S=1, past=6144,
             ragged=True, chunk=2048),
        # the new tokens of 64 conversations
        dict(name="append_b64", kind="append", dtype="bf16", B=64, Hq=32, Hkv=8, D=128, page=64, S=1, past=8191,
             ragged=True, chunk=0),
        # a prompt's chunk among them, far into its document
        dict(name="append_chunk", kind="append", dtype="bf16", B=17, Hq=32, Hkv=8, D=128, page=16, S=1, past=30011,
             ragged=True, chunk=8192),
        # sixteen forks of one sequence: its last page, in all layers of the 8B-shaped model
        dict(name="copy_fork", kind="copy", dtype="bf16", planes=64, Hkv=8, D=128, page=16, pool=64, moves=16, fork=True),
        # the pool compacted after a third of its sequences ended
        dict(name="copy_compact", kind="copy", dtype="bf16", planes=64, Hkv=8, D=128, page=64, pool=200, moves=67,
             fork=False),
        # interactive, drafts looked up in the prompt: no draft model
        dict(name="verify_b1_lookup", kind="verify", dtype="bf16", B=1, K=4, vocab=128256, q=False, temp=0.8),
        # the generation benchmark's batch with a small draft model
        dict(name="verify_b16", kind="verify", dtype="bf16", B=16, K=4, vocab=128256, q=True, temp=0.8),
        # serving, eight drafts, every sequence at a temperature of its own (greedy ones among them)
        dict(name="verify_b48_mixed", kind="verify", dtype="bf16", B=48, K=8, vocab=128256, q=True, temp=-1.0),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_MOST = {"attn": 1.2e9, "append": 2.0e8, "copy": 1.1e9, "verify": 2.0e8}  # bytes of the largest listed cases
_MOST_FLOPS = 2.5e11  # (bf16)


def draw(rng):
    dtype = "f32" if rng.random() < 0.25 else "bf16"
    kind = rng.choice(["attn", "attn", "attn", "append", "copy", "verify", "verify"])
    D = rng.choice([32, 64, 128] if dtype == "f32" else [64, 128])
    Hkv = rng.choice([1, 2, 4, 8, 16])
    page = rng.choice([16, 32, 64, 128])
    if kind == "verify":
        c = dict(kind=kind, dtype=dtype, B=_log(rng, 1, 48), K=rng.randint(1, 8),
                 vocab=rng.choice([32000, 128256, _log(rng, 500, 160000), _log(rng, 500, 160000)]),
                 q=rng.random() < 0.6, temp=rng.choice([0.0, 1.0, rng.uniform(0.3, 1.5), -1.0]))
        while work(c)["bytes"] > _MOST[kind]:
            c["B"] = max(1, c["B"] // 2)
            c["vocab"] = c["vocab"] if c["B"] > 1 else c["vocab"] * 3 // 4
        return c
    if kind == "copy":
        pool = _log(rng, 4, 300)
        fork = rng.random() < 0.5
        c = dict(kind=kind, dtype=dtype, planes=2 * rng.choice([1, 2, 6, 16, 32]), Hkv=Hkv, D=D, page=page, pool=pool,
                 moves=rng.randint(1, pool // 2), fork=fork)
        while work(c)["bytes"] > _MOST[kind]:
            c["planes"] = max(2, c["planes"] // 4 * 2)
            c["pool"] = max(4, c["pool"] // 2)
            c["moves"] = max(1, c["moves"] // 2)
        return c
    Hq = min(64, Hkv * rng.choice([1, 2, 4, 8]))
    c = dict(kind=kind, dtype=dtype, B=_log(rng, 1, 64), Hq=Hq, Hkv=Hkv, D=D, page=page,
             S=rng.choice([1, 1, 1, rng.randint(2, 9), _log(rng, 10, 300)]), past=rng.choice([0, _log(rng, 1, 32000)]),
             ragged=rng.random() < 0.7, chunk=rng.choice([0, 0, _log(rng, 10, 4096)]))
    while (work(c)["bytes"] > _MOST[kind] or work(c)["flops"] > _MOST_FLOPS / (16 if dtype == "f32" else 1)
           or Hq * _lens(c)[-1] * (c["past"] + _lens(c)[-1]) > 1e9):
        c["B"] = max(1, c["B"] // 2)
        c["past"] = c["past"] * 2 // 3
        c["S"] = max(1, c["S"] * 3 // 4)
        c["chunk"] = c["chunk"] * 3 // 4
    return c


def _pasts(case):
    """Keys that each sequence holds before the call."""
    B, n = case["B"], case["past"]
    past = [n * ((5 * b + 3) % B + 1) // B for b in range(B)] if case["ragged"] else [n] * B
    past[-1] = n
    return past


def _lens(case):
    """New tokens of each sequence."""
    lens = [case["S"]] * case["B"]
    if case["chunk"]:
        lens[-1] = case["chunk"]
    return lens


def work(case):
    """Each input read once and each output written once; a product's term counts two."""
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    if c["kind"] == "verify":
        rows = c["B"] * (c["K"] + 1 + (c["K"] if c["q"] else 0))
        return {"bytes": rows * c["vocab"] * size + c["B"] * (c["K"] + 1) * 24, "flops": 4 * rows * c["vocab"]}
    if c["kind"] == "copy":
        return {"bytes": 2 * c["moves"] * c["planes"] * c["Hkv"] * c["page"] * c["D"] * size, "flops": 0}
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    past, lens = _pasts(c), _lens(c)
    if c["kind"] == "append":
        return {"bytes": 2 * sum(lens) * (Hq + 2 * Hkv) * D * size, "flops": 3 * sum(lens) * (Hq + Hkv) * D}
    keys = sum(past) + sum(lens)
    pairs = sum(n * s + s * (s + 1) // 2 for n, s in zip(past, lens))
    return {"bytes": (2 * Hkv * D * keys + 2 * sum(lens) * Hq * D) * size, "flops": 4.0 * D * Hq * pairs}


# ---------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------
def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DT[c["dtype"]]

    def rnd(*shape, std=1.0):
        if math.prod(shape) < 1 << 28:
            return (torch.randn(shape, generator=g, device="cuda") * std).to(dt)
        out = torch.empty(shape, dtype=dt, device="cuda")
        for part in out.view(-1).split(1 << 28):
            part.copy_(torch.randn(part.shape, generator=g, device="cuda") * std)
        return out

    def whole(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    if c["kind"] == "verify":
        B, K, V = c["B"], c["K"], c["vocab"]
        # logits as a language model gives them: falling with the logarithm of a token's rank, ranks scattered over
        # the vocabulary, noise on top; the draft model's are the target's with noise of their own
        rank = torch.stack([torch.rand((K + 1, V), generator=g, device="cuda").argsort(1) for _ in range(B)])
        x = -1.3 * torch.log(rank + 1.0) + torch.randn((B, K + 1, V), generator=g, device="cuda") + 8.0
        y = x[:, :K] + 0.7 * torch.randn((B, K, V), generator=g, device="cuda")
        temp = c["temp"]
        if temp < 0:  # what the requests of the batch ask for
            temp = 0.5 + 0.8 * torch.rand(B, generator=g, device="cuda")
            temp = torch.where(torch.rand(B, generator=g, device="cuda") < 0.2, 0.0, temp)
        t = torch.as_tensor(temp, device="cuda").reshape(-1, 1, 1)
        # drafts drawn from the draft model's distribution (Gumbel's way), or its first choice
        noise = -torch.log(-torch.log(torch.rand((B, K, V), generator=g, device="cuda").clamp(1e-7, 1 - 1e-7)))
        drafts = (y.to(dt).float() + (t * noise if c["q"] else 0.0)).argmax(2)
        if K > 1:  # one sequence has a draft less than the others
            drafts[0, K - 1] = -1
        return dict(kind="verify", logits=x.to(dt), drafts=drafts, u=torch.rand((B, K + 1), generator=g, device="cuda"),
                    draft_logits=y.to(dt) if c["q"] else None, temperature=temp)
    Hkv, D, page = c["Hkv"], c["D"], c["page"]
    if c["kind"] == "copy":
        order = torch.randperm(c["pool"], generator=torch.Generator().manual_seed(int(seed))).tolist()
        n = c["moves"]
        src = [order[0]] * n if c["fork"] else order[:n]
        return dict(kind="copy", pages=rnd(c["planes"], c["pool"], Hkv, page, D), src=src, dst=order[n:2 * n])
    Hq = c["Hq"]
    past, lens = _pasts(c), _lens(c)
    T = sum(lens)
    need = [(n + s + page - 1) // page for n, s in zip(past, lens)]
    n_pages = sum(need) + 3
    # the pool's pages in the order in which the sequences happened to take them
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(int(seed))).tolist()
    table = np.full((c["B"], max(need)), -1, dtype=np.int32)
    for b, n in enumerate(need):
        table[b, :n] = order[:n]
        order = order[n:]
    starts = np.concatenate([[0], np.cumsum(lens)])
    s = dict(kind=c["kind"], k=rnd(n_pages, Hkv, page, D), v=rnd(n_pages, Hkv, page, D),
             table=torch.from_numpy(table).cuda(), past=past, lens=lens, n_past=whole(past),
             starts=whole(starts.tolist()), max_new=max(lens), max_keys=max(n + m for n, m in zip(past, lens)))
    if c["kind"] == "append":
        s.update(qkv=rnd(T, (Hq + 2 * Hkv) * D), Hq=Hq, Hkv=Hkv, base=5e5)
    else:
        s.update(q=rnd(T, Hq, D, std=1.5), scale=1.0 / math.sqrt(D))
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _plain_attn(s):
    """A sequence at a time: its keys gathered, one softmax over them, in 32 bits."""
    q, (_, Hkv, page, D) = s["q"], s["k"].shape
    out = torch.empty_like(q)
    G = q.shape[1] // Hkv
    t0 = 0
    for b, (n, m) in enumerate(zip(s["past"], s["lens"])):
        pages = s["table"][b, :(n + m + page - 1) // page].long()
        k = s["k"][pages].float().transpose(0, 1).reshape(Hkv, -1, D)[:, :n + m]
        v = s["v"][pages].float().transpose(0, 1).reshape(Hkv, -1, D)[:, :n + m]
        qb = q[t0:t0 + m].float().view(m, Hkv, G, D).permute(1, 2, 0, 3).reshape(Hkv, G * m, D)
        x = torch.bmm(qb, k.transpose(1, 2).contiguous()) * s["scale"]
        unseen = torch.arange(n + m, device=q.device) > n + torch.arange(m, device=q.device)[:, None]
        x = x.view(Hkv, G, m, n + m).masked_fill(unseen, float("-inf")).view(Hkv, G * m, n + m)
        p = torch.exp(x - x.amax(2, keepdim=True))
        o = torch.bmm(p / p.sum(2, keepdim=True), v.contiguous())
        out[t0:t0 + m] = o.view(Hkv, G, m, D).permute(2, 0, 1, 3).reshape(m, Hkv * G, D).to(q.dtype)
        t0 += m
    return out


def _plain_append(s):
    """Angles in 64 bits (at position 30000 those of 32 bits are off by 1e-3), the rotation in 32."""
    qkv, Hq, Hkv = s["qkv"], s["Hq"], s["Hkv"]
    _, _, page, D = s["k"].shape
    T = qkv.shape[0]
    seq = torch.repeat_interleave(torch.arange(len(s["lens"]), device=qkv.device), (s["starts"][1:] - s["starts"][:-1]).long(),
                                  output_size=T)
    pos = s["n_past"].long()[seq] + torch.arange(T, device=qkv.device) - s["starts"].long()[seq]
    inv = s["base"] ** (-torch.arange(0, D, 2, dtype=torch.float64, device=qkv.device) / D)
    angle = pos.double()[:, None] * inv
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    x = qkv.view(T, Hq + 2 * Hkv, D)
    even, odd = x[:, :Hq + Hkv, 0::2].float(), x[:, :Hq + Hkv, 1::2].float()
    y = torch.stack([even * cos - odd * sin, even * sin + odd * cos], 3).view(T, Hq + Hkv, D).to(qkv.dtype)
    at = s["table"][seq, pos // page].long()
    s["k"][at, :, pos % page] = y[:, Hq:]
    s["v"][at, :, pos % page] = x[:, Hq + Hkv:]
    return y[:, :Hq].contiguous(), s["k"], s["v"]


def _plain_verify(logits, drafts, u, draft_logits, temperature):
    """In 64 bits: a token's border among 1e5 others is narrower than 32 bits resolve."""
    B, n, V = logits.shape
    K = n - 1
    t = torch.as_tensor(temperature, dtype=torch.float64, device=logits.device).reshape(-1, 1, 1).expand(B, 1, 1)

    def weights(x):
        x = x.double()
        w = torch.exp((x - x.amax(2, keepdim=True)) / torch.where(t > 0, t, 1.0))
        first = torch.zeros_like(w).scatter_(2, x.argmax(2, keepdim=True), 1.0)
        w = torch.where(t > 0, w, first)
        return w / w.sum(2, keepdim=True)

    p = weights(logits)
    real = (drafts >= 0) & (drafts < V)
    at = torch.where(real, drafts, 0).unsqueeze(2)
    one = torch.zeros((B, K, V), dtype=torch.float64, device=logits.device).scatter_(2, at, 1.0)
    q = one if draft_logits is None else weights(draft_logits)
    passed = real & (u[:, :K].double() * q.gather(2, at)[..., 0] < p[:, :K].gather(2, at)[..., 0])
    accepted = passed.long().cumprod(1).sum(1)
    seq = torch.arange(B, device=logits.device)
    last = p[seq, accepted]
    tried = (accepted < K) & real[seq, accepted.clamp(max=K - 1)]
    rest = (last - torch.where(tried[:, None], q[seq, accepted.clamp(max=K - 1)], 0.0)).clamp(min=0.0)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, last)
    run = rest.cumsum(1)
    token = (run <= u[:, K:].double() * run[:, -1:]).sum(1)
    tokens = torch.cat([drafts, drafts[:, :1]], 1)
    tokens = torch.where(torch.arange(K + 1, device=logits.device) < accepted[:, None], tokens, -1)
    tokens[seq, accepted] = token
    return tokens, accepted.to(torch.int32)


def run(state):
    s = state
    if s["kind"] == "verify":
        a = (s["logits"], s["drafts"], s["u"], s["draft_logits"], s["temperature"])
        if own:
            from teenyformers_amd import ops
            return ops.verify_drafts(*a)
        return _plain_verify(*a)
    if s["kind"] == "copy":
        if own:
            from teenyformers_amd import ops
            return ops.copy_pages(s["pages"], s["src"], s["dst"])
        dev = s["pages"].device
        src, dst = torch.tensor(s["src"], device=dev), torch.tensor(s["dst"], device=dev)
        s["pages"][:, dst] = s["pages"][:, src]
        return s["pages"]
    if s["kind"] == "append":
        if own:
            from teenyformers_amd import ops
            q = ops.paged_qkv_rope_split(s["qkv"], s["k"], s["v"], s["table"], s["n_past"], s["Hq"], s["base"],
                                         starts=s["starts"])
            return q, s["k"], s["v"]
        return _plain_append(s)
    if own:
        from teenyformers_amd import ops
        return ops.paged_attention(s["q"], s["k"], s["v"], s["table"], s["n_past"], s["scale"], starts=s["starts"],
                                   max_new=s["max_new"], max_keys=s["max_keys"])
    return _plain_attn(s)


# ---------------------------------------------------------------------------
# from the definition, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] == "copy":
        return None
    s = prepare(case, seed)
    if case["kind"] == "verify":
        return _exact_verify(s)
    _, Hkv, page, D = s["k"].shape
    if case["kind"] == "append":
        Hq = s["Hq"]
        x = s["qkv"].view(-1, Hq + 2 * Hkv, D // 2, 2).cpu().double().numpy()
        q, k, v = np.empty((x.shape[0], Hq, D)), s["k"].double(), s["v"].double()
        rate = np.exp(-2.0 * math.log(s["base"]) / D * np.arange(D // 2))
        table, t = s["table"].cpu().numpy(), 0
        for b, (n, m) in enumerate(zip(s["past"], s["lens"])):
            at = np.arange(n, n + m)
            turn = np.exp(1j * (at[:, None] * rate))[:, None]
            z = x[t:t + m, :Hq + Hkv]
            z = (z[..., 0] + 1j * z[..., 1]) * turn
            z = np.stack([z.real, z.imag], -1).reshape(m, Hq + Hkv, D)
            q[t:t + m] = z[:, :Hq]
            page_of = torch.from_numpy(table[b, at // page].astype(np.int64)).to(k.device)
            row = torch.from_numpy(at % page).to(k.device)
            k[page_of, :, row] = torch.from_numpy(z[:, Hq:]).to(k.device)
            v[page_of, :, row] = torch.from_numpy(x[t:t + m, Hq + Hkv:].reshape(m, Hkv, D)).to(k.device)
            t += m
        return torch.from_numpy(q).to(k.device), k, v
    q = s["q"].double()
    out = torch.empty_like(q)
    G = q.shape[1] // Hkv
    t = 0
    for b, (n, m) in enumerate(zip(s["past"], s["lens"])):
        at = torch.arange(n + m, device=q.device)
        page_of, row = s["table"].long()[b, at // page], at % page
        seen = at[None, :] <= n + torch.arange(m, device=q.device)[:, None]
        for j in range(Hkv):
            keys, values = s["k"][page_of, j, row].double(), s["v"][page_of, j, row].double()
            for h in range(j * G, (j + 1) * G):
                score = torch.where(seen, q[t:t + m, h].mm(keys.t()) * s["scale"], -math.inf)
                out[t:t + m, h] = torch.softmax(score, 1).mm(values)
        t += m
    return out


def _exact_verify(s):
    B, n, V = s["logits"].shape
    K = n - 1
    drafts, u = s["drafts"].cpu().numpy(), s["u"].double().cpu().numpy()
    T = s["temperature"]
    T = T.double().cpu().numpy() if torch.is_tensor(T) else np.full(B, float(T))

    def probs(x, b):
        x = x.double().cpu().numpy()
        if T[b] <= 0:
            return np.eye(1, V, int(np.argmax(x)))[0]
        w = np.exp((x - x.max()) / T[b])
        return w / w.sum()

    tokens, accepted = np.full((B, n), -1, dtype=np.int64), np.zeros(B, dtype=np.int32)
    for b in range(B):
        rest = None
        for i in range(K):
            d = int(drafts[b, i])
            p = probs(s["logits"][b, i], b)
            if not 0 <= d < V:
                rest = p
                break
            q = np.eye(1, V, d)[0] if s["draft_logits"] is None else probs(s["draft_logits"][b, i], b)
            if u[b, i] * q[d] < p[d]:
                tokens[b, i] = d
                accepted[b] += 1
                continue
            rest = np.maximum(p - q, 0.0)
            rest = rest if rest.sum() > 0 else p
            break
        if rest is None:
            rest = probs(s["logits"][b, K], b)
        c = np.cumsum(rest)
        tokens[b, accepted[b]] = np.searchsorted(c, u[b, K] * c[-1], side="right")
    return torch.from_numpy(tokens), torch.from_numpy(accepted)
