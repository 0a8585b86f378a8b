"""ops.verify_drafts against its definition in 64 bits (numpy).

The outputs are whole numbers, equal to the definition's wherever that is decided by more
than the kernels' error.  A weight is fp32, 2^(x c - K): what rounds K is common to a row's
weights; c is rounded (2^-24 relative, so a weight d octaves down moves by d 2^-24 octaves) and
so is the fused exponent (|d| 2^-24): below 64 octaves, where a weight is under 2^-64, that is
2 * 64 * 2^-24 ln 2 < 6e-6 relative, and for a weight w at most 2 -log2(w) w 2^-24 ln 2 < 5e-8 of
the largest.  exp2 adds 2^-22 relative, sums of eight 2^-21, the scaled difference of two rows
3 2^-24.  So a probability is within 1e-6 relative plus 1e-7 of the largest, running sums of
them within 1.2e-6 of the whole, and a difference p - q within 2.4e-6: borders nearer than 5e-6
(relative to the sum drawn from) are left out."""
import math

import numpy as np
import pytest
import torch

from teenyformers_amd import ops

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
EDGE = 5e-6


def probs(x, T):
    """Probabilities of a row (no token with weight: zeros)."""
    x = np.where(np.isnan(x), -np.inf, x)
    m = x.max()
    if m == -np.inf:
        return np.zeros_like(x)
    if not T > 0:
        p = np.zeros_like(x)
        p[np.argmax(x)] = 1.0
        return p
    with np.errstate(invalid="ignore"):
        w = np.where(x == m, 1.0, np.where(x > -np.inf, np.exp((x - m) / T), 0.0))
    return w / w.sum()


def reference(logits, drafts, u, draft_logits, T):
    """(tokens, accepted, sure): sure is False where a border lies within EDGE."""
    x = logits.double().cpu().numpy()
    y = None if draft_logits is None else draft_logits.double().cpu().numpy()
    d, u = drafts.cpu().numpy(), u.double().cpu().numpy()
    B, n, V = x.shape
    T = np.broadcast_to(T.double().cpu().numpy() if torch.is_tensor(T) else float(T), B)
    tokens, accepted, sure = np.full((B, n), -1, dtype=np.int64), np.zeros(B, dtype=np.int32), np.ones(B, bool)
    for b in range(B):
        rest = None
        for i in range(n - 1):
            p = probs(x[b, i], T[b])
            if not 0 <= d[b, i] < V:
                rest = p
                break
            q = np.zeros(V)
            q[d[b, i]] = 1.0
            if y is not None:
                q = probs(y[b, i], T[b])
            pd, qd = p[d[b, i]], q[d[b, i]]
            # (a draft's own weights are formed in 64 bits, only the sums under them in 32: relative)
            if T[b] > 0 and pd != qd and abs(u[b, i] * qd - pd) <= EDGE * max(pd, qd):
                sure[b] = False
            if u[b, i] * qd < pd:
                tokens[b, i] = d[b, i]
                accepted[b] += 1
                continue
            rest = np.maximum(p - q, 0.0)
            if T[b] > 0 and 0 < rest.sum() < 1e-3:
                sure[b] = False  # (a difference of near equals)
            rest = rest if rest.sum() > 0 else p
            break
        if rest is None:
            rest = probs(x[b, n - 1], T[b])
        c = np.cumsum(rest)
        if c[-1] == 0:
            continue
        t = u[b, n - 1] * c[-1]
        at = min(int(np.searchsorted(c, t, side="right")), V - 1)
        near = min(abs(c[at] - t), abs(t - (c[at - 1] if at else -1.0)))
        if T[b] > 0 and near <= EDGE * c[-1] / min(1.0, max(rest.sum(), 1e-3)):
            sure[b] = False
        tokens[b, accepted[b]] = at
    return tokens, accepted, sure


def case(dtype, B, K, V, seed, with_q, noise=0.7, T=0.8, spread=1.3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rank = torch.rand((B, K + 1, V), generator=g, device="cuda").argsort(2)
    x = -spread * torch.log(rank + 1.0) + torch.randn((B, K + 1, V), generator=g, device="cuda") + 8.0
    y = x[:, :K] + noise * torch.randn((B, K, V), generator=g, device="cuda")
    x, y = x.to(dtype), y.to(dtype)
    t = torch.as_tensor(T, device="cuda").reshape(-1, 1, 1)
    gum = -torch.log(-torch.log(torch.rand((B, K, V), generator=g, device="cuda").clamp(1e-7, 1 - 1e-7)))
    drafts = (y.float() + (t * gum if with_q else 0.0)).argmax(2)
    u = torch.rand((B, K + 1), generator=g, device="cuda")
    return x, drafts, u, y if with_q else None


def check(x, drafts, u, y, T, least=0.9):
    tokens, accepted = ops.verify_drafts(x, drafts, u, y, T)
    want_t, want_a, sure = reference(x, drafts, u, y, T)
    assert sure.mean() >= least
    tokens, accepted = tokens.cpu().numpy(), accepted.cpu().numpy()
    assert np.array_equal(accepted[sure], want_a[sure])
    assert np.array_equal(tokens[sure], want_t[sure])
    return accepted


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("with_q", [False, True])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (3, 2, 7), (17, 4, 1000), (5, 8, 8191), (4, 3, 8193), (64, 1, 300),
                                   (2, 5, 50257), (3, 4, 128256), (2, 64, 500)])
def test_random(cuda, dtype, with_q, B, K, V):
    a = case(dtype, B, K, V, 7 * B + K + V, with_q)
    check(*a, 0.8, least=0.5 if B < 5 else 0.9)


@pytest.mark.parametrize("with_q", [False, True])
def test_temperatures(cuda, with_q):
    """One per sequence, greedy ones among them; a number; far ones."""
    g = torch.Generator(device="cuda").manual_seed(1)
    T = 0.3 + torch.rand(40, generator=g, device="cuda")
    T[::5] = 0.0
    a = case(F32, 40, 3, 3000, 5, with_q, T=T)
    check(*a, T)
    # at temperature 30 the two rows are nearly equal (what a refused draft leaves is 1 % of them,
    # over 3000 tokens): a border then lies within EDGE of most draws, and they are left out
    for t, least in ((0.0, 0.8), (0.05, 0.8), (1.0, 0.8), (30.0, 0.3)):
        check(*a, t, least=least)


def test_accepts_all_of_the_same_model(cuda):
    """q = p: every draft is accepted, whatever u below 1 is."""
    x, d, u, _ = case(BF, 30, 4, 5000, 3, True, noise=0.0)
    u[:, :4] = torch.tensor([0.0, 0.5, 1 - 2.0 ** -24, 0.999], device="cuda")
    tokens, accepted = ops.verify_drafts(x, d, u, x[:, :4], 0.8)
    assert (accepted == 4).all() and torch.equal(tokens[:, :4], d)


def test_greedy(cuda):
    """Drafts are accepted while they are the target's first choice, the lowest index of equal ones."""
    x, d, u, y = case(BF, 50, 4, 300, 3, False, noise=0.3)
    x = (x * 2).round() / 2  # equal maxima
    best = x.float().argmax(2)
    best = (x == x.amax(2, keepdim=True)).int().argmax(2)
    d = torch.where(torch.rand(50, 4, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0)) < 0.7,
                    best[:, :4], d)
    for q in (None, y):
        tokens, accepted = ops.verify_drafts(x, d, u, x[:, :4].contiguous() if q is not None else None, 0.0)
        n = (d == best[:, :4]).int().cumprod(1).sum(1)
        if q is None:
            assert torch.equal(accepted.long(), n)
        assert torch.equal(tokens.gather(1, accepted.long()[:, None]), best.gather(1, accepted.long()[:, None]))


@pytest.mark.parametrize("with_q", [False, True])
def test_drafts_that_are_none(cuda, with_q):
    x, d, u, y = case(BF, 24, 5, 999, 9, with_q, noise=0.05)
    d[0] = -1
    d[1, 2:] = -1
    d[2, 1] = 999          # past the vocabulary: ends the sequence's drafts
    d[3, 0] = 2 ** 40
    d[4, 4] = -2 ** 40
    x[1, 3:] = float("nan")  # behind the last real draft: not read
    accepted = check(x, d, u, y, 0.8)
    assert accepted[0] == 0 and accepted[1] <= 2 and accepted[2] <= 1 and accepted[3] == 0


def test_masked_logits(cuda):
    """-inf, the type's lowest values, NaN and +inf among the logits; rows without a token."""
    for dtype in (F32, BF):
        x, d, u, y = case(dtype, 32, 3, 700, 11, True)
        low = torch.finfo(dtype).min
        x[:8, :, ::2] = -math.inf
        x[8:12, :, 1::2] = low
        x[12:14, :, 5] = float("nan")
        x[14, 1] = -math.inf
        x[15] = -math.inf
        y[16:18, :, ::3] = -math.inf
        y[18] = -math.inf
        x[19, 0, 44] = math.inf
        y[20, 0, 44] = math.inf
        d[20, 0] = 44
        check(x, d, u, y, 0.8)
        check(x, d, u, None, 0.8)
        tokens, accepted = ops.verify_drafts(x, d, u, y, 0.8)
        assert accepted[15] == 0 and tokens[15, 0] == -1


def test_equal_logits_split_exactly(cuda):
    """Borders of equal weights lie where the definition has them."""
    V, B = 10, 11
    x = torch.zeros((B, 2, V), dtype=F32, device="cuda")
    d = torch.full((B, 1), 3, dtype=torch.int64, device="cuda")
    u = torch.zeros((B, 2), device="cuda")
    u[:, 1] = torch.arange(B, device="cuda") / 16.0
    tokens, accepted = ops.verify_drafts(x, d, u, None, 1.0)  # accepted (u = 0): from p_1
    assert (accepted == 1).all() and torch.equal(tokens[:, 1], (u[:, 1] * V).floor().long())
    d[:] = -1
    tokens, _ = ops.verify_drafts(x, d, u, None, 1.0)
    assert torch.equal(tokens[:, 0], (u[:, 1] * V).floor().long())
    d[:] = 3
    u[:, 0] = 0.5  # refused: of the nine others
    tokens, accepted = ops.verify_drafts(x, d, u, None, 1.0)
    want = (u[:, 1] * 9).floor().long()
    assert (accepted == 0).all() and torch.equal(tokens[:, 0], want + (want >= 3))


def test_rows_that_lie_apart(cuda):
    """Logits cut from padded products, at odd offsets."""
    for dtype in (F32, BF):
        x, d, u, y = case(dtype, 6, 3, 2500, 2, True)
        want = ops.verify_drafts(x, d, u, y, 0.8)
        for pad, off in ((63, 0), (9, 3), (64, 8)):
            big = torch.full((6, 5, 2500 + pad), 1e4, dtype=dtype, device="cuda")
            bigq = torch.full((6, 4, 2500 + 2 * pad), 1e4, dtype=dtype, device="cuda")
            big[:, :4, off:off + 2500] = x
            bigq[:, :3, 1:2501] = y
            got = ops.verify_drafts(big[:, :4, off:off + 2500], d, u, bigq[:, :3, 1:2501], 0.8)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    x1, d1, u1, y1 = case(BF, 2, 1, 100, 4, True)
    same = x1[:1].expand(2, -1, -1)  # one target row for all
    check(same, d1, u1, y1, 0.8, least=0.5)


def test_distribution(cuda):
    """The drawn tokens are the target's: 40000 sequences of one draft, frequencies of the first
    token within 5 standard deviations."""
    B, V = 40000, 6
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.tensor([1.0, 0.2, -0.5, 2.0, -1.0, 0.0], device="cuda").expand(B, 2, V).contiguous()
    y = torch.tensor([0.0, 1.5, 0.5, 0.1, 0.3, -2.0], device="cuda").expand(B, 1, V).contiguous()
    d = torch.multinomial(torch.softmax(y[0, 0], 0).expand(B, V), 1, generator=g)
    u = torch.rand((B, 2), generator=g, device="cuda")
    p = torch.softmax(x[0, 0].double(), 0)
    for i in range(0, B, 16000):
        s = slice(i, i + 16000)
        t, a = ops.verify_drafts(x[s], d[s], u[s], y[s], 1.0)
        n = t.shape[0]
        f = torch.bincount(t[:, 0], minlength=V).double() / n
        assert ((f - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all()
        assert ((t[:, 0] == d[s, 0]) == (a == 1)).logical_or(a == 0).all()


def test_captured_and_replayed(cuda):
    x, d, u, y = case(BF, 8, 4, 4000, 1, True)
    T = torch.full((8,), 0.8, device="cuda")
    out = ops.verify_drafts(x, d, u, y, T)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        ops.verify_drafts(x, d, u, y, T, tokens=out[0], accepted=out[1])
    for seed in range(2, 6):
        for mine, new in zip((x, d, u, y), case(BF, 8, 4, 4000, seed, True)):
            mine.copy_(new)
        T.fill_(0.4 * seed)
        out[0].fill_(-7)
        gr.replay()
        want = ops.verify_drafts(x, d, u, y, T)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_two_streams(cuda):
    a, b = case(BF, 8, 4, 60000, 1, True), case(BF, 16, 2, 9000, 2, False)
    want = ops.verify_drafts(*a, 0.8), ops.verify_drafts(*b, 0.8)
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(8):
        with torch.cuda.stream(s):
            got.append((ops.verify_drafts(*a, 0.8), 0))
        with torch.cuda.stream(t):
            got.append((ops.verify_drafts(*b, 0.8), 1))
    torch.cuda.synchronize()
    for r, i in got:
        assert torch.equal(r[0], want[i][0]) and torch.equal(r[1], want[i][1])


def test_refusals(cuda):
    x, d, u, y = case(BF, 3, 2, 50, 1, True)
    for a in ((x[0], d, u, y), (x[:, :1], d, u, y), (x, d.int(), u, y), (x, d[:, :1], u, y), (x, d, u[:, :2], y),
              (x, d, u.double(), y), (x, d, u, y[:, :1]), (x, d.cpu(), u, y), (x, d, u, y.cpu()),
              (x.cpu(), d, u, y), (x, d, u, y, -0.1), (x, d, u, y, float("nan")), (x, d, u, y, torch.ones(3)),
              (x, d, u, y, torch.ones(2, device="cuda"))):
        with pytest.raises(ValueError):
            ops.verify_drafts(*a)
    for a in ((x.half(), d, u), (x, d, u, y.float())):
        with pytest.raises(TypeError):
            ops.verify_drafts(*a)
    with pytest.raises(ValueError):
        ops.verify_drafts(x, d, u, y, 0.8, tokens=torch.empty((3, 2), dtype=torch.int64, device="cuda"))
    from teenyformers_amd._lib import TeenyError
    with pytest.raises(TeenyError):
        ops.verify_drafts(x, d, u, y, 0.8, workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))
    n = 65
    with pytest.raises(TeenyError):
        ops.verify_drafts(torch.zeros((1, n + 1, 8), device="cuda"), torch.zeros((1, n), dtype=torch.int64, device="cuda"),
                          torch.zeros((1, n + 1), device="cuda"))
    t, a = ops.verify_drafts(x[:0], d[:0], u[:0], y[:0])
    assert t.shape == (0, 3) and a.shape == (0,)


def test_extreme_temperatures_and_logits(cuda):
    """Factors and logits whose product is past fp32: the largest logit and its equals share the
    draw, as in the limit."""
    x, d, u, y = case(F32, 16, 2, 300, 6, True)
    x[8:, :, 7] = x[8:].amax(2)          # two equal maxima (at most; 7 may be one)
    best = x == x.amax(2, keepdim=True)
    for T in (1e-36, 1e-40, 1e-44):
        tokens, accepted = ops.verify_drafts(x, d, u, None, T)
        for b in range(16):
            n = int(accepted[b])
            assert best[b, n, tokens[b, n]] or (n < 2 and not best[b, n, d[b, n]])
            assert best[b, n, tokens[b, n]]
            for i in range(n):
                assert best[b, i, d[b, i]]
    low = torch.finfo(F32).min
    z = torch.full((4, 2, 100), low, device="cuda")
    z[1, :, 40] = 3e38
    z[2, :, 10:12] = 1e38
    z[3] = 0.0
    drafts = torch.full((4, 1), -1, dtype=torch.int64, device="cuda")
    uu = torch.tensor([[0.5, 0.5]] * 4, device="cuda")
    tokens, _ = ops.verify_drafts(z, drafts, uu, None, 0.25)
    assert tokens[:, 0].tolist() == [50, 40, 11, 50]
    tokens, _ = ops.verify_drafts(z, drafts, uu, None, math.inf)
    assert tokens[3, 0] == 50


def outcomes(x, d, u, y, T):
    """One sequence: {accepted: the tokens that may be drawn there} for weights off by the derived
    error: acceptance within EDGE relative, a running sum within EDGE of the whole.  Greedy: exact."""
    n, V = x.shape
    may, edge = {}, EDGE if T > 0 else 0.0

    def draw(at, w, rest, but=-1):
        c = np.cumsum(rest)
        before = np.concatenate([[0.0], c[:-1]])
        t = u[n - 1] * c[-1]
        ok = (c > t - edge) & (before <= t + edge) & (w > 0)
        if not T > 0:
            ok = rest > 0
        ok[[i for i in (but,) if i >= 0]] = False
        may.setdefault(at, set()).update(np.nonzero(ok)[0].tolist() if c[-1] > 0 or ok.any() else [-1])

    for i in range(n - 1):
        p = probs(x[i], T)
        if not 0 <= d[i] < V:
            draw(i, p, p)
            return may
        q = np.zeros(V)
        q[d[i]] = 1.0
        if y is not None:
            q = probs(y[i], T)
        pd, qd = p[d[i]], q[d[i]]
        slack = edge * max(pd, qd) if pd != qd else 0.0
        if not u[i] * qd < pd - slack:  # may be refused
            rest = np.maximum(p - q, 0.0)
            if rest.sum() > 0:
                draw(i, np.where(p > 0, 1.0, 0.0), rest, d[i])
            if rest.sum() <= edge:
                draw(i, p, p)
        if not u[i] * qd < pd + slack:  # must be
            return may
    p = probs(x[n - 1], T)
    draw(n - 1, p, p)
    return may


def check_every_row(x, drafts, u, y, T):
    tokens, accepted = ops.verify_drafts(x, drafts, u, y, T)
    tokens, accepted = tokens.cpu().numpy(), accepted.cpu().numpy()
    x, d, un = x.double().cpu().numpy(), drafts.cpu().numpy(), u.double().cpu().numpy()
    y = None if y is None else y.double().cpu().numpy()
    T = np.broadcast_to(T.double().cpu().numpy() if torch.is_tensor(T) else float(T), len(x))
    for b in range(len(x)):
        may, n = outcomes(x[b], d[b], un[b], None if y is None else y[b], T[b]), int(accepted[b])
        assert n in may, (b, n, sorted(may))
        assert tokens[b, n] in may[n], (b, n, tokens[b, n], sorted(may[n])[:8])
        assert (tokens[b, :n] == d[b, :n]).all() and (tokens[b, n + 1:] == -1).all()
        assert (d[b, :n] >= 0).all()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("with_q", [False, True])
@pytest.mark.parametrize("T", [0.0, 0.05, 0.8, 30.0])
def test_every_row_is_the_definition_within_the_error(cuda, dtype, with_q, T):
    """No sequence is left out: those next to a border have one of the outcomes beside it."""
    for B, K, V in ((1, 1, 1), (40, 3, 3000), (60, 1, 300), (4, 2, 8193), (3, 5, 50257), (2, 64, 500)):
        check_every_row(*case(dtype, B, K, V, 3 * B + V, with_q, T=max(T, 0.3)), T)
    x, d, u, y = case(dtype, 32, 3, 700, 12, with_q)
    x[:8, :, ::2] = -math.inf
    x[8:10, 1] = -math.inf
    x[10:12, :, 5] = float("nan")
    d[12:15, 1] = -1
    d[15, 0] = 700
    if with_q:
        y[16:20, :, ::3] = -math.inf
        y[20:24] = x[20:24, :3]  # nearly every draft accepted
    check_every_row(x, d, u, y, T)
