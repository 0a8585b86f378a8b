"""ops.shared_prefix_attention against softmax attention over the concatenated
keys in 64 bits.

Bound per value, with A = sum_k p_k |v_k| (so |o| <= A) and u the half step of the
storage type (bf16 2^-8, fp32 2^-24):
  scores   a product of D terms in fp32 is off by at most (D + 2) 2^-24 sum |q k|;
           times scale this moves p by e_s relative at most; exp2 and its
           argument's rounding add 2^-21 + |s| 2^-23 (|s| <= sum |q k| scale)
  P        bf16: rounded to 2^-8 relative, in the numerator and in the sum
  sums     n terms in fp32: n 2^-24 relative each, numerator and denominator
  output   one rounding, u |o|
so |o - ref| <= A (2 (e_s + e_x + [2^-8]) + 2 n 2^-24) + u |ref|, and second-order
terms within 5 % of that."""
import math

import pytest
import torch

from teenyformers_amd import ops

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
NAN = float("nan")


def reference(q, kp, vp, k, v, n_prefix, past, scale):
    """[B, Hq, S, D] in 64 bits, and the bound of the doc string."""
    B, Hq, S, D = q.shape
    G, L = Hq // k.shape[1], k.shape[2]
    u = 2.0 ** -8 if q.dtype == BF else 2.0 ** -24
    out = torch.zeros((B, Hq, S, D), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for b in range(B):
        for s in range(S):
            n = max(0, min(past[b] + s + 1, L))
            if n + n_prefix == 0:
                continue
            K = torch.cat([kp[:, :n_prefix], k[b, :, :n]], 1).double().repeat_interleave(G, 0)
            V = torch.cat([vp[:, :n_prefix], v[b, :, :n]], 1).double().repeat_interleave(G, 0)
            x = q[b, :, s].double()
            sc = (K * x[:, None, :]).sum(2) * scale
            mag = (K.abs() * x[:, None, :].abs()).sum(2).amax(1) * abs(scale)
            p = torch.softmax(sc, 1)
            o = (p[:, :, None] * V).sum(1)
            A = (p[:, :, None] * V.abs()).sum(1)
            e = (D + 2) * 2.0 ** -24 * mag + 2.0 ** -21 + mag * 2.0 ** -23
            e = e + (2.0 ** -8 if q.dtype == BF else 0.0) + (n + n_prefix) * 2.0 ** -24
            out[b, :, s] = o
            tol[b, :, s] = 1.05 * (2 * e[:, None] * A + u * o.abs())
    return out, tol


def make(cuda, dtype, B, Hq, Hkv, S, D, P, L, seed=0, prefix_len=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    lp = prefix_len or max(P, 1)
    return [(1.5 * r(B, Hq, S, D)).to(dtype)] + [t.to(dtype) for t in (
        r(Hkv, lp, D), r(Hkv, lp, D), r(B, Hkv, L, D), r(B, Hkv, L, D))]


def spoil(t, past, S):
    """Rows that no query sees hold NaN."""
    for b, n in enumerate(past):
        t[b, :, max(0, n + S):] = NAN


def check(ts, P, past, S, scale=None, as_tensor=True, **kw):
    q, kp, vp, k, v = ts
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    want, tol = reference(q, kp, vp, k, v, P, past, scale)
    for t in (k, v):
        spoil(t, past, S)
    for t in (kp, vp):
        t[:, P:] = NAN
    n = torch.tensor(past, dtype=torch.int32, device="cuda") if as_tensor else past[0]
    got = ops.shared_prefix_attention(q, kp, vp, k, v, P, n, scale, **kw)
    assert got.shape == q.shape and got.dtype == q.dtype
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float((got.double() - want).abs().max()))
    rel = float((got.double() - want).norm() / want.norm().clamp_min(1e-30))
    assert rel <= (6e-3 if q.dtype == BF else 2e-6), rel
    return got


# (B, Hq, Hkv, S, D, prefix, cache, past of each sequence)
SHAPES = [
    (1, 1, 1, 1, 64, 1, 1, [0]),
    (1, 4, 4, 1, 128, 0, 40, [17]),
    (2, 8, 2, 1, 64, 33, 5, [0, 4]),
    (3, 8, 8, 1, 128, 31, 70, [0, 31, 69]),
    (4, 32, 8, 1, 128, 700, 300, [299, 0, 5, 128]),
    (17, 8, 2, 1, 64, 517, 64, [i * 3 for i in range(17)]),
    (33, 32, 8, 1, 128, 257, 40, [i for i in range(33)]),
    (70, 8, 1, 1, 64, 100, 33, [i % 33 for i in range(70)]),
    (1, 64, 1, 1, 128, 2049, 10, [3]),
    (2, 40, 1, 1, 64, 90, 130, [64, 129]),
    (3, 8, 2, 5, 128, 130, 101, [0, 31, 96]),
    (2, 4, 4, 9, 64, 1, 9, [0, 0]),
    (2, 8, 2, 33, 128, 65, 80, [0, 47]),
    (1, 4, 2, 130, 64, 259, 131, [1]),
    (9, 6, 2, 7, 64, 0, 50, [0, 1, 2, 3, 30, 31, 32, 33, 43]),
    # rows enough for the forward kernel (bf16): 128 workgroups of 128 rows and more
    (16, 32, 8, 17, 128, 70, 40, [i for i in range(16)]),
    (33, 16, 4, 33, 64, 0, 70, [i for i in range(33)]),
    (8, 64, 8, 40, 64, 129, 45, [5, 0, 1, 2, 3, 4, 5, 5]),
    (24, 24, 8, 50, 128, 33, 114, [0, 64] * 12),
    (4, 16, 16, 300, 64, 31, 364, [0, 64, 1, 31]),
]


# A longer cache (never read past its used rows) is what makes bf16 share few rows'
# keys out; short ones run the forward kernel over them.
LONGER = pytest.mark.parametrize("longer", [0, 3000], ids=["", "long"])


@LONGER
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=[str(s[:7]) for s in SHAPES])
def test_against_definition(cuda, dtype, shape, longer):
    B, Hq, Hkv, S, D, P, L, past = shape
    check(make(cuda, dtype, B, Hq, Hkv, S, D, P, L + longer, prefix_len=P + 3), P, past, S)


def test_both_ways_are_tested(cuda):
    """Of the shapes above, in bf16, some run the forward kernel and some share keys."""
    need = ops._lib.lib().teeny_shared_prefix_attention_workspace_bytes
    kinds = {(longer, need(B, Hq, Hkv, S, P, L + longer, D, 1) > 0)
             for B, Hq, Hkv, S, D, P, L, _ in SHAPES for longer in (0, 3000)}
    assert {(0, False), (3000, True), (3000, False)} <= kinds


@pytest.mark.parametrize("D", [8, 16, 32, 64, 128])
@pytest.mark.parametrize("P,L", [(45, 300), (20, 60), (0, 21)])
@pytest.mark.parametrize("S", [1, 4, 21])
def test_f32_head_dims(cuda, D, S, P, L):
    """Shares of the keys, and whole walks over few of them."""
    check(make(cuda, F32, 3, 6, 3, S, D, P, L), P, [0, 7 if L > 40 else 0, L - S], S)


@pytest.mark.parametrize("D", [32, 64, 128])
def test_f32_many_rows(cuda, D):
    """Whole walks because rows fill the device, over many keys."""
    past = [0, 3, 50, 31] * 8
    check(make(cuda, F32, 32, 16, 16, 32, D, 150, 90), 150, past, 32)


@LONGER
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("P", [31, 32, 33, 63, 64, 65, 95, 127, 128, 129, 1000])
def test_prefix_lengths(cuda, dtype, P, longer):
    check(make(cuda, dtype, 2, 8, 2, 1, 64, P, 34 + longer, seed=P), P, [0, 33], 1)


@LONGER
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("past", [0, 30, 31, 32, 62, 63, 64, 400, 2000])
def test_past_lengths(cuda, dtype, past, longer):
    """One length for all, given by the host and by one device value."""
    ts = make(cuda, dtype, 3, 8, 2, 1, 128, 40, past + 1 + longer, seed=past)
    a = check(ts, 40, [past] * 3, 1, as_tensor=False)
    one = torch.tensor([past], dtype=torch.int32, device="cuda")
    b = ops.shared_prefix_attention(*ts, 40, one)
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_rows_that_see_nothing_and_past_the_cache(cuda, dtype):
    """Device lengths that leave no key (zeros), some rows without a key, and rows
    past the cache's end (the whole cache); few rows, and as many as the forward
    kernel takes."""
    for B, Hkv, S, D, L in ((4, 2, 3, 64, 35), (4, 2, 3, 128, 3000), (4, 2, 40, 64, 3000),
                            (8, 16, 64, 128, 96)):
        q, kp, vp, k, v = make(cuda, dtype, B, 2 * Hkv, Hkv, S, D, 1, L)
        past = [-S, 1 - S, L, -100] * (B // 4)
        want, tol = reference(q, kp, vp, k, v, 0, past, 0.125)
        n = torch.tensor(past, dtype=torch.int32, device="cuda")
        got = ops.shared_prefix_attention(q, kp[:, :0], vp[:, :0], k, v, 0, n, 0.125)
        assert ((got.double() - want).abs() <= tol).all()
        assert (got[0] == 0).all() and (got[1, :, :-1] == 0).all() and (got[3] == 0).all()
        assert (got[1, :, -1] != 0).any()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_large_scores_and_offsets(cuda, dtype):
    """Scores far from zero, the largest in either part: one softmax over both
    (exponents past the forward kernel's 2^31 above its first tile among them)."""
    for B, Hkv, S, longer in ((3, 2, 1, 0), (3, 2, 1, 3000), (16, 16, 32, 0)):
        ts = make(cuda, dtype, B, 2 * Hkv, Hkv, S, 64, 90, 49 + S + longer)
        q, kp, vp, k, v = ts
        q.mul_(8.0)
        k[1] *= 3.0
        kp[0] *= 3.0
        check(ts, 90, [10, 49, 30, 3] * (B // 4) if B > 3 else [10, 49, 30], S)


@pytest.mark.parametrize("D", [64, 128])
@LONGER
@pytest.mark.parametrize("B,S", [(3, 1), (3, 3), (3, 40), (66, 40)])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_merged_layout(cuda, dtype, B, S, D, longer):
    ts = make(cuda, dtype, B, 8, 2, S, D, 77, 60 + longer)
    past = torch.tensor([0, 5, 60 - S] * (B // 3), dtype=torch.int32, device="cuda")
    a = ops.shared_prefix_attention(*ts, 77, past)
    b = ops.shared_prefix_attention(*ts, 77, past, merged=True)
    assert torch.equal(ops.merge_heads(a), b)
    if S == 1:
        c = ops.shared_prefix_attention(ts[0][:, :, 0].contiguous(), *ts[1:], 77, past)
        assert torch.equal(c, a[:, :, 0])


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_equals_attention_over_copies(cuda, dtype):
    """The prefix copied into every sequence's cache: what decode_attention gives."""
    B, Hq, Hkv, D, P, n = 5, 8, 2, 64, 333, 41
    ts = make(cuda, dtype, B, Hq, Hkv, 1, D, P, n)
    q, kp, vp, k, v = ts
    full = [torch.cat([p.expand(B, -1, -1, -1), c], 2).contiguous() for p, c in ((kp, k), (vp, v))]
    a = ops.decode_attention(q[:, :, 0].contiguous(), *full, P + n)
    b = ops.shared_prefix_attention(*ts, P, n - 1)[:, :, 0]
    bound = 4 * 2.0 ** -8 if dtype == BF else 1e-5  # two roundings of P and of o each
    assert (a.double() - b.double()).abs().max() <= bound * float(v.abs().max())


def test_prefix_from_a_one_sequence_cache(cuda):
    ts = make(cuda, BF, 4, 8, 2, 1, 128, 50, 20, prefix_len=64)
    a = ops.shared_prefix_attention(*ts, 50, 7)
    b = ops.shared_prefix_attention(ts[0], ts[1][None], ts[2][None], *ts[3:], 50, 7)
    assert torch.equal(a, b)


def test_offsets_past_32_bits(cuda):
    """Caches of more than 2^31 elements: the last sequence's rows."""
    B, Hkv, L, D = 9, 2, 1 << 20, 128
    k = torch.empty((B, Hkv, L, D), dtype=BF, device="cuda")
    v = torch.empty_like(k)
    assert k.numel() > 2 ** 31
    q, kp, vp, ko, vo = make(cuda, BF, 1, 4, Hkv, 1, D, 50, 300)
    past = [-1] * 8 + [299]
    k[8, :, :300], v[8, :, :300] = ko[0], vo[0]
    n = torch.tensor(past, dtype=torch.int32, device="cuda")
    got = ops.shared_prefix_attention(q.expand(B, -1, -1, -1).contiguous(), kp, vp, k, v, 50, n)
    want, tol = reference(q, kp, vp, ko, vo, 50, [299], 1 / math.sqrt(D))
    assert ((got[8:].double() - want).abs() <= tol).all()
    k[0, :, :300], v[0, :, :300] = ko[0], vo[0]
    k[0, :, L - 300:], v[0, :, L - 300:] = ko[0], vo[0]
    k[0, :, 300:L - 300] = 0
    v[0, :, 300:L - 300] = 0
    n[0] = L - 1
    got = ops.shared_prefix_attention(q.expand(B, -1, -1, -1).contiguous(), kp, vp, k, v, 50, n)
    # keys of zeros score 0 with value 0: softmax over all of them in closed form
    s = (torch.cat([kp, ko[0], ko[0]], 1).double().repeat_interleave(2, 0)
         * q[0].double()).sum(2) / math.sqrt(D)
    V = torch.cat([vp, vo[0], vo[0]], 1).double().repeat_interleave(2, 0)
    e = torch.exp(s)
    want = (e[:, :, None] * V).sum(1) / (e.sum(1, keepdim=True) + L - 600)
    A = (e[:, :, None] * V.abs()).sum(1) / (e.sum(1, keepdim=True) + L - 600)
    # (2^20 equal terms: sums of bf16 P in fp32 chains of at most 2^15 each)
    assert ((got[0, :, 0].double() - want).abs() <= A * (4 * 2.0 ** -8 + 2.0 ** -8)).all()


@LONGER
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_captured_and_replayed(cuda, dtype, longer):
    """The lengths are read at replay."""
    ts = make(cuda, dtype, 4, 8, 2, 1, 64, 300, 90 + longer)
    n = torch.zeros(4, dtype=torch.int32, device="cuda")
    out = torch.zeros_like(ts[0])
    ops.shared_prefix_attention(*ts, 300, n, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.shared_prefix_attention(*ts, 300, n, out=out)
    for i in range(4):
        n.copy_(torch.tensor([i, 20 * i, 89, 3], dtype=torch.int32))
        ts[0].normal_()
        g.replay()
        torch.cuda.synchronize()
        want = ops.shared_prefix_attention(*ts, 300, n)
        assert torch.equal(out, want)


def test_another_stream(cuda):
    ts = make(cuda, BF, 8, 32, 8, 1, 128, 2000, 90)
    want = ops.shared_prefix_attention(*ts, 2000, 50)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = ops.shared_prefix_attention(*ts, 2000, 50)
    s.synchronize()
    assert torch.equal(got, want)


def test_refusals(cuda):
    ts = make(cuda, BF, 2, 4, 2, 2, 64, 10, 20)
    q, kp, vp, k, v = ts
    f = ops.shared_prefix_attention
    for args in [(q, kp, vp, k, v, 11, 0), (q, kp, vp, k, v, -1, 0), (q, kp, vp, k, v, 10, 19),
                 (q, kp, vp, k, v, 10, -1), (q, kp[:1], vp[:1], k, v, 10, 0), (q, kp, vp[:, :5], k, v, 5, 0),
                 (q[0, 0], kp, vp, k, v, 10, 0), (q, kp, vp, k[:1], v[:1], 10, 0), (q.cpu(), kp, vp, k, v, 10, 0),
                 (q.transpose(1, 2), kp, vp, k, v, 10, 0), (q, kp, vp, k, v[..., :32], 10, 0)]:
        with pytest.raises(ValueError):
            f(*args)
    for args in [(q.float(), kp, vp, k, v, 10, 0), (q, kp, vp, k, v, 10, torch.zeros(2, device="cuda")),
                 (q, kp, vp, k, v, 10, torch.zeros(3, dtype=torch.int32, device="cuda")),
                 (q, kp, vp, k, v, 10, torch.zeros(2, dtype=torch.int32))]:
        with pytest.raises(TypeError):
            f(*args)
    with pytest.raises(ValueError):
        f(*ts, 10, 0, out=torch.empty_like(q).float())
    for kw in (dict(softmax_scale=0.0), dict(softmax_scale=NAN)):
        with pytest.raises(Exception, match="-7"):
            f(*ts, 10, 0, **kw)
    with pytest.raises(Exception, match="workspace"):
        f(*make(cuda, BF, 2, 4, 2, 2, 64, 10, 3000), 10, 0,
          workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))
    odd = torch.empty(q.numel() + 1, dtype=BF, device="cuda")[1:].view(q.shape)
    with pytest.raises(Exception, match="-7"):
        f(odd, kp, vp, k, v, 10, 0)


@pytest.mark.parametrize("S,P,L", [(5, 45, 300), (5, 20, 60), (40, 45, 300), (40, 0, 90)])
@pytest.mark.parametrize("D", [8, 32, 64, 128])
@pytest.mark.parametrize("G", [1, 3])
def test_f32_new_tokens_that_are_not_finite(cuda, G, D, S, P, L):
    """A new token's V of Inf, or K of NaN, reaches that token's row and later ones;
    earlier ones keep their values."""
    past = [17, 3]
    ts = make(cuda, F32, 2, 2 * G, 2, S, D, P, L)
    q, kp, vp, k, v = ts
    want, tol = reference(q, kp, vp, k, v, P, past, 0.25)
    t0, t1 = 2, S - 1
    v[0, :, past[0] + t0, 3] = float("inf")
    k[1, :, past[1] + t1] = NAN
    v[1, :, past[1] + t1] = NAN
    n = torch.tensor(past, dtype=torch.int32, device="cuda")
    got = ops.shared_prefix_attention(q, kp, vp, k, v, P, n, 0.25).double()
    others = [d for d in range(D) if d != 3]
    ok = (got - want).abs() <= tol
    assert ok[0, :, :t0].all() and ok[0][:, :, others].all() and ok[1, :, :t1].all()
    assert not torch.isfinite(got[0, :, t0, 3]).any() and torch.isnan(got[1, :, t1]).all()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_two_streams_at_once(cuda, dtype):
    """Calls in flight together, each with a workspace of its own."""
    shapes = [(8, 8, 2, 1, 64, 700, 3000), (4, 8, 2, 3, 128, 900, 3000)]
    ts = [make(cuda, dtype, *s, seed=i) for i, s in enumerate(shapes)]
    run = lambda i: ops.shared_prefix_attention(*ts[i], shapes[i][5], 900 + i)  # noqa: E731
    want = [run(0), run(1)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(run(i))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


# (type, new tokens, q heads, kv heads, D, cache rows past the new tokens, by shares)
NEGATIVE = [
    (BF, 300, 8, 2, 64, 0, False), (BF, 512, 4, 2, 128, 0, False),
    (BF, 300, 8, 2, 64, 9000, True), (BF, 512, 4, 2, 128, 9000, True), (BF, 1, 8, 2, 128, 3000, True),
    (F32, 300, 4, 2, 64, 0, True), (F32, 300, 16, 4, 64, 0, False), (F32, 1, 8, 2, 128, 0, True),
]


@pytest.mark.parametrize("P", [33, 1000])
@pytest.mark.parametrize("dtype,S,Hq,Hkv,D,more,shares", NEGATIVE, ids=[
    f"{'bf16' if c[0] == BF else 'f32'}-{c[1:]}" for c in NEGATIVE])
def test_negative_lengths_behind_a_prefix(cuda, dtype, S, Hq, Hkv, D, more, shares, P):
    """Device lengths below zero: rows that see the prefix alone, all of it, in each
    way that the call may run."""
    past = [-S, 1 - S, -100, -1, 0]
    L = S + more + (60 if S == 1 else 0)
    need = ops._lib.lib().teeny_shared_prefix_attention_workspace_bytes(
        len(past), Hq, Hkv, S, P, L, D, 1 if dtype == BF else 0)
    # (fp32: up to 128 keys are walked whole)
    assert (need > 0) == (shares and not (dtype == F32 and P + L <= 128))
    got = check(make(cuda, dtype, len(past), Hq, Hkv, S, D, P, L, prefix_len=P + 2), P, past, S)
    assert (got != 0).any(3).all()


def test_workspace_is_sized_on_the_device_of_the_launch(cuda, monkeypatch):
    """The shares go by the device's CUs, so both are asked of q's device."""
    from types import SimpleNamespace
    ts = make(cuda, BF, 2, 8, 2, 1, 64, 700, 3000)
    want = ops.shared_prefix_attention(*ts, 700, 50)
    on = []

    class Device:
        def __enter__(self):
            on.append(True)

        def __exit__(self, *a):
            on.clear()

    need, here = ops._lib.lib().teeny_shared_prefix_attention_workspace_bytes, []
    lib = SimpleNamespace(
        teeny_shared_prefix_attention_workspace_bytes=lambda *a: here.append(bool(on)) or need(*a))
    monkeypatch.setattr(ops, "_on_device_of", lambda t: Device())
    monkeypatch.setattr(ops, "_lib", SimpleNamespace(lib=lambda: lib))
    assert torch.equal(ops.shared_prefix_attention(*ts, 700, 50), want)
    assert here == [True]


# of each size: one token, a few, prompts; the keys' shares or a walk without them
REPEATED = [(BF, 16, 32, 8, 1, 128, 2048, 128, 101), (BF, 4, 32, 8, 1, 128, 32000, 320, 257),
            (BF, 32, 16, 16, 1, 64, 1021, 320, 300), (BF, 8, 32, 8, 5, 128, 3001, 128, 90),
            (BF, 8, 32, 8, 257, 128, 4096, 320, 0), (F32, 4, 4, 4, 1, 64, 61, 64, 8),
            (F32, 4, 8, 8, 3, 64, 700, 300, 200)]


@pytest.mark.parametrize("dtype,B,Hq,Hkv,S,D,P,L,past", REPEATED, ids=[str(c[1:]) for c in REPEATED])
def test_calls_repeat_themselves(cuda, dtype, B, Hq, Hkv, S, D, P, L, past):
    """The same bits each time: shares are merged in one order, without atomics."""
    ts = make(cuda, dtype, B, Hq, Hkv, S, D, P, L)
    want = ops.shared_prefix_attention(*ts, P, past)
    assert all(torch.equal(ops.shared_prefix_attention(*ts, P, past), want) for _ in range(10))
