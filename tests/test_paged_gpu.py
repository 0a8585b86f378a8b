"""A cache in pages on the GPU: ops.paged_qkv_rope_split, ops.paged_attention and
ops.copy_pages against their definitions in 64 bits.

Bound of an attention value, with A = sum_k p_k |v_k| and u the half step of the
storage type (bf16 2^-8, fp32 2^-24):
  scores   a product of D terms in fp32 is off by at most (D + 2) 2^-24 sum |q k|;
           times scale this moves p by e_s relative at most; exp2 and its
           argument's rounding add 2^-21 + |s| 2^-23 (|s| <= sum |q k| scale)
  P        bf16: rounded to 2^-8 relative, in the numerator and in the sum
  sums     n terms in fp32: n 2^-24 relative each, numerator and denominator
  output   one rounding, u |o|
so |o - ref| <= A (2 (e_s + e_x + [2^-8]) + 2 n 2^-24) + u |ref|, and second-order
terms within 5 % of that.

Bound of a rotated value x0 c - x1 s: c and s are within 2^-23 of theirs (an angle in 64
bits, one rounding each, and the angle's own error, far below), each product and the
difference rounds once in fp32, and the output once: 4 2^-24 (|x0| + |x1|) + u |ref|."""
import math

import pytest
import torch

from teenyformers_amd import ops

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


def half_step(dtype):
    return 2.0 ** -8 if dtype == BF else 2.0 ** -24


class Batch:
    """Sequences of past[b] keys and lens[b] new tokens over a pool whose pages are in a
    random order.  fill: what every row holds that is not a key of a sequence."""

    def __init__(self, dtype, Hq, Hkv, D, page, past, lens, seed=0, extra=0, fill=NAN, width=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.g, self.dtype, self.past, self.lens, self.page = g, dtype, past, lens, page
        need = [max(0, -(-(n + m) // page)) for n, m in zip(past, lens)]
        n_pages = sum(need) + 2
        order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
        width = width or max(1, max(need))
        table = torch.full((len(past), width), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            table[b, :n] = torch.tensor(order[:n], dtype=torch.int32)
            order = order[n:]
        self.table = table.cuda()
        shape = (n_pages, Hkv, page, D)
        self.k = torch.full(shape, fill, dtype=dtype, device="cuda")
        self.v = torch.full(shape, fill, dtype=dtype, device="cuda")
        for b, (n, m) in enumerate(zip(past, lens)):
            for j in range(need[b]):
                rows = min(page, n + m - j * page)
                for t in (self.k, self.v):
                    t[table[b, j], :, :rows] = self.rnd(Hkv, rows, D)
        self.T = sum(lens) + extra
        self.q = (1.5 * self.rnd(self.T, Hq, D).float()).to(dtype)
        starts = [0]
        for m in lens:
            starts.append(starts[-1] + m)
        self.starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.n_past = torch.tensor(past, dtype=torch.int32, device="cuda")

    def rnd(self, *shape):
        return torch.randn(shape, generator=self.g, device="cuda").to(self.dtype)

    def keys(self, b, n):
        """K and V [Hkv, n, D] of the first n keys, and which are present."""
        at = torch.arange(n, device="cuda")
        pages = self.table[b].long()[at // self.page]
        there = (pages >= 0) & (pages < self.k.shape[0])
        pages = torch.where(there, pages, 0)
        return [t[pages, :, at % self.page].transpose(0, 1) for t in (self.k, self.v)] + [there]

    def run(self, **kw):
        kw.setdefault("starts", self.starts)
        return ops.paged_attention(self.q, self.k, self.v, self.table, self.n_past, **kw)

    def reference(self, scale=None):
        T, Hq, D = self.q.shape
        Hkv = self.k.shape[1]
        G = Hq // Hkv
        scale = 1.0 / math.sqrt(D) if scale is None else scale
        u = half_step(self.dtype)
        out = torch.zeros((T, Hq, D), dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(out)
        t0 = 0
        cap = self.table.shape[1] * self.page
        for b, (past, m) in enumerate(zip(self.past, self.lens)):
            for i in range(m):
                n = max(0, min(past + i + 1, cap))
                K, V, there = self.keys(b, n)
                K, V = K[:, there].double(), V[:, there].double()
                n = K.shape[1]
                if n == 0:
                    continue
                x = self.q[t0 + i].double().view(Hkv, G, D)
                sc = torch.matmul(x, K.transpose(1, 2).contiguous()) * scale
                mag = torch.matmul(x.abs(), K.abs().transpose(1, 2).contiguous()).amax(2) * abs(scale)
                p = torch.softmax(sc, 2)
                o = torch.matmul(p, V)
                A = torch.matmul(p, V.abs())
                e = (D + 2) * 2.0 ** -24 * mag + 2.0 ** -21 + mag * 2.0 ** -23
                e = e + (2.0 ** -8 if self.dtype == BF else 0.0) + n * 2.0 ** -24
                out[t0 + i] = o.reshape(Hq, D)
                tol[t0 + i] = (1.05 * (2 * e[..., None] * A + u * o.abs())).reshape(Hq, D)
            t0 += m
        return out, tol

    def check(self, got, scale=None):
        ref, tol = self.reference(scale)
        n = sum(self.lens)
        bad = ~((got[:n].double() - ref[:n]).abs() <= tol[:n])
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(),
                               (got[:n].double() - ref[:n])[bad][:4], tol[:n][bad][:4])


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,Hq,Hkv,D", [
    (F32, 4, 4, 64), (F32, 2, 1, 8), (F32, 3, 1, 16), (F32, 8, 2, 32), (F32, 8, 4, 128),
    (BF, 8, 2, 128), (BF, 4, 4, 64), (BF, 16, 2, 64), (BF, 5, 1, 128), (BF, 40, 1, 128)])
@pytest.mark.parametrize("page", [16, 32, 128])
def test_attention_ragged(cuda, dtype, Hq, Hkv, D, page):
    past = [0, 1, 15, 16, 31, 63, 200, 517, 0]
    lens = [1, 1, 2, 1, 5, 1, 3, 1, 40]
    c = Batch(dtype, Hq, Hkv, D, page, past, lens, seed=page)
    c.check(c.run())
    c.check(c.run(max_new=40, max_keys=520))


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("S,past", [(1, [700]), (1, [4095, 4096, 5000, 0]), (5, [3001, 2, 90]),
                                    (33, [129, 700]), (130, [0, 1000])])
def test_attention_uniform(cuda, dtype, S, past):
    c = Batch(dtype, 8, 2, 64, 16, past, [S] * len(past), seed=S)
    c.check(c.run(starts=None, max_keys=max(past) + S))
    c.check(c.run(starts=None))


@pytest.mark.parametrize("dtype,D", [(F32, 64), (BF, 128), (BF, 64)])
def test_attention_chunk_among_steps(cuda, dtype, D):
    """A long prompt's chunk, sequences of one token, and some without a new one."""
    past = [40, 300, 1111, 7, 0, 513]
    lens = [1, 0, 421, 1, 0, 7]
    c = Batch(dtype, 8, 2, D, 32, past, lens)
    c.check(c.run(max_new=421, max_keys=1600))


@pytest.mark.parametrize("dtype", [F32, BF])
def test_attention_rows_behind_the_last_sequence(cuda, dtype):
    c = Batch(dtype, 4, 2, 64, 16, [20, 5, 300], [1, 40, 2], extra=9)
    out = torch.full_like(c.q, 7.0)
    got = c.run(out=out)
    assert got is out
    c.check(got)
    assert (got[43:] == 7.0).all()


@pytest.mark.parametrize("dtype", [F32, BF])
def test_attention_absent_pages(cuda, dtype):
    """Pages given back behind a window, entries past the pool, a sequence without any."""
    past, lens = [300, 300, 50, 2000], [1, 70, 3, 1]
    c = Batch(dtype, 8, 2, 64, 16, past, lens)
    c.table[0, 0:7] = -1
    c.table[1, 3] = c.k.shape[0]
    c.table[1, 18:] = 2 ** 31 - 1  # of new tokens too
    c.table[2] = -5
    c.table[3, ::2] = -1
    got = c.run()
    c.check(got)
    assert (got[71:74] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_attention_later_tokens_have_no_influence(cuda, dtype, where, bad):
    """A new token whose key or value is not finite: tokens before it do not see it."""
    for lens, at in (([6, 3], 4), ([90, 70], 50)):
        c = Batch(dtype, 8, 2, 128, 16, [30, 500], lens)
        ref, (o, tol) = c.run(), c.reference()
        pos = c.past[0] + at
        getattr(c, where)[c.table[0, pos // 16], 1, pos % 16] = bad
        got = c.run()
        assert ((got[:at].double() - o[:at]).abs() <= tol[:at]).all()  # before it
        assert torch.equal(got[:, :4], ref[:, :4])                 # other heads
        assert torch.equal(got[lens[0]:], ref[lens[0]:])           # the other sequence
        assert not got[at:lens[0], 4:].isfinite().all()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("Hkv", [1, 2, 3, 4, 6, 8, 12, 16, 24])
def test_kv_heads(cuda, dtype, Hkv):
    """Every way of dealing kv heads to the caches' parts of the device: a long sequence among short
    ones, its keys in one share or several."""
    for past, lens in (([150, 0, 700], [1, 300, 2]), ([2500, 40], [130, 1])):
        c = Batch(dtype, 2 * Hkv, Hkv, 64, 16, past, lens, seed=Hkv)
        c.check(c.run(max_new=max(lens), max_keys=max(n + m for n, m in zip(past, lens))))
        c.check(c.run())


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("page", [64, 256, 512, 1024])
def test_page_sizes(cuda, dtype, page):
    """Few rows, rows enough for the forward's walk, and keys written by the split, in large pages."""
    c = Batch(dtype, 8, 2, 64, page, [2 * page - 1, page, 0, 700], [1, 3, 2, 1], seed=page)
    c.check(c.run())
    c = Batch(dtype, 8, 2, 64, page, [2 * page - 1, 0, 700], [60, 20, 1], seed=page)
    c.check(c.run())
    qkv = c.rnd(c.T, (8 + 2 * 2) * 64)
    ops.paged_qkv_rope_split(qkv, c.k, c.v, c.table, c.n_past, 8, 1e4, starts=c.starts)
    want, t = qkv.view(c.T, 12, 64)[:, 10:], 0
    for b, (past, m) in enumerate(zip(c.past, c.lens)):
        V = c.keys(b, past + m)[1]
        assert torch.equal(V[:, past:].transpose(0, 1), want[t:t + m])
        t += m
    c.check(c.run())


def test_attention_lowest_scores(cuda):
    """Rows whose scores lie far below zero, and keys of the type's lowest values."""
    for dtype in (F32, BF):
        c = Batch(dtype, 4, 1, 64, 16, [100, 33], [40, 1])
        c.k.copy_(torch.where(c.k.isnan(), c.k, -(c.k.abs() + 1)))
        c.q.copy_(c.q.abs() * 20 + 10)
        c.check(c.run())


def test_attention_far_offsets(cuda):
    """Pools past 2^32 bytes and 2^31 elements."""
    n_pages, Hkv, page, D = 17000, 8, 128, 128
    k = torch.empty((n_pages, Hkv, page, D), dtype=BF, device="cuda")
    v = torch.empty_like(k)
    assert k.numel() > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(1)
    c = Batch(BF, 16, Hkv, D, page, [200, 130], [1, 50])
    pages = [n_pages - 1, 5, n_pages - 2, n_pages - 3]
    table = torch.full((2, 2), -1, dtype=torch.int32)
    for b in range(2):
        for j in range(2):
            table[b, j] = pages[2 * b + j]
            k[pages[2 * b + j]] = torch.randn((Hkv, page, D), generator=g, device="cuda").to(BF)
            v[pages[2 * b + j]] = torch.randn((Hkv, page, D), generator=g, device="cuda").to(BF)
    c.k, c.v, c.table = k, v, table.cuda()
    c.check(c.run())


def test_attention_table_of_a_larger_one(cuda):
    """The rows of a table that lie apart."""
    c = Batch(BF, 8, 2, 128, 16, [100, 40, 9], [1, 1, 1])
    big = torch.full((3, 50), 10 ** 6, dtype=torch.int32, device="cuda")
    big[:, :c.table.shape[1]] = c.table
    want = c.run(max_keys=128)
    c.table = big[:, :c.table.shape[1]]
    assert torch.equal(c.run(max_keys=128), want)


def test_attention_shares_pages(cuda):
    """Sequences that go on from the same pages, and one page twice in a table."""
    c = Batch(BF, 8, 2, 64, 16, [64, 64, 40], [1, 1, 1])
    c.table[1, :4] = c.table[0, :4]
    c.table[2, 1] = c.table[2, 0]
    c.check(c.run())


def test_attention_captured_and_replayed(cuda):
    """A captured call reads the table, lengths and starts of each replay."""
    for past, lens in (([40, 3000, 9, 100], [1, 1, 1, 1]), ([500, 3000, 9, 100], [60, 1, 1, 5])):
        c = Batch(BF, 8, 2, 128, 16, past, lens, width=256)
        out = torch.empty_like(c.q)
        c.run(out=out)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            c.run(out=out)
        for seed in range(1, 4):
            d = Batch(BF, 8, 2, 128, 16, [n // seed for n in past], lens, seed=seed, width=256)
            c.q.copy_(d.q)
            for mine, other in ((c.k, d.k), (c.v, d.v)):
                mine[:other.shape[0]].copy_(other[:mine.shape[0]])
            c.table.copy_(d.table)
            c.n_past.copy_(d.n_past)
            c.past = d.past
            out.fill_(NAN)
            gr.replay()
            want = c.run()
            assert torch.equal(out, want)
            c.check(out)


def test_attention_two_streams(cuda):
    c = Batch(BF, 8, 2, 128, 16, [3000, 40, 9000], [1, 1, 1])
    d = Batch(BF, 8, 2, 128, 16, [2000, 4000], [70, 1], seed=5)
    want = c.run(), d.run()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(8):
        with torch.cuda.stream(a):
            got.append((c.run(), 0))
        with torch.cuda.stream(b):
            got.append((d.run(), 1))
    torch.cuda.synchronize()
    for x, i in got:
        assert torch.equal(x, want[i])


# ---------------------------------------------------------------------------
# the writer
# ---------------------------------------------------------------------------
def rotated(x, pos, base):
    """x [T, H, D] rotated in 64 bits, and the bound."""
    D = x.shape[2]
    inv = torch.exp(-2.0 * math.log(base) / D * torch.arange(D // 2, dtype=torch.float64, device="cuda"))
    a = (pos.double()[:, None] * inv)[:, None]
    c, s = torch.cos(a), torch.sin(a)
    x0, x1 = x[..., 0::2].double(), x[..., 1::2].double()
    y = torch.stack([x0 * c - x1 * s, x0 * s + x1 * c], 3).reshape(x.shape)
    e = (x0.abs() + x1.abs()).repeat_interleave(2, dim=2)
    return y, 4 * 2.0 ** -24 * e + half_step(x.dtype) * y.abs()


@pytest.mark.parametrize("dtype,Hq,Hkv,D", [(F32, 4, 4, 64), (F32, 2, 1, 8), (F32, 6, 2, 128),
                                            (BF, 8, 2, 128), (BF, 4, 4, 64), (BF, 32, 8, 128)])
@pytest.mark.parametrize("past,lens,page", [
    ([0, 5, 15, 16, 100000], [1, 1, 1, 1, 1], 16), ([3, 40, 0, 7], [130, 0, 1, 17], 32),
    ([30000, 9], [1100, 3], 64)])
def test_split(cuda, dtype, Hq, Hkv, D, past, lens, page):
    c = Batch(dtype, Hq, Hkv, D, page, past, [n + 1 for n in lens], extra=0)  # a spare row each
    c.starts = torch.tensor([0] + [sum(lens[:i + 1]) for i in range(len(lens))], dtype=torch.int32,
                            device="cuda")
    T = sum(lens) + 2  # two behind the last
    qkv = c.rnd(T, (Hq + 2 * Hkv) * D)
    before = c.k.clone(), c.v.clone()
    q = torch.full((T, Hq, D), 7.0, dtype=dtype, device="cuda")
    got = ops.paged_qkv_rope_split(qkv, c.k, c.v, c.table, c.n_past, Hq, 5e5, starts=c.starts,
                                   q_out=q)
    assert got is q and (q[T - 2:] == 7.0).all()
    x = qkv[:T - 2].view(-1, Hq + 2 * Hkv, D)
    pos = torch.cat([torch.arange(n, n + m) for n, m in zip(past, lens)]).cuda()
    seq = torch.cat([torch.full((m,), b) for b, m in enumerate(lens)]).cuda()
    y, tol = rotated(x[:, :Hq + Hkv], pos, 5e5)
    assert ((q[:T - 2].double() - y[:, :Hq]).abs() <= tol[:, :Hq]).all()
    at = c.table[seq, pos // page].long()
    assert ((c.k[at, :, pos % page].double() - y[:, Hq:]).abs() <= tol[:, Hq:]).all()
    assert torch.equal(c.v[at, :, pos % page], x[:, Hq + Hkv:])
    for now, then in zip((c.k, c.v), before):  # nothing else was written
        now[at, :, pos % page] = then[at, :, pos % page]
        assert torch.equal(now.nan_to_num(1.0), then.nan_to_num(1.0))


def test_split_near_positions_as_the_other_splits(cuda):
    """Up to a few hundred positions the angles of 32 and 64 bits give the same bf16 but for
    values next to a rounding border; the values themselves are equal in fp32 within the
    angle's error."""
    Hq, Hkv, D, S = 4, 2, 64, 200
    c = Batch(F32, Hq, Hkv, D, 16, [0], [S])
    qkv = c.rnd(S, (Hq + 2 * Hkv) * D)
    q = ops.paged_qkv_rope_split(qkv, c.k, c.v, c.table, 0, Hq, 1e4)
    q0 = torch.empty((1, Hq, S, D), device="cuda")
    k0, v0 = torch.empty((1, Hkv, S, D), device="cuda"), torch.empty((1, Hkv, S, D), device="cuda")
    ops.qkv_rope_split(qkv.view(1, S, -1), q0, k0, v0, 0, Hq, Hkv, 1e4)
    K, V, _ = c.keys(0, S)
    # the fp32 angle: position, rate (two roundings) and product: 3 2^-24 S
    e = (4 + 3 * S) * 2.0 ** -24 * 2 * qkv.abs().max().item()
    assert (q.transpose(0, 1) - q0[0]).abs().max() <= e
    assert (K - k0[0]).abs().max() <= e
    assert torch.equal(V, v0[0])


@pytest.mark.parametrize("dtype", [BF])
def test_split_of_partials(cuda, dtype):
    Hq, Hkv, D, T = 8, 2, 128, 6
    c = Batch(dtype, Hq, Hkv, D, 16, [100, 3, 47], [2, 2, 2])
    slabs = torch.randn((5, T, (Hq + 2 * Hkv) * D), generator=c.g, device="cuda")
    parts = ops.Partials(slabs, (T, slabs.shape[2]), dtype)
    k, v = c.k.clone(), c.v.clone()
    q = ops.paged_qkv_rope_split(parts, c.k, c.v, c.table, c.n_past, Hq, 1e4)
    total = slabs[0].clone()
    for s in slabs[1:]:
        total += s
    q1 = ops.paged_qkv_rope_split(total.to(dtype), k, v, c.table, c.n_past, Hq, 1e4)
    assert torch.equal(q, q1)
    assert torch.equal(c.k.nan_to_num(1.0), k.nan_to_num(1.0))
    assert torch.equal(c.v.nan_to_num(1.0), v.nan_to_num(1.0))


def test_split_outside_the_table(cuda):
    """Positions behind the table's last page and of absent pages are not written."""
    Hq, Hkv, D = 4, 2, 64
    c = Batch(BF, Hq, Hkv, D, 16, [30, 10, 60], [2, 2, 2], width=4)
    c.table[1, 0] = -1
    c.table[0, 1] = c.k.shape[0]
    before = c.k.clone()
    c.n_past[2] = 63
    qkv = c.rnd(6, (Hq + 2 * Hkv) * D)
    q = ops.paged_qkv_rope_split(qkv, c.k, c.v, c.table, c.n_past, Hq, 1e4)
    pos = torch.tensor([30, 31, 10, 11, 63, 64], device="cuda")
    y, tol = rotated(qkv.view(6, -1, D)[:, :Hq + Hkv], pos, 1e4)
    assert ((q.double() - y[:, :Hq]).abs() <= tol[:, :Hq]).all()
    # sequence 0: position 31 is the table's entry 1 (absent) like 30; 2: 63 is written, 64 not
    page, row = c.table[2, 3].long(), 15
    assert ((c.k[page, :, row].double() - y[4, Hq:]).abs() <= tol[4, Hq:]).all()
    c.k[page, :, row] = before[page, :, row]
    assert torch.equal(c.k.nan_to_num(1.0), before.nan_to_num(1.0))


# ---------------------------------------------------------------------------
# page copies
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("lead,n_pages,tail,n", [
    ((), 5, (1, 16, 8), 2), ((4,), 40, (3, 16, 64), 20), ((3, 2), 1000, (2, 16, 8), 499),
    ((2,), 7, (8, 128, 128), 3)])
def test_copy_pages(cuda, dtype, lead, n_pages, tail, n):
    g = torch.Generator(device="cuda").manual_seed(3)
    pages = torch.randn((*lead, n_pages, *tail), generator=g, device="cuda").to(dtype)
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(n)).tolist()
    src, dst = order[:n], order[n:2 * n]
    want = pages.clone()
    want[..., dst, :, :, :] = pages[..., src, :, :, :]
    assert ops.copy_pages(pages, src, dst) is pages
    assert torch.equal(pages, want)
    ops.copy_pages(pages, [], [])
    ops.copy_pages(pages, [order[0]] * (n_pages - 1), order[1:])  # a fork: one source
    assert torch.equal(pages, pages[..., order[:1], :, :, :].expand_as(pages))


def test_refusals(cuda):
    c = Batch(BF, 8, 2, 128, 16, [20, 5], [1, 1])

    def att(**kw):
        a = dict(q=c.q, k=c.k, v=c.v, t=c.table, n=c.n_past)
        more = {k: kw.pop(k) for k in list(kw) if k not in a}
        a.update(kw)
        return ops.paged_attention(a["q"], a["k"], a["v"], a["t"], a["n"], **more)

    att()
    for kw in (dict(q=c.q.cpu()), dict(q=c.q[:, :, :64]), dict(q=c.q[:, :3].contiguous()), dict(t=c.table.long()),
               dict(t=c.table.cpu()), dict(t=c.table[0]), dict(n=c.n_past[:1]), dict(n=c.n_past.long()),
               dict(n=-1), dict(n=10 ** 6), dict(k=c.k[:, :1].contiguous()), dict(starts=c.starts[:2]),
               dict(starts=c.starts.cpu()), dict(out=c.q[:1]), dict(max_new=-1), dict(max_keys=-1),
               dict(q=c.q[:1]), dict(workspace=torch.empty(8, dtype=torch.uint8)),
               dict(k=c.k[:, :, :8].contiguous(), v=c.v[:, :, :8].contiguous())):
        with pytest.raises(ValueError):
            att(**kw)
    for kw in (dict(q=c.q.float()), dict(v=c.v.float()), dict(k=c.k.half(), v=c.v.half(), q=c.q.half())):
        with pytest.raises(TypeError):
            att(**kw)
    from teenyformers_amd._lib import TeenyError
    for kw in (dict(softmax_scale=0.0), dict(softmax_scale=NAN)):
        with pytest.raises(TeenyError):
            att(**kw)
    long = Batch(BF, 8, 2, 128, 16, [9000], [1])
    with pytest.raises(TeenyError):
        long.run(workspace=torch.empty(64, dtype=torch.uint8, device="cuda"))
    pages = torch.zeros((2, 6, 2, 16, 64), device="cuda")
    for src, dst in (([0], [6]), ([-1], [1]), ([0, 1], [2]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([3], [3])):
        with pytest.raises(ValueError):
            ops.copy_pages(pages, src, dst)
    with pytest.raises(ValueError):
        ops.copy_pages(pages[0, 0], [0], [1])


@pytest.mark.parametrize("dtype,lens,most", [(BF, [1, 7, 1], 1), (BF, [1, 1, 5], 2), (F32, [2, 40, 1], 2),
                                             (BF, [9, 20, 3], 9), (BF, [40, 70, 1], 40)])
def test_more_new_tokens_than_said(cuda, dtype, lens, most):
    """A sequence with more new tokens than max_new: the others are as they should be, and nothing
    behind the workspace is written."""
    past = [3000, 2000, 2500]
    c = Batch(dtype, 8, 2, 64, 16, past, lens)
    T, Hq, D = c.q.shape
    from teenyformers_amd import _lib
    need = _lib.lib().teeny_paged_attention_workspace_bytes(3, T, most, 3000 + most, Hq, 2, D,
                                                            1 if dtype == BF else 0)
    assert need > 0
    ws = torch.full((need + 65536,), 0x5a, dtype=torch.uint8, device="cuda")
    out = torch.full_like(c.q, 7.0)
    c.run(out=out, max_new=most, max_keys=3000 + most, workspace=ws)
    assert (ws[need:] == 0x5a).all()
    ref, tol = c.reference()
    t = 0
    for n in lens:
        if n <= most:
            assert ((out[t:t + n].double() - ref[t:t + n]).abs() <= tol[t:t + n]).all()
        t += n


@pytest.mark.parametrize("dtype,lens,most", [(F32, [2, 40, 1], 2), (F32, [5, 6, 1], 5), (BF, [1, 7, 1], 1),
                                             (BF, [9, 20, 3], 9)])
def test_more_new_tokens_than_said_are_left_out(cuda, dtype, lens, most):
    """... and such a sequence's rows stay as they were, in one share or several."""
    for past in (40, 3000):
        c = Batch(dtype, 8, 2, 64, 16, [past] * 3, lens)
        out = torch.full_like(c.q, 7.0)
        c.run(out=out, max_new=most, max_keys=past + most)
        ref, tol = c.reference()
        t = 0
        for n in lens:
            if n <= most:
                assert ((out[t:t + n].double() - ref[t:t + n]).abs() <= tol[t:t + n]).all()
            else:
                assert (out[t:t + n] == 7.0).all()
            t += n


def test_copies_of_far_numbers(cuda):
    pages = torch.arange(2 * 2000, device="cuda").view(2, 2000, 1, 1, 1).expand(2, 2000, 1, 16, 8).float().contiguous()
    want = pages.clone()
    for src, dst in (([2 ** 31], [0]), ([0], [2 ** 40]), ([0], [-2 ** 40])):
        with pytest.raises(ValueError):
            ops.copy_pages(pages, src, dst)
    assert torch.equal(pages, want)
    src, dst = range(1000, 2000), torch.arange(1000)  # more than one launch's pairs; any iterables of whole numbers
    ops.copy_pages(pages, src, dst)
    want[:, :1000] = want[:, 1000:]
    assert torch.equal(pages, want)


def test_no_new_tokens(cuda):
    for dtype in (BF, F32):
        c = Batch(dtype, 8, 2, 64, 16, [100, 40], [1, 1])
        before = c.k.clone(), c.v.clone()
        starts = torch.zeros_like(c.starts)
        for kw in (dict(), dict(starts=starts)):
            assert ops.paged_attention(c.q[:0], c.k, c.v, c.table, c.n_past, **kw).shape == (0, 8, 64)
            qkv = c.rnd(0, (8 + 2 * 2) * 64)
            assert ops.paged_qkv_rope_split(qkv, c.k, c.v, c.table, c.n_past, 8, 1e4, **kw).shape == (0, 8, 64)
        out = torch.full_like(c.q, 7.0)  # tokens, but nobody's
        c.starts = starts
        c.run(out=out)
        assert (out == 7.0).all()
        assert torch.equal(c.k.view(torch.uint8), before[0].view(torch.uint8))
        assert torch.equal(c.v.view(torch.uint8), before[1].view(torch.uint8))


def test_device_values_out_of_their_ranges(cuda):
    """starts that fall or lie past the batch, lengths of any size: bounded, and a sequence that is
    well described is not disturbed."""
    for dtype in (BF, F32):
        c = Batch(dtype, 8, 2, 64, 16, [100, 40, 40, 9], [5, 1, 1, 1])
        ref, tol = c.reference()
        c.starts.copy_(torch.tensor([0, 5, 2 ** 31 - 1, -7, 10 ** 6], dtype=torch.int32))
        c.n_past.copy_(torch.tensor([100, 2 ** 31 - 1, -2 ** 31, 10 ** 9], dtype=torch.int32))
        c.k.nan_to_num_(0.5)  # (any row may be read)
        c.v.nan_to_num_(0.5)
        out = c.run()
        assert ((out[:5].double() - ref[:5]).abs() <= tol[:5]).all()
        qkv = c.rnd(8, (8 + 2 * 2) * 64)
        before = c.k.clone()
        q = ops.paged_qkv_rope_split(qkv, c.k, c.v, c.table, c.n_past, 8, 1e4, starts=c.starts)
        y, e = rotated(qkv[:5].view(5, 12, 64)[:, :10], torch.arange(100, 105, device="cuda"), 1e4)
        assert ((q[:5].double() - y[:, :8]).abs() <= e[:, :8]).all()
        changed = (c.k != before).flatten(1).any(1)
        assert set(changed.nonzero().view(-1).tolist()) <= set(c.table[0].tolist())


def test_far_lengths_of_one_sequence(cuda):
    """One sequence of 100000 keys: shares of the keys, positions far out."""
    for dtype, D in ((BF, 128), (F32, 32)):
        c = Batch(dtype, 4, 1, D, 64, [100000], [1])
        c.check(c.run(max_keys=100001))
        c.check(c.run())


@pytest.mark.parametrize("dtype,Hq,Hkv,D", [(F32, 4, 2, 64), (BF, 8, 2, 64), (BF, 8, 2, 128)])
@pytest.mark.parametrize("where", ["q", "k"])
def test_attention_of_nan_is_nan(cuda, dtype, Hq, Hkv, D, where):
    """A row whose scores are NaN, all of them or those of one share's keys, is NaN in one share and
    in several; the others are as they were."""
    for past, lens in (([40, 30], [2, 1]), ([9000, 30], [2, 1]), ([40, 3000], [60, 2]), ([9000, 30], [60, 1])):
        c = Batch(dtype, Hq, Hkv, D, 16, past, lens)
        keys = max(n + m for n, m in zip(past, lens))
        ref = c.run(max_new=max(lens), max_keys=keys)
        c.check(ref)
        if where == "q":
            c.q[1] = NAN  # one token of the first sequence
        else:
            c.k[c.table[0, :128 if past[0] > 2048 else 1].long()] = NAN  # its first keys: whole shares
        got = c.run(max_new=max(lens), max_keys=keys)
        if where == "q":
            assert got[1].isnan().all()
            assert torch.equal(got[:1], ref[:1]) and torch.equal(got[2:], ref[2:])
        else:
            assert got[:lens[0]].isnan().all()
            assert torch.equal(got[lens[0]:], ref[lens[0]:])


@pytest.mark.parametrize("dtype", [F32, BF])
def test_sequences_behind_one_of_broken_starts(cuda, dtype):
    """A sequence whose starts lie outside the batch, or fall, has no tokens; those behind it have
    theirs, in the split as in the attention."""
    past, lens = [20, 9, 2500, 50], [3, 0, 5, 2]
    for broken in ([0, 10 ** 6, 3, 8, 10], [0, -9, 3, 8, 10], [7, 0, 3, 8, 10], [2 ** 31 - 1, -2 ** 31, 3, 8, 10]):
        c = Batch(dtype, 8, 2, 64, 16, past, lens)
        qkv = c.rnd(10, (8 + 2 * 2) * 64)
        k, v = c.k.clone(), c.v.clone()
        want_q = ops.paged_qkv_rope_split(qkv, k, v, c.table, c.n_past, 8, 1e4, starts=c.starts)
        want = ops.paged_attention(c.q, k, v, c.table, c.n_past, starts=c.starts, max_keys=2600)
        c.starts.copy_(torch.tensor(broken, dtype=torch.int64).to(torch.int32))
        q = torch.full_like(want_q, 7.0)
        ops.paged_qkv_rope_split(qkv, c.k, c.v, c.table, c.n_past, 8, 1e4, starts=c.starts, q_out=q)
        assert torch.equal(q[3:], want_q[3:])
        for b in (2, 3):
            for got, there in zip((c.k, c.v), (k, v)):
                pages = c.table[b][c.table[b] >= 0].long()
                assert torch.equal(got[pages].nan_to_num(1.0), there[pages].nan_to_num(1.0))
        out = torch.full_like(c.q, 7.0)
        c.run(out=out, max_keys=2600)
        assert torch.equal(out[3:], want[3:])


@pytest.mark.parametrize("dtype", [F32, BF])
def test_split_far_behind_the_table(cuda, dtype):
    """q is rotated by the token's own position, however far behind the table that lies."""
    Hq, Hkv, D = 4, 2, 64
    c = Batch(dtype, Hq, Hkv, D, 16, [30, 10, 60], [2, 2, 2], width=4)
    before = c.k.clone(), c.v.clone()
    qkv = c.rnd(6, (Hq + 2 * Hkv) * D)
    x = qkv.view(6, -1, D)[:, :Hq]
    for n in ([64, 65, 1000], [100, 300000, 10 ** 9]):
        c.n_past.copy_(torch.tensor(n, dtype=torch.int32))
        q = ops.paged_qkv_rope_split(qkv, c.k, c.v, c.table, c.n_past, Hq, 1e4)
        pos = (torch.tensor(n)[:, None] + torch.arange(2)).view(-1).cuda()
        y, tol = rotated(x, pos, 1e4)
        # (angles of 1e9 in 64 bits: 1e9 times three roundings of 2^-53)
        tol = tol + (4e-7 if n[2] > 10 ** 6 else 0.0) * x.abs().max().item()
        assert ((q.double() - y).abs() <= tol).all()
        for now, then in zip((c.k, c.v), before):
            assert torch.equal(now.nan_to_num(1.0), then.nan_to_num(1.0))


@pytest.mark.parametrize("dtype,D", [(F32, 64), (BF, 64), (BF, 128)])
def test_one_key_of_nan(cuda, dtype, D):
    """A key of NaN makes the rows that see it NaN, whatever share or tile it lies in, and no other."""
    for past, lens in ((70, 3), (9000, 3), (70, 90), (3000, 90)):
        c = Batch(dtype, 8, 2, D, 16, [past, 40], [lens, 1])
        ref = c.run(max_new=lens, max_keys=past + lens)
        for at in (0, past // 2, past - 1, past + 1, past + lens - 1):
            page, row = c.table[0, at // 16], at % 16
            was = c.k[page, 1, row].clone()
            c.k[page, 1, row] = NAN
            got = c.run(max_new=lens, max_keys=past + lens)
            c.k[page, 1, row] = was
            first = max(0, at - past)  # the first token that sees it
            assert got[first:lens, 4:].isnan().all(), at
            assert got[:first, 4:].isfinite().all(), at
            assert torch.equal(got[:, :4], ref[:, :4]) and torch.equal(got[lens:], ref[lens:])
