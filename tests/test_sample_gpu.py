"""ops.sample_rows against the definition in 64 bits.

Tolerance: the kernel holds a weight to 2^-45 of the row's largest and evaluates
it to 2^-46 relative, so a running weight over V < 2^19 tokens is off by less
than V 2^-45 + 2^-46 of the total: below 1e-7 even if every error had one sign,
and below 1e-10 for the sizes here (V <= 130000: rounding errors of one sign only
up to sqrt(V)).  A token is accepted if the definition draws it for some u within
1e-9 of the given one; equal weights (exact) are compared without that margin."""
import numpy as np
import pytest
import torch

from teenyformers_amd import ops

pytestmark = pytest.mark.gpu
INF = float("inf")


def weights(x, T):
    """exp((x - max) / T) of one row, in 64 bits; -inf and NaN give 0."""
    x = np.where(np.isnan(x), -INF, x.astype(np.float64))
    m = x.max()
    if m == INF:
        return x, (x == INF).astype(np.float64)
    with np.errstate(under="ignore"):
        return x, np.exp((x - m) / T) if T < INF else np.isfinite(x).astype(np.float64)


def draw(x, u, T=1.0, k=0, p=1.0, m=0.0):
    """The definition for one row, and the set it keeps."""
    if not T > 0:
        T, k, p, m = 1.0, 1, 1.0, 0.0
    x = np.where(np.isnan(x), -INF, x.astype(np.float64))
    if not len(x) or x.max() == -INF:
        return -1
    x, w = weights(x, T)
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -INF]
    if x.max() == INF:
        order = order[x[order] == INF]
    if 0 < k < len(x):
        order = order[:k]
    if p < 1:
        run = np.cumsum(w[order])
        before = run - w[order]
        order = order[(before < max(p, 0.0) * run[-1]) | (np.arange(len(order)) == 0)]
    if m > 0:
        order = order[w[order] >= min(m, 1.0)]
    kept = np.sort(order)
    run = np.cumsum(w[kept])
    i = np.searchsorted(run, u * run[-1], side="right")
    return int(kept[min(i, len(kept) - 1)])


def check(logits, u, T=1.0, k=0, p=1.0, m=0.0, exact=False, **kw):
    got = ops.sample_rows(logits, u, T, k, p, m, **kw).reshape(-1).cpu().numpy()
    x = logits.reshape(-1, logits.shape[-1]).double().cpu().numpy()
    at = lambda v, r: float(v.reshape(-1)[r]) if torch.is_tensor(v) else v  # noqa: E731
    for r in range(x.shape[0]):
        a = (at(T, r), int(at(k, r)), at(p, r), at(m, r))
        us = float(u.reshape(-1)[r])
        want = {draw(x[r], us, *a)}
        if not exact:
            want |= {draw(x[r], max(0.0, us - 1e-9), *a), draw(x[r], us + 1e-9, *a)}
        assert got[r] in want, (r, got[r], want, a, us)
    return got


def make(rows, V, dtype, seed, cuda, zipf=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, V), generator=g, device="cuda")
    if zipf:
        x = x - 1.2 * torch.log(torch.rand((rows, V), generator=g, device="cuda").argsort(1) + 1.0)
    return x.to(dtype), torch.rand(rows, generator=g, device="cuda")


HOW = {
    "plain": {}, "cold": dict(T=0.3), "hot": dict(T=4.0), "topk": dict(k=50), "k1": dict(k=1),
    "topp": dict(p=0.9), "topp_hot": dict(T=3.0, p=0.97), "tiny_p": dict(p=1e-6), "minp": dict(m=0.05),
    "minp1": dict(m=1.0), "all": dict(T=0.8, k=40, p=0.9, m=0.02), "kp": dict(k=5000, p=0.99),
    "greedy": dict(T=0.0),
}


@pytest.mark.parametrize("how", sorted(HOW))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [1, 2, 7, 9, 300, 8191, 8193, 32001])
def test_against_definition(cuda, V, dtype, how):
    x, u = make(5, V, dtype, 100 + V, cuda)
    check(x, u, **HOW[how])


@pytest.mark.parametrize("how", ["plain", "topk", "topp", "topp_hot", "minp", "all"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_vocabulary(cuda, dtype, how):
    x, u = make(9, 128256, dtype, 7, cuda)
    check(x, u, **HOW[how])


@pytest.mark.parametrize("how", ["topp", "kp", "all", "topp_hot"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_border_bin_larger_than_the_list(cuda, dtype, how):
    """Nearly flat rows: one bin holds more tokens than LDS collects."""
    x, u = make(4, 60000, dtype, 11, cuda, zipf=False)
    check(x * 0.01, u, **HOW[how])


@pytest.mark.parametrize("V", [1, 5, 1000, 8192, 20000, 524280])
@pytest.mark.parametrize("how", [dict(), dict(k=3), dict(k=700), dict(p=0.5), dict(k=600, p=0.25),
                                 dict(m=1.0), dict(T=INF), dict(T=1e-30)])
def test_equal_logits_are_ordered_by_index(cuda, V, how):
    """Every weight is 1: running sums are exact, the borders are whole tokens."""
    u = torch.tensor([0.0, 0.25, 0.5, 0.9990234375], device="cuda")
    x = torch.full((4, V), -3.25, dtype=torch.bfloat16, device="cuda")
    check(x, u, exact=True, **how)


def test_two_levels_of_equal_logits(cuda):
    """0 (weight 1) and -1 at T = 1 / ln 2 (weight 1/2 to rounding): top-k and
    top-p end among equal tokens spread over several chunks."""
    V = 30000
    x = torch.full((1, V), -1.0, device="cuda")
    x[0, 5::7] = 0.0
    n = int((x == 0).sum())
    u = torch.tensor([0.77], device="cuda")
    for k in (1, n - 1, n, n + 1, n + 9000, V - 1):
        check(x, u, k=k)
    for p in (0.1, 0.3001, 0.61, 0.87):
        check(x, u, p=p)
        check(x, u, k=n + 9000, p=p)


@pytest.mark.parametrize("how", ["plain", "topk", "topp", "minp", "all", "greedy"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_and_infinite_logits(cuda, dtype, how):
    x, u = make(8, 9001, dtype, 3, cuda)
    x[0] = -INF                              # nothing left
    x[1] = float("nan")
    x[2, 1:] = -INF                          # one token
    x[3, :8500] = -INF                       # the last chunk only
    x[4, 100:] = torch.finfo(dtype).min      # masked with the type's lowest value
    x[5] = torch.finfo(dtype).min            # everything masked so: all equal
    x[6, 17] = INF
    x[6, 9000] = INF
    x[7, ::2] = float("nan")
    got = check(x, u, **HOW[how])
    assert got[0] == -1 and got[1] == -1 and got[2] == 0


def test_signed_zeros_are_equal(cuda):
    x = torch.full((1, 4), -50.0, device="cuda")
    x[0, 1], x[0, 2] = 0.0, -0.0
    u = torch.tensor([0.0], device="cuda")
    assert int(ops.sample_rows(x, u, top_k=1)) == 1
    x[0, 1], x[0, 2] = -0.0, 0.0
    assert int(ops.sample_rows(x, u, temperature=0.0)) == 1


def test_u_at_its_borders(cuda):
    x, _ = make(6, 777, torch.float32, 5, cuda)
    u = torch.tensor([0.0, -1.0, float("nan"), 1.0, 7.0, 1 - 2.0 ** -24], device="cuda")
    got = ops.sample_rows(x, u).tolist()
    assert got[:5] == [0, 0, 0, 776, 776]
    check(x[5:], u[5:])


def test_settings_per_row(cuda):
    rows = 40
    x, u = make(rows, 12345, torch.bfloat16, 9, cuda)
    g = torch.Generator(device="cuda").manual_seed(1)
    f = lambda lo, hi: lo + (hi - lo) * torch.rand(rows, generator=g, device="cuda")  # noqa: E731
    T, p, m = f(0.2, 2.0), f(0.3, 1.1), f(-0.1, 0.2)
    k = f(-5.0, 300.0).to(torch.int32)
    T[::7] = 0.0
    check(x, u, T, k, p, m)
    # odd values that only a device tensor can bring: off, or one token
    T = torch.tensor([float("nan"), -1.0, INF, 1.0, 1.0, 1.0], device="cuda")
    p = torch.tensor([1.0, 1.0, 1.0, 0.0, -2.0, float("nan")], device="cuda")
    m = torch.tensor([0.0, 0.0, 0.0, 0.0, float("nan"), 5.0], device="cuda")
    got = ops.sample_rows(x[:6], u[:6], T, 0, p, m).tolist()
    top = x[:6].double().argmax(1).tolist()
    assert [got[i] for i in (0, 1, 3, 4)] == [top[i] for i in (0, 1, 3, 4)]
    assert got[2] == draw(x[2].double().cpu().numpy(), float(u[2]), INF)
    assert float(x[5, got[5]]) == float(x[5].max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("first", [0, 1, 3])
def test_rows_apart_and_unaligned(cuda, dtype, first):
    """Rows cut from a wider product: what lies around them is not read as theirs."""
    x, u = make(6, 8200, dtype, 21, cuda)
    wide = torch.full((6, 8200 + 37), 1e4, dtype=dtype, device="cuda")
    part = wide[:, first:first + 8200]
    part.copy_(x)
    for how in ("plain", "topk", "topp"):
        a = check(part, u, **HOW[how])
        assert (a == ops.sample_rows(x, u, *_args(**HOW[how])).cpu().numpy()).all()


def _args(T=1.0, k=0, p=1.0, m=0.0):
    return T, k, p, m


def test_one_row_for_all_and_shapes(cuda):
    x, u = make(1, 5003, torch.bfloat16, 2, cuda)
    us = torch.rand(33, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    a = ops.sample_rows(x.expand(33, -1), us, 0.9, 20)
    b = ops.sample_rows(x.repeat(33, 1), us, 0.9, 20)
    assert torch.equal(a, b)
    x3 = x.repeat(6, 1).view(2, 3, 5003)
    c = ops.sample_rows(x3, us[:6], 0.9, 20)
    assert c.shape == (2, 3) and torch.equal(c.reshape(-1), a[:6])
    d = ops.sample_rows(x3.transpose(0, 2).contiguous().transpose(0, 2), us[:6], 0.9, 20)
    assert torch.equal(d, c)
    one = ops.sample_rows(x[0], us[:1], 0.9, 20)
    assert one.shape == () and int(one) == int(a[0])
    assert ops.sample_rows(x[:0], us[:0]).shape == (0,)


def test_row_results_do_not_depend_on_the_batch(cuda):
    x, u = make(70, 128256, torch.bfloat16, 31, cuda)
    a = ops.sample_rows(x, u, 0.8, 0, 0.95)
    b = torch.cat([ops.sample_rows(x[i:i + 1], u[i:i + 1], 0.8, 0, 0.95) for i in range(0, 70, 9)])
    assert torch.equal(a[::9], b)
    assert torch.equal(a, ops.sample_rows(x, u, 0.8, 0, 0.95))


def test_draws_follow_the_distribution(cuda):
    """Evenly spaced u hit each token in proportion to its probability, to one draw."""
    n = 4096
    x = torch.tensor([[0.3, -1.0, 2.0, 0.0, -INF, 1.1]], device="cuda")
    u = (torch.arange(n, device="cuda") + 0.5) / n
    got = ops.sample_rows(x.expand(n, -1), u).bincount(minlength=6).double().cpu()
    assert (got - torch.softmax(x[0].double(), 0).cpu() * n).abs().max() <= 1.0


def test_captured_and_replayed(cuda):
    """A captured draw reads the logits, u and settings of each replay, and moves
    the position on."""
    x, u = make(5, 40000, torch.bfloat16, 13, cuda)
    T = torch.full((5,), 0.8, device="cuda")
    p = torch.full((5,), 0.9, device="cuda")
    out = torch.zeros(5, dtype=torch.int64, device="cuda")
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.sample_rows(x, u, T, 50, p, out=out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        ops.sample_rows(x, u, T, 50, p, out=out, advance=pos)
    for i in range(4):
        y, v = make(5, 40000, torch.bfloat16, 50 + i, cuda)
        x.copy_(y)
        u.copy_(v)
        T.fill_(0.5 + 0.2 * i)
        g.replay()
        torch.cuda.synchronize()
        assert int(pos) == i + 1
        assert torch.equal(out, ops.sample_rows(y, v, T, 50, p))


def test_another_stream(cuda):
    x, u = make(3, 128256, torch.bfloat16, 17, cuda)
    want = ops.sample_rows(x, u, 0.7, 0, 0.9)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = ops.sample_rows(x, u, 0.7, 0, 0.9)
    s.synchronize()
    assert torch.equal(got, want)


def test_refusals(cuda):
    x = torch.zeros((2, 10), device="cuda")
    u = torch.zeros(2, device="cuda")
    bad = [dict(temperature=-1.0), dict(temperature=float("nan")), dict(top_k=-1), dict(top_p=0.0),
           dict(top_p=1.5), dict(min_p=-0.1), dict(min_p=2.0),
           dict(temperature=torch.ones(3, device="cuda")), dict(temperature=torch.ones(2)),
           dict(top_k=torch.ones(2, device="cuda")), dict(top_p=torch.ones(2, device="cuda").double()),
           dict(out=torch.zeros(2, dtype=torch.int32, device="cuda")),
           dict(advance=torch.zeros(1, device="cuda"))]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.sample_rows(x, u, **kw)
    for args in [(x, u[:1]), (x, u.double()), (x, u.cpu()), (x.cpu(), u), (x[:, :0], u)]:
        with pytest.raises(ValueError):
            ops.sample_rows(*args)
    with pytest.raises(TypeError):
        ops.sample_rows(x.half(), u)
    with pytest.raises(Exception, match="workspace"):
        ops.sample_rows(x, u, workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))
    with pytest.raises(Exception, match="shape"):
        ops.sample_rows(torch.zeros((1, 524281), dtype=torch.bfloat16, device="cuda"), u[:1])


DENSE = {
    "minp": dict(m=0.985), "topp_low": dict(p=0.3), "k_topp": dict(k=20000, p=0.9),
    "few": dict(k=300, p=0.5), "few_minp": dict(k=500, m=0.99),
    "all": dict(k=30000, p=0.5, m=0.985), "k_minp": dict(k=60001, m=0.99),
}


@pytest.mark.parametrize("how", sorted(DENSE))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,spread", [(70000, 0.01), (128256, 0.002), (128256, 0.3)])
def test_borders_of_flat_rows(cuda, V, spread, dtype, how):
    """Each border in a bin of thousands of tokens: of few keys and of many, with
    one border after another in the same bin and in different ones."""
    x, u = make(3, V, dtype, 23, cuda, zipf=False)
    check(x * spread, u, **DENSE[how])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_flat_rows_apart_and_unaligned(cuda, dtype):
    x, u = make(4, 50003, dtype, 29, cuda, zipf=False)
    for first in (0, 3, 5):
        check((x * 0.01)[:, first:49999], u, k=9000, p=0.7)


def test_two_streams_at_once(cuda):
    """Calls in flight together, each with a workspace of its own."""
    xs = [make(32, 40000, torch.bfloat16, 31 + i, cuda) for i in range(2)]
    how = [dict(top_p=0.9), dict(top_k=700, top_p=0.95, min_p=0.001)]
    want = [ops.sample_rows(x, u, **h) for (x, u), h in zip(xs, how)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.sample_rows(*xs[i], **how[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


@pytest.mark.parametrize("how", sorted(HOW))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,V", [(300, 1), (270, 61), (270, 8185), (150, 8193), (60, 40001)])
def test_more_chunks_than_workgroups_at_once(cuda, rows, V, dtype, how):
    """Rows enough for the scan's other workgroup size, and its rows' ends."""
    x, u = make(rows, V, dtype, 300 + V, cuda)
    check(x, u, **HOW[how])


@pytest.mark.parametrize("how", sorted(DENSE))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_flat_rows(cuda, dtype, how):
    x, u = make(40, 60000, dtype, 37, cuda, zipf=False)
    check(x * 0.01, u, **DENSE[how])


def test_results_do_not_depend_on_the_workgroups(cuda):
    """One row alone and among many: the same token."""
    x, u = make(300, 20000, torch.bfloat16, 41, cuda)
    x[7, 100:9000] = -INF
    x[8] = -INF
    x[9, 5] = INF
    for how in (dict(), dict(top_k=50, top_p=0.9), dict(top_k=600), dict(top_p=0.95), dict(min_p=0.05)):
        got = ops.sample_rows(x, u, 0.9, **how)
        for i in (0, 7, 8, 9, 299):
            assert torch.equal(got[i:i + 1], ops.sample_rows(x[i:i + 1], u[i:i + 1], 0.9, **how))


@pytest.mark.parametrize("n", [2, 63, 64, 65, 130])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_borders_among_a_few_equal_tokens(cuda, dtype, n):
    """n equal tokens spread over the row, and the border at each kind of place
    among them: by count, by weight, one after the other."""
    V = 20011
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.rand((6, V), generator=g, device="cuda") * 4 - 12
    at = torch.randperm(V, generator=g, device="cuda")[:n + 9]
    x[:, at[:n]] = 2.0
    x[:, at[n:]] = 3.0 + torch.rand((6, 9), generator=g, device="cuda")
    x = x.to(dtype)
    u = torch.tensor([0.0, 0.2, 0.5, 0.7, 0.9, 0.9999], device="cuda")
    for k in (8, 9, 10, 9 + n // 2, 8 + n, 9 + n, 10 + n, 600):
        check(x, u, k=k)
        check(x, u, k=k, p=0.95)
        check(x, u, T=2.0, k=k + 513, p=0.9)
    for p in (0.3, 0.8, 0.9, 0.97):
        check(x, u, p=p)
        check(x, u, T=0.5, p=p)


def test_a_batch_without_rows_moves_the_position_on(cuda):
    x, u = make(2, 10, torch.float32, 1, cuda)
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert ops.sample_rows(x[:0], u[:0], advance=pos).shape == (0,) and int(pos) == 1
    assert ops.sample_rows(x, u, advance=pos).shape == (2,) and int(pos) == 2


@pytest.mark.parametrize("k", [200, 215, 230, 300, 512, 513])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_top_k_around_what_the_chunks_write_out(cuda, dtype, k):
    """16 chunks of 128256 columns: the draw takes in what they write out for a k of
    200, and weighs larger ones by bins."""
    x, u = make(4, 128256, dtype, 43, cuda)
    for how in (dict(), dict(p=0.9), dict(T=0.5, m=0.01), dict(T=1.3, p=0.95, m=0.002)):
        check(x, u, k=k, **how)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_least_weight_that_is_drawn(cuda, dtype):
    """Without filters down to 2^-45 of the largest of the token's 8192 columns, with
    them to 2^-45 of the row's."""
    x = torch.full((3, 20000), -100.0, device="cuda")
    x[:, 9000] = 0.0
    x[:, 5] = -30.0
    x[:, 0] = torch.tensor([-70.0, -77.0, -44.0], device="cuda")
    u = torch.zeros(3, device="cuda")
    for scale in (1.0, 0.5):  # the logits in octaves
        T = scale / np.log(2.0)
        y = (x * scale).to(dtype)
        assert ops.sample_rows(y, u, T).tolist() == [0, 5, 0]
        assert ops.sample_rows(y, u, T, top_k=19999).tolist() == [5, 5, 0]


@pytest.mark.parametrize("rows", [1, 16, 300])
def test_calls_repeat_themselves(cuda, rows):
    x, u = make(rows, 128256, torch.bfloat16, 47, cuda)
    for how in (dict(), dict(top_k=50, top_p=0.9), dict(top_k=300), dict(top_p=0.95), dict(min_p=0.01)):
        want = ops.sample_rows(x, u, 1.3, **how)
        assert all(torch.equal(ops.sample_rows(x, u, 1.3, **how), want) for _ in range(5))


@pytest.mark.parametrize("how", [dict(k=1), dict(k=300, p=0.5), dict(k=500, m=0.99), dict(k=500, p=0.7, m=0.985)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,spread", [(8000, 0.01), (40000, 0.01), (49000, 0.3), (49000, 0.002)])
def test_small_top_k_of_flat_rows(cuda, V, spread, dtype, how):
    """Chunks whose first bins hold more than they write out: passes over the row."""
    x, u = make(3, V, dtype, 53, cuda, zipf=False)
    check(x * spread, u, **how)
