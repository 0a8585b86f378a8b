"""Continuations of one prompt: the QKV split behind a prefix, the shared-prefix
cache, the captured sampling step, and the command that uses them, run together.

Logits of the shared-prefix path against the per-sequence cache, in fp32: each
side's attention is within 2e-6 (2-norm) of the exact one (the bound that the
attention's own tests hold it to) and everything else is the same arithmetic on
these inputs up to fp32 rounding of the same size, so two layers of both sides
stay within 2 * 2 * 2 * 2e-6 < 2e-5 of each other."""
import io
import json
from contextlib import redirect_stdout

import pytest
import torch

from teenyformers_amd import generate, llama, ops

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
TINY = dict(d_model=256, n_heads=4, n_layers=2, vocab_size=96, eps=1e-5, rope_base=1e4,
            intermediate_size=256, n_kv_heads_=2)


def model_of(dtype, std=0.08, **kw):
    cfg = llama.LlamaConfig(**{**TINY, **kw})
    return llama.Llama(cfg, llama.init_weights(cfg, dtype=dtype, seed=5, std=std))


def ids_of(B, S, seed=1, vocab=96):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, vocab, (B, S), generator=g, device="cuda")


def u_of(n, B, seed=2):
    return torch.rand((n, B), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("S", [1, 3, 37])
def test_qkv_split_behind_a_prefix(cuda, dtype, S):
    """Row r of a cache behind P prefix rows holds what row P + r of one cache does."""
    B, Hq, Hkv, D, P, L = 3, 8, 2, 64, 101, 50
    g = torch.Generator(device="cuda").manual_seed(0)
    qkv = torch.randn((B, S, (Hq + 2 * Hkv) * D), generator=g, device="cuda").to(dtype)
    new = lambda n: torch.full((B, Hkv, n, D), 7.0, dtype=dtype, device="cuda")  # noqa: E731
    qa, qb = (torch.empty((B, Hq, S, D), dtype=dtype, device="cuda") for _ in range(2))
    ka, va, kb, vb = new(P + L), new(P + L), new(L), new(L)
    ops.qkv_rope_split(qkv, qa, ka, va, P + 4, Hq, Hkv, 1e4)
    ops.qkv_rope_split(qkv, qb, kb, vb, 4, Hq, Hkv, 1e4, rope_offset=P)
    assert torch.equal(qa, qb) and torch.equal(ka[:, :, P:], kb) and torch.equal(va[:, :, P:], vb)
    # a position per sequence; one that is partly past the cache is written up to its end
    rows = [0, 9, L - (S + 1) // 2]
    pos = torch.tensor(rows, dtype=torch.int32, device="cuda")
    kc, vc, qc = new(L), new(L), torch.empty_like(qa)
    ops.qkv_rope_split(qkv, qc, kc, vc, pos, Hq, Hkv, 1e4, rope_offset=P)
    for b, r in enumerate(rows):
        k1, v1, q1 = (t[:1].clone() for t in (new(2 * P + 2 * L), new(2 * P + 2 * L), qa))
        ops.qkv_rope_split(qkv[b:b + 1].contiguous(), q1, k1, v1, P + r, Hq, Hkv, 1e4)
        n = min(S, L - r)
        assert torch.equal(qc[b], q1[0])
        assert torch.equal(kc[b, :, r:r + n], k1[0, :, P + r:P + r + n])
        assert torch.equal(vc[b, :, r:r + n], v1[0, :, P + r:P + r + n])
        keep = torch.ones(L, dtype=torch.bool, device="cuda")
        keep[r:r + n] = False
        assert (kc[b][:, keep] == 7).all() and (vc[b][:, keep] == 7).all()


def test_qkv_split_behind_a_prefix_from_slabs(cuda):
    """K-split slabs of a decode step, per-sequence positions: the same bits as
    their sum as a tensor."""
    B, Hq, Hkv, D, L = 5, 8, 2, 64, 40
    g = torch.Generator(device="cuda").manual_seed(0)
    slabs = torch.randn((3, B, (Hq + 2 * Hkv) * D), generator=g, device="cuda")
    parts = ops.Partials(slabs, (B, 1, (Hq + 2 * Hkv) * D), BF)
    pos = torch.tensor([0, 39, 5, -1, 40], dtype=torch.int32, device="cuda")
    out = []
    for src in (parts, parts.sum()):
        q = torch.empty((B, Hq, 1, D), dtype=BF, device="cuda")
        k, v = (torch.zeros((B, Hkv, L, D), dtype=BF, device="cuda") for _ in range(2))
        ops.qkv_rope_split(src, q, k, v, pos, Hq, Hkv, 1e4, rope_offset=17)
        out.append((q, k, v))
    for a, b in zip(*out):
        assert torch.equal(a, b)
    assert (out[0][1][3:] == 0).all()  # rows outside the cache are not written


@pytest.mark.parametrize("P", [1, 45, 300])
def test_logits_equal_the_copied_prefix(cuda, P):
    """fp32: several prompts behind one prefix, then decode steps, against each
    sequence run alone."""
    m = model_of(F32)
    prefix, own = ids_of(1, P), ids_of(4, 9, seed=3)
    lengths = torch.tensor([9, 1, 4, 7], device="cuda")
    cache, _ = m.share_prefix(prefix, 4, 20)
    logits = m.extend(cache, own, lengths)
    alone = []
    for b, n in enumerate(lengths.tolist()):
        alone.append(m.prefill(torch.cat([prefix, own[b:b + 1, :n]], 1), P + 20))
    nxt = ids_of(4, 1, seed=4)
    for step in range(5):
        for b, (c, want) in enumerate(alone):
            err = float((logits[b] - want[0]).norm() / want.norm())
            assert err <= 2e-5, (step, b, err)
        logits = m.decode_step(cache, nxt)
        alone = [(c, m.decode_step(c, nxt[b:b + 1])) for b, (c, _) in enumerate(alone)]
    assert cache.length == 14 and cache.lengths.tolist() == [14, 6, 9, 12]


def test_bf16_logits_near_the_copied_prefix(cuda):
    """bf16: P is rounded to 2^-8 on both sides, activations in between as often;
    the two paths' logits differ by a few roundings (2-norm)."""
    m = model_of(BF)
    prefix = ids_of(1, 200)
    cache, a = m.share_prefix(prefix, 3, 8)
    plain, b = m.prefill(prefix.expand(3, -1).contiguous(), 208)
    assert float((a.float() - b[:1].float()).norm() / b[:1].float().norm()) <= 2e-2
    for step in range(4):
        nxt = ids_of(3, 1, seed=10 + step)
        a, b = m.decode_step(cache, nxt), m.decode_step(plain, nxt)
        assert float((a.float() - b.float()).norm() / b.float().norm()) <= 2e-2


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("how", [dict(), dict(temperature=0.7, top_k=20, top_p=0.9, min_p=0.01),
                                 dict(temperature=0.0)])
def test_captured_steps_draw_what_eager_ones_do(cuda, dtype, how):
    m = model_of(dtype)
    u = u_of(7, 5)
    a = m.generate_samples(ids_of(1, 33), u, graph=True, **how)
    b = m.generate_samples(ids_of(1, 33), u, graph=False, **how)
    assert a.shape == (5, 7) and torch.equal(a, b)
    if how.get("temperature") == 0.0:
        assert (a == a[:1]).all()
    else:
        assert (a != a[:1]).any()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_padded_prompts_behind_the_prefix(cuda, dtype):
    """What padding holds changes nothing, captured or not."""
    m = model_of(dtype)
    own, lengths = ids_of(4, 11, seed=3), torch.tensor([11, 2, 5, 1], device="cuda")
    u = u_of(6, 4)
    runs = []
    for pad in (0, 95):
        x = own.clone()
        for b, n in enumerate(lengths.tolist()):
            x[b, n:] = pad
        for graph in (True, False):
            runs.append(m.generate_samples(ids_of(1, 70), u, 0.9, 30, ids=x, lengths=lengths,
                                           graph=graph))
    assert all(torch.equal(r, runs[0]) for r in runs[1:])


def test_greedy_samples_equal_generate(cuda):
    m = model_of(F32)
    prompt = ids_of(1, 40)
    a = m.generate_samples(prompt, u_of(8, 3), temperature=0.0)
    assert torch.equal(a, m.generate(prompt, 8).expand(3, -1))


def test_one_step_and_one_sample(cuda):
    m = model_of(BF)
    u = u_of(1, 4)
    assert m.generate_samples(ids_of(1, 5), u).shape == (4, 1)
    a = m.generate_samples(ids_of(1, 5), u_of(5, 4)[:, :1].contiguous())
    b = m.generate_samples(ids_of(1, 5), u_of(5, 4))
    assert a.shape == (1, 5) and a[0, 0] == b[0, 0]


def test_sampling_graph_over_a_plain_cache(cuda):
    """SampleGraph with per-sequence prompts (KVCache), settings changed between replays."""
    m = model_of(BF)
    prompt = ids_of(3, 20)
    u = u_of(6, 3)
    T = torch.full((3,), 0.8, device="cuda")
    cache, logits = m.prefill(prompt, 30)
    first = ops.sample_rows(logits, u[0], T).view(-1, 1)
    sg = llama.SampleGraph(m, cache, first, u[1].contiguous(), T)
    got = [first, sg.ids.clone()]
    for i in range(2, 6):
        T.fill_(0.8 if i < 4 else 1e-3)
        sg.replay(u[i])
        got.append(sg.ids.clone())
    cache, logits = m.prefill(prompt, 30)
    for i in range(6):
        t = 0.8 if i < 4 else 1e-3
        nxt = ops.sample_rows(logits, u[i].contiguous(), torch.full((3,), t, device="cuda")).view(-1, 1)
        assert torch.equal(nxt, got[i]), i
        logits = m.decode_step(cache, nxt)


def test_two_graphs_over_one_prefix(cuda):
    """Two batches of samples of one prompt, their captured steps replayed in turn."""
    m = model_of(BF)
    prompt, u = ids_of(1, 64), u_of(6, 4)
    cache, logits = m.share_prefix(prompt, 4, 8)
    other = llama.SharedPrefixCache(m.cfg, cache.prefix, 4, 8)
    first = ops.sample_rows(logits.expand(4, -1), u[0]).view(-1, 1)
    a = llama.SampleGraph(m, cache, first, u[1].contiguous())
    b = llama.SampleGraph(m, other, first, u[1].contiguous(), 0.5)
    got = [[a.ids.clone()], [b.ids.clone()]]
    for i in range(2, 6):
        for k, g in enumerate((a, b)):
            g.replay(u[i])
            got[k].append(g.ids.clone())
    for k, t in enumerate((1.0, 0.5)):
        c = llama.SharedPrefixCache(m.cfg, cache.prefix, 4, 8)
        nxt = first
        for i in range(1, 6):
            nxt = ops.sample_rows(m.decode_step(c, nxt), u[i].contiguous(), t).view(-1, 1)
            assert torch.equal(nxt, got[k][i - 1]), (k, i)


def test_refusals(cuda):
    m = model_of(BF)
    with pytest.raises(ValueError):
        m.share_prefix(ids_of(2, 5), 2, 4)
    cache, _ = m.share_prefix(ids_of(1, 5), 2, 4)
    for ids, lengths in [(ids_of(2, 5), None), (ids_of(3, 2), None),
                         (ids_of(2, 3), torch.tensor([0, 1])), (ids_of(2, 3), torch.tensor([4, 1])),
                         (ids_of(2, 3), torch.tensor([1.0, 1.0])), (ids_of(2, 3), torch.tensor([1]))]:
        with pytest.raises(ValueError):
            m.extend(cache, ids, lengths)
    m.extend(cache, ids_of(2, 4), torch.tensor([1, 4]))
    with pytest.raises(ValueError):
        m.extend(cache, ids_of(2, 1))
    with pytest.raises(ValueError):  # full: the longest sequence has no row left
        m.decode_step(cache, ids_of(2, 1))
    with pytest.raises(ValueError):
        m.generate_samples(ids_of(1, 5), u_of(2, 2).double())
    with pytest.raises(ValueError):
        llama.SharedPrefixCache(m.cfg, m.prefill(ids_of(2, 5), 8)[0], 2, 4)
    g = dict(n_heads_q=4, n_heads_kv=2, rope_base=1e4, rope_offset=5)
    qkv = torch.zeros((2, 1, 512), dtype=BF, device="cuda")
    q = torch.zeros((2, 4, 1, 64), dtype=BF, device="cuda")
    with pytest.raises(TypeError):
        ops.qkv_rope_split(qkv, q, cache.k[0], cache.v[0], torch.zeros(2, device="cuda"), **g)
    with pytest.raises(ValueError):
        ops.qkv_rope_split(qkv, q[:1], cache.k[0], cache.v[0], 0, **g)
    with pytest.raises(Exception, match="shape"):
        ops.qkv_rope_split(qkv, q, cache.k[0], cache.v[0], 4, **g)


def test_command_draws_samples(cuda, tmp_path):
    """--num-samples and the filters on a checkpoint: what generate_samples draws."""
    from tokenizers import Tokenizer, models, pre_tokenizers

    from tests.test_generate import _hf_tensors, _write_checkpoint
    cfg = llama.LlamaConfig(**TINY)
    _write_checkpoint(str(tmp_path), cfg, _hf_tensors(cfg, seed=3))
    words = [f"w{i}" for i in range(cfg.vocab_size)]
    tok = Tokenizer(models.WordLevel({w: i for i, w in enumerate(words)}, unk_token="w0"))
    tok.pre_tokenizer = pre_tokenizers.Whitespace()
    tok.save(str(tmp_path / "tokenizer.json"))
    buf = io.StringIO()
    with redirect_stdout(buf):
        assert generate.main(["--model-dir", str(tmp_path), "--prompt", "w5 w17 w3", "--max-new-tokens",
                              "5", "--num-samples", "3", "--temperature", "0.9", "--top-k", "40",
                              "--top-p", "0.95", "--min-p", "0.001", "--seed", "7"]) == 0
    m = llama.Llama(cfg, llama.load_hf_weights(cfg, str(tmp_path)))
    want = m.generate_samples(torch.tensor([[5, 17, 3]], device="cuda"), u_of(5, 3, seed=7), 0.9, 40,
                              0.95, 0.001).tolist()
    text = "w5 w17 w3\n"
    for i, row in enumerate(want):
        row = row[:row.index(2)] if 2 in row else row
        text += f"--- {i + 1}\n" + tok.decode(row) + "\n"
    assert buf.getvalue() == text


def test_preset_with_samples(cuda, monkeypatch):
    monkeypatch.setitem(generate.PRESETS, "tiny", dict(TINY))
    buf = io.StringIO()
    with redirect_stdout(buf):
        assert generate.main(["--preset", "tiny", "--batch", "1", "--prompt-len", "20", "--num-samples",
                              "4", "--max-new-tokens", "5", "--temperature", "1.0"]) == 0
    line = json.loads(buf.getvalue())
    assert line["num_samples"] == 4 and line["decode_ms_per_step"] > 0


def test_sample_steps_stop_with_the_caller(cuda, monkeypatch):
    """The steps of generate_samples, run as their tokens are asked for."""
    m = model_of(BF)
    u = u_of(9, 3)
    want = m.generate_samples(ids_of(1, 12), u, 0.9)
    replays = []
    replay = llama.SampleGraph.replay
    monkeypatch.setattr(llama.SampleGraph, "replay", lambda self, u: replays.append(1) or replay(self, u))
    for graph in (True, False):
        got = []
        for ids in m.sample_steps(ids_of(1, 12), u, 0.9, graph=graph):
            got.append(ids)
            if len(got) == 5:
                break
        assert torch.equal(torch.cat(got, 1), want[:, :5])
    assert len(replays) == 3


@pytest.mark.parametrize("lengths", [None, torch.tensor([1, 4])], ids=["one", "each"])
def test_a_full_cache_takes_no_captured_step(cuda, lengths):
    """Prompts that fill the sequences' rows: no step draws from keys without its own."""
    m = model_of(BF)
    cache, _ = m.share_prefix(ids_of(1, 5), 2, 4)
    m.extend(cache, ids_of(2, 4), lengths)
    nxt, u = ids_of(2, 1), u_of(1, 2)[0]
    with pytest.raises(RuntimeError, match="full"):
        llama.SampleGraph(m, cache, nxt, u)
    with pytest.raises(RuntimeError, match="full"):
        llama.DecodeGraph(m, cache, nxt)
    assert cache.length == 4
    plain, _ = m.prefill(ids_of(2, 6), 6)
    with pytest.raises(RuntimeError, match="full"):
        llama.DecodeGraph(m, plain, nxt)


@pytest.mark.parametrize("n_new", [1, 2, 3])
def test_preset_rates_are_of_steps_that_ran(cuda, monkeypatch, n_new):
    """The first two tokens come before the first replay, whose time is printed."""
    monkeypatch.setitem(generate.PRESETS, "tiny", dict(TINY))
    buf = io.StringIO()
    with redirect_stdout(buf):
        assert generate.main(["--preset", "tiny", "--batch", "1", "--prompt-len", "20", "--num-samples",
                              "4", "--max-new-tokens", str(n_new)]) == 0
    line = json.loads(buf.getvalue())
    if n_new < 3:
        assert line["decode_ms_per_step"] is None and line["decode_tokens_per_s"] is None
    else:
        assert line["decode_ms_per_step"] > 0 and line["decode_tokens_per_s"] > 0


def test_extend_keeps_lengths_of_its_own(cuda):
    """The caller's int32 lengths may change after the call."""
    m = model_of(F32)
    own, lengths = ids_of(3, 6, seed=3), torch.tensor([6, 2, 4], dtype=torch.int32, device="cuda")
    nxt, out = ids_of(3, 1, seed=4), []
    for change in (0, 1):
        cache, _ = m.share_prefix(ids_of(1, 9), 3, 8)
        given = lengths.clone()
        m.extend(cache, own, given)
        given += change
        out.append(m.decode_step(cache, nxt))
        assert cache.lengths.tolist() == [7, 3, 5]
    assert torch.equal(*out)


def test_command_draws_one_sample(cuda, tmp_path, monkeypatch):
    """One sample behind its prompt's text, up to its end; no step follows it."""
    from tokenizers import Tokenizer, models, pre_tokenizers

    from tests.test_generate import _hf_tensors, _write_checkpoint
    cfg = llama.LlamaConfig(**TINY)
    _write_checkpoint(str(tmp_path), cfg, _hf_tensors(cfg, seed=3))
    tok = Tokenizer(models.WordLevel({f"w{i}": i for i in range(cfg.vocab_size)}, unk_token="w0"))
    tok.pre_tokenizer = pre_tokenizers.Whitespace()
    tok.save(str(tmp_path / "tokenizer.json"))
    m = llama.Llama(cfg, llama.load_hf_weights(cfg, str(tmp_path)))
    row = m.generate_samples(torch.tensor([[5, 17, 3]], device="cuda"), u_of(9, 1, seed=7), 1.0, 40).tolist()[0]
    replays = []
    replay = llama.SampleGraph.replay
    monkeypatch.setattr(llama.SampleGraph, "replay", lambda self, u: replays.append(1) or replay(self, u))
    for eos in (None, row[4]):
        replays.clear()
        monkeypatch.setattr(generate, "eos_id", lambda t: -5 if eos is None else eos)
        buf = io.StringIO()
        with redirect_stdout(buf):
            assert generate.main(["--model-dir", str(tmp_path), "--prompt", "w5 w17 w3", "--max-new-tokens",
                                  "9", "--top-k", "40", "--seed", "7"]) == 0
        end = 9 if eos is None else row.index(eos)
        assert buf.getvalue() == "w5 w17 w3" + tok.decode(row[:end]) + "\n"
        assert len(replays) == (7 if eos is None else max(0, end - 1))
