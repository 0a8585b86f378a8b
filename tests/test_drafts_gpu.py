"""The paged cache, its attention, page copies and the verification of drafts run
together through the model: run_paged, draft_steps and the command.

Logits in fp32 against the model without pages: each side's attention is within 2e-6
(2-norm) of the exact one and the rest is the same arithmetic up to fp32 rounding; the
rotary angles of the other side are fp32 products, off by 3 2^-24 a position, which below
300 positions moves a rotated row by 300 * 3 * 2^-24 = 5.4e-5 of itself in one plane, so its
scores (a few units at these weights) by 2e-4 and the two layers' outputs by less than 5e-4."""
import io
from contextlib import redirect_stdout

import numpy as np
import pytest
import torch

from teenyformers_amd import generate, llama, ops
from tests.test_verify_gpu import reference

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
TINY = dict(d_model=256, n_heads=4, n_layers=2, vocab_size=96, eps=1e-5, rope_base=1e4,
            intermediate_size=256, n_kv_heads_=2)
CLOSE = 5e-4


def model_of(dtype, std=0.08, seed=5, **kw):
    cfg = llama.LlamaConfig(**{**TINY, **kw})
    return llama.Llama(cfg, llama.init_weights(cfg, dtype=dtype, seed=seed, std=std))


def ids_of(n, seed=1, vocab=96):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, vocab, (n,), generator=g, device="cuda")


def off(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


@pytest.mark.parametrize("page", [16, 64])
def test_run_paged_against_forward(cuda, page):
    """Ragged prompts in chunks, then single tokens: the logits of whole passes."""
    m = model_of(F32)
    texts = [ids_of(n, seed=n) for n in (1, 40, 133, 17)]
    cache = llama.PagedKVCache(m.cfg, 300 // page + 12, page, F32)
    seqs = [cache.add() for _ in texts]
    at = [0] * 4
    for chunk in ([1, 20, 100, 17], [0, 19, 1, 0], [0, 1, 32, 0]):
        now = [i for i in range(4) if chunk[i]]
        rows = m.run_paged(cache, [seqs[i] for i in now], [texts[i][at[i]:at[i] + chunk[i]] for i in now],
                           all_rows=True)
        r = 0
        for i in now:
            want = m.forward(texts[i][None, :at[i] + chunk[i]])[0, at[i]:]
            assert off(rows[r:r + chunk[i]], want) < CLOSE
            at[i] += chunk[i]
            r += chunk[i]
    assert [cache.lengths[s] for s in seqs] == [1, 40, 133, 17]
    more = ids_of(4, seed=9)
    last = m.run_paged(cache, seqs, [[int(t)] for t in more])
    for i, t in enumerate(texts):
        want = m.forward(torch.cat([t, more[i:i + 1]])[None])[0, -1]
        assert off(last[i], want) < CLOSE


def test_run_paged_bf16_against_forward(cuda):
    """bf16: both sides round each stage; within the model tests' bar of each other."""
    m = model_of(BF)
    texts = [ids_of(n, seed=n) for n in (200, 3, 77)]
    cache = llama.PagedKVCache(m.cfg, 20, 32, BF)
    seqs = [cache.add() for _ in texts]
    got = m.run_paged(cache, seqs, texts)
    for i, t in enumerate(texts):
        assert off(got[i], m.forward(t[None])[0, -1]) < 2e-2


def test_forks_copy_before_they_write(cuda):
    """Continuations of one prompt, each as if it had been alone; then a compacted pool."""
    m = model_of(F32)
    prompt = ids_of(45)
    cache = llama.PagedKVCache(m.cfg, 30, 16, F32)
    gone = cache.add()
    m.run_paged(cache, [gone], [ids_of(100, seed=8)])  # the first pages: free later
    first = cache.add()
    m.run_paged(cache, [first], [prompt])
    forks = cache.fork(first, 4)
    own = [ids_of(n, seed=20 + n) for n in (1, 5, 20, 2)]
    got = m.run_paged(cache, forks, own)
    again = m.run_paged(cache, [first], [[7]])
    for i, t in enumerate(own):
        assert off(got[i], m.forward(torch.cat([prompt, t])[None])[0, -1]) < CLOSE
    assert off(again[0], m.forward(torch.cat([prompt, prompt.new_tensor([7])])[None])[0, -1]) < CLOSE
    cache.remove(gone)
    cache.truncate(forks[2], 47)
    assert cache.compact() == 30 - cache.free_pages
    got = m.run_paged(cache, [forks[2], forks[0]], [[3, 4], [5]])
    assert off(got[0], m.forward(torch.cat([prompt, own[2][:2], prompt.new_tensor([3, 4])])[None])[0, -1]) < CLOSE
    assert off(got[1], m.forward(torch.cat([prompt, own[0], prompt.new_tensor([5])])[None])[0, -1]) < CLOSE


def greedy(m, prompt, n):
    """Greedy tokens by whole passes, and whether each choice is clear of the paths' difference."""
    seq, clear = prompt.tolist(), True
    for _ in range(n):
        x = m.forward(torch.tensor([seq], device="cuda"))[0, -1].double()
        top = x.topk(2).values
        clear = clear and (top[0] - top[1]) > 2 * CLOSE * x.norm()
        seq.append(int(x.argmax()))
    return seq[len(prompt):], clear


@pytest.mark.parametrize("how", ["lookup", "model", "same"])
@pytest.mark.parametrize("K", [1, 3, 6])
def test_greedy_drafts(cuda, how, K):
    """Temperature 0: the tokens of greedy decoding, whatever drafted them."""
    m = model_of(F32, std=0.15)
    d = None if how == "lookup" else m if how == "same" else model_of(F32, std=0.15, seed=6, n_layers=1)
    prompts = [ids_of(n, seed=n) for n in (9, 30, 2)]
    n_new = 20
    u = torch.rand((n_new, 3, (2 if d else 1) * K + 1), device="cuda")
    steps = list(m.draft_steps(prompts, u, K, temperature=0.0, draft=d, page_size=16))
    got = [sum((s[i] for s in steps), []) for i in range(3)]
    clear = 0
    for p, t in zip(prompts, got):
        want, ok = greedy(m, p, n_new)
        assert len(t) == n_new
        clear += ok
        if ok:
            assert t == want
    assert clear >= 1
    if how == "same" and clear == 3:  # every draft is right: K + 1 tokens a step
        assert len(steps) == 1 + -(-(n_new - 1) // (K + 1))


def test_drafts_draw_what_the_definition_draws(cuda):
    """Temperature 0.9, two samples of a prompt: the run replayed by the definition in 64 bits on
    whole passes' logits."""
    m, d = model_of(F32), model_of(F32, seed=5, std=0.075)
    prompt, K, n_new = ids_of(21), 3, 14
    for draft in (None, d):
        g = torch.Generator(device="cuda").manual_seed(4)
        u = torch.rand((n_new, 2, (2 if draft else 1) * K + 1), generator=g, device="cuda")
        got = m.generate_drafted([prompt], u, K, temperature=0.9, draft=draft, samples=2, page_size=16)
        for b in range(2):
            text, step, sure, per_step = prompt.tolist(), 0, True, []
            logits = m.forward(prompt[None])[:, -1:]
            none = torch.full((1, 1), -1)
            t, _, s = reference(logits.expand(1, 2, -1), none, torch.stack([u[0, b, K], u[0, b, K]])[None], None, 0.9)
            made = [int(t[0, 0])]
            sure = sure and s[0]
            while len(made) < n_new and sure:
                step += 1
                # (the other sample's drafts decide how many rows this step has, not what they are)
                room = min(K, n_new - len(made) - 1)
                text = prompt.tolist() + made
                if draft is None:
                    guess, q = llama.lookup_drafts(text, room), None
                else:
                    guess, q = [], []
                    for j in range(room):
                        x = draft.forward(torch.tensor([text + guess], device="cuda"))[:, -1:]
                        q.append(x)
                        t, _, s = reference(x.expand(1, 2, -1), none, u[step, b, K + 1 + j].expand(1, 2), None, 0.9)
                        sure = sure and s[0]
                        guess.append(int(t[0, 0]))
                k = len(guess)
                x = m.forward(torch.tensor([text + guess], device="cuda"))[:, len(text) - 1:]
                pick = torch.cat([u[step, b, :k], u[step, b, K:K + 1]])[None]
                if k == 0:
                    t, a, s = reference(x.expand(1, 2, -1), none, pick.expand(1, 2), None, 0.9)
                else:
                    t, a, s = reference(x, torch.tensor([guess]), pick, torch.cat(q, 1) if q else None, 0.9)
                sure = sure and s[0]
                made += t[0, :a[0] + 1].tolist()
            made = made[:n_new]
            # the logits of the two paths differ by up to CLOSE: a draw in a hundred may lie
            # between; the first ones of 14 agree in any case that is not one of those
            same = sum(x == y for x, y in zip(made, got[b]))
            assert len(got[b]) == n_new and (same == n_new or same >= 3)


def test_drafts_with_filters_and_ends(cuda):
    """Filters draw row by row: the tokens of a run without drafts at the same numbers are not the
    same ones, but every token is one that the filters leave; eos ends a sequence alone."""
    m = model_of(F32)
    prompts, K, n_new = [ids_of(12, seed=1), ids_of(33, seed=2)], 4, 16
    g = torch.Generator(device="cuda").manual_seed(4)
    u = torch.rand((n_new, 2, K + 1), generator=g, device="cuda")
    got = m.generate_drafted(prompts, u, K, temperature=1.0, top_k=3, page_size=16)
    for p, t in zip(prompts, got):
        assert len(t) == n_new
        x = m.forward(torch.tensor([p.tolist() + t], device="cuda"))[0].double()
        for i, tok in enumerate(t):
            row = x[len(p) - 1 + i]
            assert row[tok] >= row.topk(3).values[-1] - 2 * CLOSE * row.norm()
    eos = got[0][5]
    short = m.generate_drafted(prompts, u, K, temperature=1.0, top_k=3, page_size=16, eos=eos)
    for s, t in zip(short, got):
        end = t.index(eos) + 1 if eos in t else n_new
        assert s[:1] == t[:1] and (s[-1] == eos or len(s) == n_new) and eos not in s[:-1]
        assert len(s) <= n_new and (len(s) == end or s != t[:len(s)])


def test_command_drafts(cuda, tmp_path):
    """--draft-len on a checkpoint, looked up and by a second one: greedy text is greedy text."""
    from tokenizers import Tokenizer, models, pre_tokenizers

    from tests.test_generate import _hf_tensors, _write_checkpoint
    cfg = llama.LlamaConfig(**TINY)
    small = llama.LlamaConfig(**{**TINY, "n_layers": 1})
    (tmp_path / "m").mkdir()
    (tmp_path / "d").mkdir()
    _write_checkpoint(str(tmp_path / "m"), cfg, _hf_tensors(cfg, seed=3))
    _write_checkpoint(str(tmp_path / "d"), small, _hf_tensors(small, seed=3))
    tok = Tokenizer(models.WordLevel({f"w{i}": i for i in range(cfg.vocab_size)}, unk_token="w0"))
    tok.pre_tokenizer = pre_tokenizers.Whitespace()
    tok.save(str(tmp_path / "m" / "tokenizer.json"))

    def run(*more):
        buf = io.StringIO()
        with redirect_stdout(buf):
            assert generate.main(["--model-dir", str(tmp_path / "m"), "--prompt", "w5 w17 w3 w5 w17", "--dtype", "f32",
                                  "--max-new-tokens", "12", "--seed", "7", *more]) == 0
        return buf.getvalue()

    m = llama.Llama(cfg, llama.load_hf_weights(cfg, str(tmp_path / "m"), dtype=F32))
    want, clear = greedy(m, torch.tensor([5, 17, 3, 5, 17]), 12)
    want = want[:want.index(2)] if 2 in want else want
    for more in (["--draft-len", "4"], ["--draft-len", "2", "--draft-dir", str(tmp_path / "d")]):
        text = run(*more)
        assert text.startswith("w5 w17 w3 w5 w17") and text.endswith("\n")
        if clear:
            assert text == "w5 w17 w3 w5 w17" + tok.decode(want) + "\n"
    two = run("--draft-len", "3", "--num-samples", "2", "--temperature", "0.8")
    assert two.count("--- ") == 2
    assert run("--draft-len", "3", "--top-k", "5").startswith("w5 w17 w3 w5 w17")


@pytest.mark.parametrize("dtype", [F32, BF])
def test_greedy_drafts_of_equal_logits(cuda, dtype):
    """Every token has a twin of the same embedding, so of the same logit: greedy decoding takes the
    last of them, with drafts as without."""
    m = model_of(dtype, std=0.15)
    m.w["model.embed_tokens.weight"][48:] = m.w["model.embed_tokens.weight"][:48]
    d = llama.Llama(m.cfg, m.w)
    prompts, n_new, K = [ids_of(9, seed=1, vocab=48), ids_of(20, seed=2, vocab=48)], 12, 3
    for draft in (None, d):
        u = torch.rand((n_new, 2, (2 if draft else 1) * K + 1), device="cuda")
        got = m.generate_drafted(prompts, u, K, temperature=0.0, draft=draft, page_size=16)
        for p, t in zip(prompts, got):
            assert min(t) >= 48 and len(t) == n_new
            assert int(m.generate(p[None], n_new).min()) >= 48
            if dtype == F32:
                seq, x = p.tolist(), None
                for tok in t:
                    x = m.forward(torch.tensor([seq], device="cuda"))[0, -1].double()
                    assert x[tok] >= x.max() - 2 * CLOSE * x.norm()
                    seq.append(tok)


def recorded(model, log):
    """The model's passes over pages, logged: their tokens by sequence, and their logits."""
    run = model.run_paged

    def wrapper(cache, seqs, ids, all_rows=False):
        rows = run(cache, seqs, ids, all_rows)
        log.append(([[int(t) for t in x] for x in ids], rows.clone()))
        return rows

    model.run_paged = wrapper


@pytest.mark.parametrize("how", ["lookup", "model", "filter", "greedy", "greedy model"])
@pytest.mark.parametrize("ends", [False, True])
def test_steps_replayed_token_by_token(cuda, how, ends):
    """Every pass of a run of drafts holds the tokens that it should and gives the logits of whole
    passes over its sequences' texts, and every step's tokens are the definition's on those logits and
    the step's random numbers, to the last one."""
    from tests.test_verify_gpu import outcomes
    m = model_of(F32)
    d = model_of(F32, std=0.075) if "model" in how else None
    T, more = (0.0 if "greedy" in how else 0.9), dict(top_k=9) if how == "filter" else {}
    prompts, samples, K, n_new, V = [[5, 17, 3, 5, 17], ids_of(33, seed=2).tolist()], 2, 3, 14, 96
    g = torch.Generator(device="cuda").manual_seed(4)
    u = torch.rand((n_new, 4, (2 if d else 1) * K + 1), generator=g, device="cuda")
    run = dict(temperature=T, draft=d, samples=samples, page_size=16, **more)
    eos = m.generate_drafted(prompts, u, K, **run)[0][6] if ends else None
    log, dlog = [], []
    recorded(m, log)
    if d:
        recorded(d, dlog)
    steps = list(m.draft_steps(prompts, u, K, eos=eos, **run))
    log = iter(log)
    un = u.double().cpu().numpy()

    def drawn(row, at, got, **more):
        """Whether got is what the row [V] gives for the random number u[at]."""
        if T == 0.0:
            return got == V - 1 - int(row.flip(0).argmax())
        if more:
            return got == int(ops.sample_rows(row[None], u[at].reshape(1), T, **more))
        x = row.double().cpu().numpy()
        return got in outcomes(np.stack([x, x]), [-1], [0.0, un[at]], None, T)[0]

    ids, rows = next(log)
    assert ids == prompts
    for p, row in zip(prompts, rows):
        assert off(row, m.forward(torch.tensor([p], device="cuda"))[0, -1]) < CLOSE
    texts = [list(p) for p in prompts for _ in range(samples)]
    if d:
        assert dlog.pop(0)[0] == prompts
    held = [len(t) for t in texts]  # of the draft model's keys
    for b in range(4):
        assert len(steps[0][b]) == 1 and drawn(rows[b // samples], (0, b, K), steps[0][b][0], **more)
    made, live, text0 = [[] for _ in range(4)], list(range(4)), [len(t) for t in texts]

    def take(step):
        for b in list(live):
            new = steps[step][b]
            assert new and len(made[b]) + len(new) <= n_new and (eos is None or eos not in new[:-1])
            made[b] += new
            texts[b] += new
            if len(made[b]) == n_new or new[-1] == eos:
                live.remove(b)

    take(0)
    step = 1
    while live:
        now = list(live)
        room = [min(K, n_new - len(made[b]) - 1) for b in now]
        k, q = max(room), None
        if d is None:
            guess = [llama.lookup_drafts(texts[b], r) for b, r in zip(now, room)]
            k = max(len(x) for x in guess)
        elif k:
            guess, q = [[] for _ in now], [[] for _ in now]
            for j in range(k):
                ids, rows = dlog.pop(0)
                for i, b in enumerate(now):
                    assert ids[i] == (guess[i][-1:] if j else texts[b][held[b]:])
                    whole = texts[b] + guess[i]
                    assert off(rows[i], d.forward(torch.tensor([whole], device="cuda"))[0, -1]) < CLOSE
                    q[i].append(rows[i])
                    if j + 1 < k:  # what was drawn: the next pass holds it, the last one's the check
                        guess[i].append(dlog[0][0][i][-1])
            held = [held[b] if b not in now else len(texts[b]) + k - 1 for b in range(4)]
        ids, rows = next(log)
        at = 0
        for i, b in enumerate(now):
            if d is not None and k:
                mine = ids[i][1:1 + room[i]]
                assert mine[:len(guess[i])] == guess[i][:room[i]]
                for j, t in enumerate(mine):
                    assert drawn(q[i][j], (step, b, K + 1 + j), t)
            else:
                mine = guess[i] if k else []
            assert ids[i] == texts[b][-1:] + mine + [0] * (k - len(mine))
            x = rows[at:at + k + 1]
            at += k + 1
            whole = m.forward(torch.tensor([texts[b] + mine], device="cuda"))[0, len(texts[b]) - 1:]
            for r in range(len(mine) + 1):
                assert off(x[r], whole[r]) < CLOSE
            new = steps[step][b]
            if more or T == 0.0:
                for r, t in enumerate(new):
                    uu = (step, b, r) if r < k else (step, b, K)
                    assert drawn(x[r], uu, t, **more)
                n = len(new) - 1
                assert new[:n] == mine[:n]
                assert len(new) == len(mine) + 1 or new[n] != mine[n] or new[n] == eos
            else:
                xs = x.double().cpu().numpy()
                ys = None if q is None else np.stack([z.double().cpu().numpy() for z in q[i][:k]])
                row = mine + [-1] * (k - len(mine))
                may = outcomes(xs, row, np.append(un[step, b, :k], un[step, b, K]), ys, T)
                n = len(new) - 1
                assert new[:n] == mine[:n]
                assert (n in may and new[n] in may[n]) or (n < len(mine) and new[n] == mine[n] == eos)
            if d is not None and k:
                held[b] = min(held[b], len(texts[b]) + len(new) - 1)
        take(step)
        assert all(steps[step][b] == [] for b in range(4) if b not in now)
        step += 1
    assert step == len(steps) and next(log, None) is None and not dlog
    for b in range(4):
        assert len(made[b]) == n_new or made[b][-1] == eos
        assert texts[b] == (prompts[b // samples] + made[b]) and text0[b] == len(prompts[b // samples])
