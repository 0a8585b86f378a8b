"""The host side of the cache in pages: tables, shared pages, copies before a write,
truncation and compaction against a model that keeps each sequence's keys as a list."""
import random

import pytest
import torch

from teenyformers_amd import generate, llama, ops

CFG = llama.LlamaConfig(d_model=8, n_heads=1, n_layers=2, vocab_size=16, intermediate_size=8, n_kv_heads_=1)


def copy_pages(pages, src, dst):
    """What ops.copy_pages does, on the host, with its refusals."""
    assert len(src) == len(dst) and len(set(dst)) == len(dst) and not set(src) & set(dst)
    pages[..., dst, :, :, :] = pages[..., src, :, :, :]
    return pages


@pytest.fixture
def cache(monkeypatch):
    monkeypatch.setattr(ops, "copy_pages", copy_pages)
    return llama.PagedKVCache(CFG, 40, 16, torch.float32, "cpu")


def write(cache, seqs, values):
    """values[i] as the next keys of seqs[i]: one number a key, in all layers."""
    counts = [len(v) for v in values]
    cache.reserve(seqs, counts)
    b = cache.batch(seqs, counts)
    assert b.starts.tolist() == [sum(counts[:i]) for i in range(len(counts) + 1)]
    assert b.n_past.tolist() == [cache.lengths[s] for s in seqs]
    assert b.max_new == max(counts) and b.max_keys == max(p + n for p, n in zip(b.n_past.tolist(), counts))
    for i, (s, v) in enumerate(zip(seqs, values)):
        for j, x in enumerate(v):
            at = int(b.n_past[i]) + j
            cache.pages[:, :, int(b.table[i, at // 16]), :, at % 16] = x
        cache.lengths[s] += len(v)


def read(cache, seq):
    return [float(cache.pages[0, 1, cache.tables[seq][i // 16], 0, i % 16, 0]) for i in range(cache.lengths[seq])]


def consistent(cache):
    uses = [0] * len(cache._uses)
    for seq, table in cache.tables.items():
        assert len(table) == -(-cache.lengths[seq] // 16)
        for page in table:
            uses[page] += 1
    assert uses == cache._uses
    assert sorted(cache._free) == [i for i, n in enumerate(uses) if n == 0]


@pytest.mark.parametrize("seed", range(12))
def test_random_use(cache, seed):
    rng = random.Random(seed)
    want, counter = {}, iter(range(10 ** 6))
    for _ in range(150):
        what = rng.choice(["add", "fork", "write", "write", "write", "write", "truncate", "remove", "compact"])
        seqs = list(want)
        if what == "add" and len(seqs) < 8:
            want[cache.add()] = []
        elif what == "fork" and seqs and len(seqs) < 8:
            s = rng.choice(seqs)
            for f in cache.fork(s, rng.randint(1, 2)):
                want[f] = list(want[s])
        elif what == "write" and seqs:
            some = rng.sample(seqs, rng.randint(1, len(seqs)))
            values = [[float(next(counter)) for _ in range(rng.choice([0, 1, 1, 3, 17, 40]))] for _ in some]
            if not any(values):
                continue
            state = [list(t) for t in cache.tables.values()], list(cache._uses), sorted(cache._free)
            try:
                write(cache, some, values)
            except RuntimeError:  # full: nothing has changed
                assert state == ([list(t) for t in cache.tables.values()], list(cache._uses), sorted(cache._free))
                continue
            for s, v in zip(some, values):
                want[s] += v
        elif what == "truncate" and seqs:
            s = rng.choice(seqs)
            n = rng.randint(0, len(want[s]))
            cache.truncate(s, n)
            want[s] = want[s][:n]
        elif what == "remove" and seqs:
            s = rng.choice(seqs)
            cache.remove(s)
            del want[s]
        elif what == "compact":
            n = cache.compact()
            assert all(p < n for t in cache.tables.values() for p in t) and n == len(cache._uses) - cache.free_pages
        consistent(cache)
        for s, v in want.items():
            assert read(cache, s) == v


def test_shared_pages_are_stored_once(cache):
    s = cache.add()
    write(cache, [s], [[float(i) for i in range(40)]])
    forks = cache.fork(s, 5)
    assert cache.free_pages == 37
    write(cache, forks, [[100.0 + f] for f in forks])  # the last page of each, not the full ones
    assert cache.free_pages == 32
    write(cache, [s], [[1.0]])  # its last page is its own by now
    assert cache.free_pages == 32
    for f in forks:
        cache.remove(f)
    assert cache.free_pages == 37


def test_refusals(cache):
    with pytest.raises(ValueError):
        llama.PagedKVCache(CFG, 0, 16, device="cpu")
    for size in (8, 24, 2048):
        with pytest.raises(ValueError):
            llama.PagedKVCache(CFG, 4, size, device="cpu")
    s = cache.add()
    for seqs, counts in (([s, s], [1, 1]), ([s], [1, 2]), ([s], [-1])):
        with pytest.raises(ValueError):
            cache.reserve(seqs, counts)
    with pytest.raises(ValueError):
        cache.truncate(s, 1)
    with pytest.raises(RuntimeError, match="free pages"):
        cache.reserve([s], [16 * 41])
    with pytest.raises(KeyError):
        cache.reserve([99], [1])
    m = llama.Llama(CFG, {})
    for seqs, ids in (([], []), ([s], [[1], [2]]), ([s], [[]])):
        with pytest.raises(ValueError):
            m.run_paged(cache, seqs, ids)
    u = torch.zeros((4, 2, 4))
    for kw in (dict(prompts=[]), dict(prompts=[[1]]), dict(n_draft=2), dict(n_draft=0), dict(samples=2),
               dict(u=u.double()), dict(prompts=[[1], []]), dict(draft=m),
               dict(draft=llama.Llama(llama.LlamaConfig(vocab_size=17), {}), u=torch.zeros((4, 2, 7)))):
        a = dict(prompts=[[1], [2]], u=u, n_draft=3)
        a.update(kw)
        with pytest.raises(ValueError):
            next(m.draft_steps(**a))


def test_forks_are_counted(cache):
    s = cache.add()
    write(cache, [s], [[1.0] * 20])
    with pytest.raises(ValueError):
        cache.fork(s, -1)
    assert cache.fork(s, 0) == []
    cache.remove(s)
    assert cache.free_pages == len(cache._uses)


@pytest.mark.parametrize("text,n,want", [
    ([1, 2, 3, 9, 1, 2, 3], 2, [9, 1]), ([1, 2, 3, 9, 1, 2, 3], 9, [9, 1, 2, 3]), ([5, 1, 5, 2, 5], 1, [2]),
    ([1, 2, 3], 4, []), ([7], 3, []), ([7, 7], 3, [7]), ([1, 2, 1], 0, [])])
def test_lookup_drafts(text, n, want):
    assert llama.lookup_drafts(text, n) == want


def test_command_refuses(capsys):
    for bad in (["--draft-len", "-1"], ["--draft-len", "65"], ["--draft-dir", "x"],
                ["--preset", "llama3-8b", "--draft-len", "4"]):
        with pytest.raises(SystemExit):
            generate.main(["--model-dir", "unread", *bad])


def test_default_temperature_with_drafts(monkeypatch):
    """Drafts change nothing about what is drawn: greedy unless asked otherwise."""
    seen = []
    monkeypatch.setattr(generate, "generate_text", lambda args: seen.append((args.temperature, args.on_device)) or 0)
    assert generate.main(["--model-dir", "unread", "--draft-len", "4"]) == 0
    assert seen == [(0.0, True)]


def state_of(cache):
    return ({s: list(t) for s, t in cache.tables.items()}, dict(cache.lengths), list(cache._uses),
            sorted(cache._free), cache.pages.clone())


def same_state(a, b):
    return a[:4] == b[:4] and torch.equal(a[4], b[4])


def counted(cache):
    """Uses and free pages are those of the tables, which may hold more than their keys need."""
    uses = [0] * len(cache._uses)
    for seq, table in cache.tables.items():
        assert len(table) >= -(-cache.lengths[seq] // 16)
        for page in table:
            uses[page] += 1
    assert uses == cache._uses
    assert sorted(cache._free) == [i for i, n in enumerate(uses) if n == 0]


@pytest.fixture
def small(monkeypatch):
    monkeypatch.setattr(ops, "copy_pages", copy_pages)
    c = llama.PagedKVCache(CFG, 8, 16, torch.float32, "cpu")
    c.pages.zero_()
    return c


def test_pages_held_ahead_are_not_others_room(small):
    """A sequence that holds more pages than a call needs brings none to the others of the call."""
    a, b = small.add(), small.add()
    small.reserve([a], [96])
    was = state_of(small)
    with pytest.raises(RuntimeError, match="free pages"):
        small.reserve([a, b], [1, 64])
    assert same_state(was, state_of(small))
    small.reserve([a, b], [1, 32])
    assert small.free_pages == 0 and len(small.tables[a]) == 6 and len(small.tables[b]) == 2
    counted(small)


def test_no_room_leaves_a_fork_its_page(small):
    """... nor takes it a fork's page away before the copy."""
    a, b = small.add(), small.add()
    write(small, [a], [[1.0, 2.0]])
    small.reserve([a], [62])
    (f,) = small.fork(a)
    was = state_of(small)
    with pytest.raises(RuntimeError, match="free pages"):
        small.reserve([a, f, b], [1, 1, 64])
    assert same_state(was, state_of(small))
    assert read(small, f) == [1.0, 2.0]


def test_forks_of_pages_held_ahead(small):
    """Shared pages that a call does not write to are not copied by it, but by the one that does."""
    a = small.add()
    write(small, [a], [[float(i) for i in range(20)]])
    small.reserve([a], [40])  # four pages, two without a key
    (f,) = small.fork(a)
    write(small, [f], [[100.0]])  # the second page alone
    assert small.free_pages == 3 and small.tables[f][2:] == small.tables[a][2:]
    write(small, [f, a], [[101.0] * 15, [200.0] * 15])  # ... and the third of each
    counted(small)
    assert read(small, f) == [float(i) for i in range(20)] + [100.0] + [101.0] * 15
    assert read(small, a) == [float(i) for i in range(20)] + [200.0] * 15


def test_a_pass_that_raises_behind_its_room(small, monkeypatch):
    """run_paged reserves before it runs: after an error the keys are as they were and the pages count."""
    m = llama.Llama(CFG, {})
    a, b = small.add(), small.add()
    write(small, [a], [[1.0, 2.0, 3.0]])
    monkeypatch.setattr(m, "hidden", lambda *_: (_ for _ in ()).throw(TypeError("mixed types")))
    with pytest.raises(TypeError):
        m.run_paged(small, [a, b], [[1] * 60, [2]])
    assert small.lengths == {a: 3, b: 0} and read(small, a) == [1.0, 2.0, 3.0]
    counted(small)
    was = state_of(small)
    with pytest.raises(RuntimeError, match="free pages"):
        small.reserve([a, b], [1, 6 * 16])
    assert same_state(was, state_of(small))
    small.truncate(a, 3)
    assert small.free_pages == 6
    counted(small)


@pytest.mark.parametrize("seed", range(8))
def test_random_use_with_room_ahead(cache, seed):
    """As test_random_use, with pages reserved ahead, shared, given back and asked for in vain."""
    rng = random.Random(1000 + seed)
    want, counter = {}, iter(range(10 ** 6))
    for _ in range(200):
        what = rng.choice(["add", "fork", "write", "write", "write", "ahead", "ahead", "truncate", "remove", "compact"])
        seqs = list(want)
        was = state_of(cache)
        if what == "add" and len(seqs) < 8:
            want[cache.add()] = []
        elif what == "fork" and seqs and len(seqs) < 8:
            s = rng.choice(seqs)
            for f in cache.fork(s, rng.randint(1, 2)):
                want[f] = list(want[s])
        elif what in ("write", "ahead") and seqs:
            some = rng.sample(seqs, rng.randint(1, len(seqs)))
            counts = [rng.choice([0, 1, 1, 3, 17, 40, 150]) for _ in some]
            try:
                if what == "ahead":
                    cache.reserve(some, counts)
                elif max(counts) > 0:
                    values = [[float(next(counter)) for _ in range(n)] for n in counts]
                    write(cache, some, values)
                    for s, v in zip(some, values):
                        want[s] += v
            except RuntimeError:
                assert [x for x in was[:4]] == [x for x in state_of(cache)[:4]]
        elif what == "truncate" and seqs:
            s = rng.choice(seqs)
            n = rng.randint(0, len(want[s]))
            cache.truncate(s, n)
            want[s] = want[s][:n]
        elif what == "remove" and seqs:
            s = rng.choice(seqs)
            cache.remove(s)
            del want[s]
        elif what == "compact":
            n = cache.compact()
            assert all(p < n for t in cache.tables.values() for p in t) and n == len(cache._uses) - cache.free_pages
        counted(cache)
        for s, v in want.items():
            assert read(cache, s) == v


def test_draft_settings_are_numbers():
    """The batch of a run of drafts shrinks as sequences end: settings of each sequence are refused
    before anything runs, not when the first one has ended."""
    m = llama.Llama(CFG, {})
    for kw in (dict(temperature=torch.ones(2)), dict(top_k=torch.ones(2, dtype=torch.int32)),
               dict(top_p=torch.ones(2)), dict(min_p=torch.zeros(2))):
        with pytest.raises(ValueError, match="are numbers"):
            next(m.draft_steps([[1], [2]], torch.zeros((4, 2, 4)), 3, **kw))
