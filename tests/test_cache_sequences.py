"""PagedLatentCache's bookkeeping (sequences, forks, pages, compaction) without a GPU: the kernels' places are taken by plain writes
through the tensors that a step hands them."""
import numpy as np
import pytest
import torch

from palu_amd.kernel import paged
from palu_amd.kernel.palu_attention import LlamaPaluAttention


@pytest.fixture
def copies(monkeypatch):
    """paged_copy on the host -> the (sources, targets) of its calls"""
    calls = []

    def copy(pool, src, dst):
        assert len(src) == len(dst) and len(set(dst)) == len(dst) and not set(src) & set(dst)
        for t in pool:
            t[:, list(dst)] = t[:, list(src)]
        calls.append((list(src), list(dst)))
    monkeypatch.setattr(paged, "paged_copy", copy)
    return calls


def _cache(num_pages=8, max_seqs=4, max_pages=4, layers=2, P=16):
    return paged.PagedLatentCache(layers=layers, num_groups=2, rank_k=8, rank_v=8, num_pages=num_pages, max_seqs=max_seqs,
                                  max_pages=max_pages, page_size=P, device="cpu")


def _write(cache, tokens):
    """row t of the open step carries tokens[t] (in the keys' pair of every layer and group)"""
    st = cache._step
    assert st.seq.shape == st.pos.shape == (len(tokens),)
    for b, p, t in zip(st.seq.tolist(), st.pos.tolist(), tokens):
        page = int(st.table[b, p // cache.page_size])
        cache.pool.k_meta[:, page, :, p % cache.page_size] = float(t)


def _read(cache, seq):
    rows = [cache.pool.k_meta[:, p].permute(2, 0, 1, 3) for p in cache.pages(seq)]
    rows = torch.cat(rows)[:cache.length(seq)] if rows else torch.zeros(0, 1, 1, 1)
    assert bool((rows == rows[:, :1, :1, :1]).all())
    return [int(r) for r in rows[:, 0, 0, 0]]


def _step(cache, ids, counts, tokens):
    cache.begin(ids, counts)
    _write(cache, tokens)
    cache.commit()


def test_a_fork_shares_pages_until_one_side_writes(copies):
    c = _cache()
    a = c.add()
    _step(c, [a], 20, range(20))
    b = c.fork(a)
    assert c.pages(a) == c.pages(b) == [0, 1] and c.num_free == 6 and not copies
    _step(c, [a], 1, [100])
    assert copies == [([1], [2])] and c.pages(a) == [0, 2] and c.pages(b) == [0, 1]
    _step(c, [b], 1, [200])                                    # b is alone on its open page now
    assert len(copies) == 1
    assert _read(c, a) == [*range(20), 100] and _read(c, b) == [*range(20), 200]
    c.free(a)
    assert c.num_free == 6 and _read(c, b) == [*range(20), 200]
    c.free(b)
    assert c.num_free == 8 and c.sequences == []


def test_sharers_of_an_open_page_that_write_in_one_step(copies):
    c = _cache()
    a = c.add()
    _step(c, [a], 3, [1, 2, 3])
    b, d = c.fork(a), c.fork(a)
    _step(c, [a, b, d], 1, [4, 5, 6])
    assert copies == [([0, 0], [1, 2])]                        # two copies, the last one keeps the page
    assert (_read(c, a), _read(c, b), _read(c, d)) == ([1, 2, 3, 4], [1, 2, 3, 5], [1, 2, 3, 6])
    assert c.num_free == 5


def test_a_fork_at_a_page_boundary_copies_nothing(copies):
    c = _cache()
    a = c.add()
    _step(c, [a], 16, range(16))
    b = c.fork(a)
    _step(c, [a, b], [1, 17], [50, *range(60, 77)])
    assert not copies and _read(c, a) == [*range(16), 50] and _read(c, b) == [*range(16), *range(60, 77)]


def test_running_out_of_pages_changes_nothing(copies):
    c = _cache(num_pages=2)
    a, b = c.add(), c.add()
    _step(c, [a], 17, range(17))
    before = (c.pages(a), c.num_free)
    with pytest.raises(paged.OutOfPages, match="needs 1 pages, 0 are free"):
        c.begin([a, b])
    e = c.fork(a)
    with pytest.raises(paged.OutOfPages):
        c.begin([e])                                           # its open page is shared: the copy has no place
    assert (c.pages(a), c.num_free) == before and _read(c, a) == _read(c, e) == list(range(17))
    c.free(e)
    _step(c, [a], 1, [17])
    assert _read(c, a) == list(range(18))


def test_a_copy_that_fails_gives_its_pages_back(monkeypatch):
    c = _cache()

    def fail(*a):
        raise RuntimeError("no launch")
    a = c.add()
    _step(c, [a], 3, [1, 2, 3])
    b = c.fork(a)
    monkeypatch.setattr(paged, "paged_copy", fail)
    with pytest.raises(RuntimeError, match="no launch"):
        c.begin([b])
    assert c.num_free == 7 and c.pages(b) == [0] and c._step is None


def test_an_aborted_step_leaves_its_pages_to_the_next(copies):
    c = _cache()
    a = c.add()
    c.begin([a], 40)
    c.abort()
    assert c.length(a) == 0 and c.pages(a) == [] and c.num_free == 5
    b = c.fork(a)                                              # of nothing: shares nothing
    _step(c, [b, a], [2, 40], [7, 8, *range(40)])
    assert c.num_free == 4 and _read(c, a) == list(range(40)) and _read(c, b) == [7, 8]
    c.free(a)
    c.free(b)
    assert c.num_free == 8


def test_compaction_and_resize(copies):
    c = _cache()
    ids = [c.add() for _ in range(4)]
    for i in ids:
        _step(c, [i], 20, range(100 * i, 100 * i + 20))
    f = c.fork(ids[3])
    c.free(ids[0])
    c.free(ids[2])
    with pytest.raises(ValueError, match="pages up to 7 are in use"):
        c.resize(4)
    copies.clear()
    assert c.compact() == 4 and len(copies) == 1 and sorted(copies[0][1]) == [0, 1]
    assert sorted(c.pages(ids[1]) + c.pages(ids[3])) == [0, 1, 2, 3] and c.pages(f) == c.pages(ids[3])
    c.resize(5)
    assert c.pool.num_pages == 5 and c.num_free == 1
    for i in (ids[1], ids[3]):
        assert _read(c, i) == list(range(100 * i, 100 * i + 20))
    assert _read(c, f) == _read(c, ids[3])
    _step(c, [f], 1, [9])
    c.resize(30)
    assert c.num_free == 25 and _read(c, f) == [*range(300, 320), 9] and _read(c, ids[3]) == list(range(300, 320))
    assert c.compact() == 5 and len(copies) == 2               # (the open page's copy; nothing had to move)


def test_steps_and_ids_are_checked(copies):
    c = _cache()
    a = c.add()
    for call in (c.commit, c.abort, lambda: c.append(0, None, None), lambda: c.attend(0, None, None), lambda: c.adopt(0, None)):
        with pytest.raises(RuntimeError, match="no step is open"):
            call()
    for bad in ([], [a, a], list(range(5))):
        with pytest.raises(ValueError):
            c.begin(bad)
    for counts in (0, -1, [1, 1], []):
        with pytest.raises(ValueError):
            c.begin([a], counts)
    with pytest.raises(ValueError, match="its 4 pages hold 64"):
        c.begin([a], 65)
    with pytest.raises(KeyError):
        c.begin([a, 99])
    c.begin([a], np.int64(64))
    with pytest.raises(ValueError, match="one token of each"):
        c.attend(0, None, None)
    for call in (lambda: c.begin([a]), lambda: c.fork(a), lambda: c.free(a), c.compact, lambda: c.resize(9)):
        with pytest.raises(RuntimeError, match="a step is open"):
            call()
    c.commit()
    c.free(a)
    for call in (c.free, c.fork, c.length, c.pages):
        with pytest.raises(KeyError):
            call(a)
    assert c.add() != a and len(c) == 2
    for kw in (dict(layers=0), dict(max_seqs=0), dict(max_pages=0), dict(num_pages=0)):
        with pytest.raises(ValueError):
            _cache(**kw)


def test_decode_steps_keep_their_addresses(copies):
    c = _cache(max_seqs=3)
    a, b = c.add(), c.add()
    seen = []
    for n in ([1, 1], [1, 1], [30, 2], [1, 1]):
        c.begin([a, b], n)
        st = c._step
        assert st.lens.tolist() == [c.length(a) + n[0], c.length(b) + n[1]] and st.table.shape == (2, 4)
        if n == [1, 1]:
            seen.append([t.data_ptr() for t in (st.lens, st.seq, st.pos, st.table)])
        _write(c, range(sum(n)))
        c.commit()
    assert seen[0] == seen[1] == seen[2]


@pytest.mark.parametrize("seed", range(6))
def test_random_lives_of_many_sequences(copies, seed):
    """adds, steps, aborted steps, forks, ends, compactions and resizes in random order against lists of tokens"""
    r = np.random.default_rng(seed)
    c = _cache(num_pages=20, max_seqs=5, max_pages=4)
    want, stamp = {}, 0
    for _ in range(300):
        act = r.choice(["add", "step", "step", "step", "abort", "fork", "free", "compact", "resize"])
        ids = list(want)
        if act == "add":
            want[c.add()] = []
        elif act in ("step", "abort") and ids:
            pick = [int(i) for i in r.permutation(ids)[:r.integers(1, 6)]]
            counts = [int(n) for n in r.integers(1, 1 + r.choice([1, 20]), len(pick))]
            state = (c.num_free, {i: c.pages(i) for i in ids})
            try:
                c.begin(pick, counts)
            except (paged.OutOfPages, ValueError):
                assert state == (c.num_free, {i: c.pages(i) for i in ids})
                continue
            tokens = list(range(stamp % 1500, stamp % 1500 + sum(counts)))      # (fp16 holds them exactly)
            stamp += sum(counts)
            _write(c, tokens)
            if act == "abort":
                c.abort()
                continue
            c.commit()
            for i, n in zip(pick, counts):
                want[i] = want[i] + tokens[:n]
                tokens = tokens[n:]
        elif act == "fork" and ids:
            i = int(r.choice(ids))
            want[c.fork(i)] = want[i]
        elif act == "free" and ids:
            i = int(r.choice(ids))
            c.free(i)
            del want[i]
        elif act == "compact":
            n = c.compact()
            assert c.num_free == c.pool.num_pages - n
        elif act == "resize":
            try:
                c.resize(int(r.integers(12, 26)))
            except ValueError:
                pass
        for i, rows in want.items():
            assert c.length(i) == len(rows) and _read(c, i) == rows
        held = {p for i in want for p in c._seqs[i].row[:c._seqs[i].pages].tolist()}
        assert not held & set(c._free) and len(held) + c.num_free == c.pool.num_pages
    assert len(copies) > 3


def test_the_module_refuses_what_pages_cannot_serve(copies):
    class Config:
        hidden_size, num_attention_heads, attention_bias, group_size, num_groups = 512, 4, False, 2, 2
        total_rank_k, total_rank_v, head_dim = 16, 16, 128
    m = LlamaPaluAttention(Config, layer_idx=0)
    c = _cache()
    a, b = c.add(), c.add()
    x = torch.zeros(2, 1, 512)
    with pytest.raises(RuntimeError, match="no step is open"):
        m(x, past_key_value=c)
    c.begin([a, b])
    with pytest.raises(ValueError, match="the open step takes"):
        m(x[:1], past_key_value=c)
    with pytest.raises(NotImplementedError, match="attention weights"):
        m(x, past_key_value=c, output_attentions=True)
    with pytest.raises(NotImplementedError, match="fp16 modules"):
        m(x, past_key_value=c)
    m.layer_idx = None
    with pytest.raises(ValueError, match="layer index"):
        m(x, past_key_value=c)
