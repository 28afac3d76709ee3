"""PagePool on the CPU: what a sequence reads through its pages is what was written for it, whatever is
forked, truncated, freed, copied and moved in between; nothing changes where pages run out."""
import numpy as np
import pytest
import torch

from vllm_sly_radiance_amd import kv4_pool
from vllm_sly_radiance_amd import radiance_kv4 as K
from vllm_sly_radiance_amd.kv4_pool import PagePool


@pytest.fixture
def pool(monkeypatch):
    """A pool of 12 pages of 16 tokens on the CPU, with `store`: what stands at each slot."""
    p = PagePool(K.new_cache(12, 1, 16, 64, device="cpu", layers=2))
    p.store = np.full((12, 16), -1, np.int64)
    p.moved = []

    def move(cache, pairs, page_table=None):
        assert cache is p.cache and pairs.dtype == torch.int32 and pairs.device.type == "cpu"
        pairs = pairs.tolist()
        src, dst = {a for a, _ in pairs}, {b for _, b in pairs}
        assert not src & dst and len(dst) == len(pairs)
        for a, b in pairs:
            p.store[b] = p.store[a]
            if page_table is not None:
                page_table[page_table == a] = b
        p.moved += pairs
    monkeypatch.setattr(kv4_pool._kv4, "move_pages", move)
    return p


def write(pool, step, names):
    slots = step.slots.numpy()
    assert len(set(slots.tolist())) == len(slots)
    pool.store.reshape(-1)[slots] = names


def read(pool, seq):
    n = pool.length(seq)
    at = np.arange(n)
    pages = np.asarray(pool.pages_of(seq), np.int64)
    assert len(pages) == -(-n // 16)
    return pool.store[pages[at // 16], at % 16].tolist() if n else []


def test_step_of_a_batch(pool):
    a, b, c = pool.add(), pool.add(), pool.add()
    pool.extend([b], [15])
    step = pool.extend([a, b, c], [17, 3, 0])
    assert step.q_starts.tolist() == [0, 17, 20, 20] and step.seq_lens.tolist() == [17, 18, 0]
    assert (step.max_q, step.max_len) == (17, 18) and step.page_table.shape == (3, 2)
    assert step.positions.tolist() == list(range(17)) + [15, 16, 17]
    assert pool.pages_of(b) == [0, 3] and pool.pages_of(a) == [1, 2]
    assert step.page_table.tolist() == [[1, 2], [0, 3], [-1, -1]]
    assert step.slots.tolist() == list(range(16, 33)) + [15, 48, 49]
    assert step.slots.dtype == step.positions.dtype == torch.int64
    assert all(t.dtype == torch.int32 for t in step.attention[:3])
    empty = pool.extend([], [])
    assert empty.slots.shape == (0,) and empty.q_starts.tolist() == [0] and empty.max_q == 0


def test_fork_copies_only_what_is_written(pool):
    a = pool.add()
    write(pool, pool.extend([a], [20]), np.arange(20))
    b, c, whole = pool.fork(a), pool.fork(a), pool.fork(a, 16)
    assert pool.free_pages == 10
    step = pool.extend([a, b, c, whole], [1, 1, 1, 1])
    # two of the three that share the second page copy it, the last keeps it; a full page is shared on
    assert [x for x, _ in pool.moved] == [1, 1] and pool.free_pages == 7
    write(pool, step, [100, 101, 102, 103])
    for s, last in ((a, 100), (b, 101), (c, 102)):
        assert read(pool, s) == list(range(20)) + [last]
    assert read(pool, whole) == list(range(16)) + [103]
    for s in (a, b, c, whole):
        pool.free(s)
    assert pool.free_pages == 12


def test_nothing_changes_where_pages_run_out(pool):
    a, b = pool.add(), pool.add()
    pool.extend([a], [170])
    c = pool.fork(a)
    before = (pool.free_pages, pool.pages_of(a), pool.length(a), pool.length(b))
    with pytest.raises(RuntimeError, match="2 pages needed, 1 of 12 free"):
        pool.extend([a, b], [1, 16])
    assert (pool.free_pages, pool.pages_of(a), pool.length(a), pool.length(b)) == before
    assert not pool.moved
    pool.free(c)
    pool.extend([a, b], [1, 16])


def test_refusals(pool):
    a = pool.add()
    pool.extend([a], [5])
    for call, what in ((lambda: pool.extend([a, a], [1, 1]), "extend"),
                       (lambda: pool.extend([a], [1, 2]), "extend"),
                       (lambda: pool.extend([a], [-1]), "extend by"),
                       (lambda: pool.fork(a, 6), "fork of 6"), (lambda: pool.fork(7), "no sequence 7"),
                       (lambda: pool.truncate(a, 6), "truncate to 6"),
                       (lambda: pool.truncate(a, -1), "truncate to -1"),
                       (lambda: PagePool(torch.zeros(3)), "cache must be")):
        with pytest.raises(RuntimeError, match=what):
            call()
    pool.free(a)
    with pytest.raises(RuntimeError, match="no sequence"):
        pool.length(a)


def test_compaction_moves_shared_pages_once_and_remaps_a_table(pool):
    a, b = pool.add(), pool.add()
    pool.extend([a], [48])
    write(pool, pool.extend([b], [40]), np.arange(40))
    c = pool.fork(b)
    table = torch.tensor([pool.pages_of(b), pool.pages_of(c)], dtype=torch.int32)
    pool.free(a)
    assert pool.compact(table) == 3 and pool.pages_of(b) == pool.pages_of(c)
    assert sorted(pool.pages_of(b)) == [0, 1, 2] and pool.free_pages == 9
    assert table.tolist() == [pool.pages_of(b)] * 2
    assert read(pool, b) == read(pool, c) == list(range(40))
    assert pool.compact() == 0


@pytest.mark.parametrize("seed", range(6))
def test_random_use_keeps_every_sequence(pool, seed):
    rng = np.random.default_rng(seed)
    want, name = {}, 0
    for _ in range(300):
        ids = list(want)
        what = rng.integers(0, 10)
        if what < 2 and len(ids) < 6:
            want[pool.add()] = []
        elif what < 4 and ids and len(ids) < 6:
            s = int(rng.choice(ids))
            n = int(rng.integers(0, len(want[s]) + 1))
            want[pool.fork(s, n)] = want[s][:n]
        elif what == 4 and ids:
            s = int(rng.choice(ids))
            n = int(rng.integers(0, len(want[s]) + 1))
            pool.truncate(s, n)
            want[s] = want[s][:n]
        elif what == 5 and ids:
            s = int(rng.choice(ids))
            pool.free(s)
            del want[s]
        elif what == 6:
            pool.compact()
            used = {p for s in want for p in pool.pages_of(s)}
            assert used == set(range(len(used)))
        elif ids:
            some = [int(s) for s in rng.permutation(ids)[:rng.integers(1, len(ids) + 1)]]
            counts = [int(n) for n in rng.integers(0, 12, len(some))]
            try:
                step = pool.extend(some, counts)
            except RuntimeError as e:
                assert "pages needed" in str(e)
                continue
            names = np.arange(name, name + sum(counts))
            name += sum(counts)
            write(pool, step, names)
            for s, a, e in zip(some, step.q_starts[:-1].tolist(), step.q_starts[1:].tolist()):
                want[s] = want[s] + names[a:e].tolist()
                assert step.positions[a:e].tolist() == list(range(len(want[s]) - (e - a), len(want[s])))
        for s in want:
            assert read(pool, s) == want[s]
        assert pool.free_pages == 12 - len({p for s in want for p in pool.pages_of(s)})
