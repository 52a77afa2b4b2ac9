"""The plan of shared-prefix decode attention (CPU): which runs of blocks it finds, and that its
items and references cover every cached position of every sequence exactly once."""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch

import augur_b200 as ab
from augur_b200 import attention
from augur_b200.attention import SharedPrefixTables, paged_shared_prefix_attention


@pytest.fixture(autouse=True)
def every_run_counts(monkeypatch):
    """Runs are taken apart however little reading they spare, so that small cases reach the shared kernels."""
    monkeypatch.setattr(attention, "_MIN_SAVED_BYTES", 0)


def _pool(bs, num_blocks, kv_heads=2, dim=64):
    shape = (1, num_blocks, kv_heads, bs, dim)
    return ab.PagedKVCache(keys=torch.zeros(shape), values=torch.zeros(shape), block_size=bs,
                           allocator=ab.BlockAllocator(num_blocks))


def _tables(bs, rows):
    return [ab.SequenceBlockTable(block_ids=list(ids), block_size=bs, seq_len=n) for ids, n in rows]


def _covered_keys(plan, pool, tables, heads):
    """For every (sequence, KV head): the (block, row) keys its references and own part attend to,
    read from the plan's device arrays as the kernels read them."""
    bs, groups = pool.block_size, heads // pool.keys.shape[2]
    items = plan._dev["items"].view(-1, 12).tolist()
    members, run_blocks = plan._dev["members"].tolist(), plan._dev["run_blocks"].tolist()
    starts, refs = plan._dev["starts"].tolist(), plan._dev["refs"].view(-1, 4).tolist()
    slabs = {}  # slab -> (item, tile's first row)
    for it in items:
        for slab, row0 in ((it[8], it[5]), (it[9], it[5] + 128)):
            if slab >= 0:
                assert slab not in slabs and slab < plan.n_slabs
                slabs[slab] = (it, row0)
    assert len(slabs) == plan.n_slabs
    for b, t in enumerate(tables):
        for h in range(pool.keys.shape[2]):
            for g in range(groups):
                keys = []
                for base, ranges, place, tiles in refs[starts[b]:starts[b + 1]]:
                    row = place * groups + g
                    for c in range(ranges):
                        it, row0 = slabs[base + (h * tiles + row // 128) * ranges + c]
                        assert it[4] == h and row0 == row // 128 * 128 and row < it[1] and it[6] % 128 == 0
                        assert members[it[0] + row // groups] == b
                        assert it[6] < it[7] <= it[3] * bs
                        keys += [(run_blocks[it[2] + p // bs], p % bs) for p in range(it[6], it[7])]
                own = range(int(plan._dev["shared"][b]), t.seq_len)
                keys += [(t.block_ids[p // bs], p % bs) for p in own]
                want = [(t.block_ids[p // bs], p % bs) for p in range(t.seq_len)]
                assert keys == want, (b, h, g)


def test_forks_of_one_prompt_are_one_run():
    bs = 16
    pool = _pool(bs, 200)
    common = list(range(40))
    tables = _tables(bs, [(common + [100 + i], 40 * bs + 1 + i) for i in range(5)])
    plan = SharedPrefixTables(pool, tables, 14)
    assert plan.runs == [([0, 1, 2, 3, 4], 0, 640)]
    assert plan.shared_lens.tolist() == [640] * 5 and plan.max_own_len == 5
    _covered_keys(plan, pool, tables, 14)


def test_nested_prefixes_and_unlike_orders():
    bs = 16
    pool = _pool(bs, 400)
    system = list(range(64))
    a, b = system + list(range(100, 140)), system + list(range(200, 232))
    rows = [(a + [300], 104 * bs + 3), (b + [301], 96 * bs + 1), (a + [302], 104 * bs + 16), (b + [303], 97 * bs),
            (list(range(310, 320)), 155), (system + [330], 64 * bs + 9)]
    tables = _tables(bs, rows)
    plan = SharedPrefixTables(pool, tables, 14)
    assert sorted(plan.runs) == [([0, 1, 2, 3, 5], 0, 1024), ([0, 2], 1024, 1664), ([1, 3], 1024, 1536)]
    assert plan.shared_lens.tolist() == [1664, 1536, 1664, 1536, 0, 1024]
    _covered_keys(plan, pool, tables, 14)


def test_a_short_common_start_joins_the_runs_behind_it():
    bs = 16
    pool = _pool(bs, 400)
    short = [0, 1]
    a, b = short + list(range(100, 140)), short + list(range(200, 240))
    tables = _tables(bs, [(x + [300 + i], 42 * bs + 2) for i, x in enumerate((a, a, b, b))])
    plan = SharedPrefixTables(pool, tables, 14)
    assert sorted(plan.runs) == [([0, 1], 0, 672), ([2, 3], 0, 672)]
    _covered_keys(plan, pool, tables, 14)


@pytest.mark.parametrize("rows", [
    [],                                                            # no sequence
    [(list(range(30)), 470)],                                      # one
    [(list(range(30)), 470), (list(range(40, 70)), 470)],          # nothing in common
    [([0, 1], 32), ([0, 2], 32)],                                  # too little in common
    [([], 0), (list(range(30)), 480), (list(range(30)), 480)],     # an empty sequence beside a shared run
    [(list(range(30)), 480), (list(range(30)), 100), (list(range(30)), 480)],  # a shorter holder ends the run
    [(list(range(30)), 479), (list(range(30)), 479)],              # the partly filled block is not part of it
])
def test_degenerate_batches(rows):
    pool = _pool(16, 100)
    tables = _tables(16, rows)
    plan = SharedPrefixTables(pool, tables, 14)
    assert (plan.shared_lens <= np.asarray([t.seq_len for t in tables])).all()
    _covered_keys(plan, pool, tables, 14)


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("heads,kv_heads,bs", [(14, 2, 16), (32, 8, 32), (16, 16, 8), (8, 1, 12)])
def test_random_forks_cover_every_position_once(seed, heads, kv_heads, bs):
    r = random.Random(seed * 100 + heads)
    pool = _pool(bs, 6000, kv_heads)
    fresh = iter(r.sample(range(6000), 6000))
    rows = [([], 0)]
    for _ in range(r.randint(1, 30)):
        ids, n = r.choice(rows)  # a fork: the parent's full blocks, then its own
        ids = ids[: n // bs]
        n = len(ids) * bs + r.randint(0, 400)
        rows.append((ids + [next(fresh) for _ in range(-(-n // bs) - len(ids))], n))
    r.shuffle(rows)
    tables = _tables(bs, rows)
    _covered_keys(SharedPrefixTables(pool, tables, heads), pool, tables, heads)


def test_refusals():
    pool = _pool(16, 100)
    tables = _tables(16, [(list(range(30)), 470)])
    with pytest.raises(ValueError, match="multiple of the cache's KV heads"):
        SharedPrefixTables(pool, tables, 13)
    with pytest.raises(ValueError, match="block_size"):
        SharedPrefixTables(pool, _tables(8, [([0], 3)]), 14)
    with pytest.raises(ValueError, match="capacity"):
        SharedPrefixTables(pool, _tables(16, [([0], 17)]), 14)
    with pytest.raises(ValueError, match="same length"):
        SharedPrefixTables(pool, tables, 14, seq_lens=[1, 2])
    with pytest.raises(ValueError, match="no CPU fallback"):
        paged_shared_prefix_attention(torch.zeros(1, 14, 64), pool, 0, tables)
    with pytest.raises(ValueError, match="one query token"):
        paged_shared_prefix_attention(torch.zeros(1, 14, 2, 64), pool, 0, tables)
    with pytest.raises(ValueError, match="kernel must be"):
        paged_shared_prefix_attention(torch.zeros(1, 14, 64), pool, 0, tables, kernel="mma")


def test_runs_must_spare_enough_reading():
    pool = _pool(16, 200)
    common = list(range(40))
    tables = _tables(16, [(common + [100 + i], 641 + i) for i in range(5)])
    spared = 4 * 640 * 2 * 64 * 2 * 4  # sequences, positions, KV heads, dims, K and V, bytes
    assert SharedPrefixTables(pool, tables, 14, min_saved_bytes=spared).runs == [([0, 1, 2, 3, 4], 0, 640)]
    plan = SharedPrefixTables(pool, tables, 14, min_saved_bytes=spared + 1)
    assert plan.runs == [] and not plan.shared_lens.any() and plan.max_own_len == 645
    _covered_keys(plan, pool, tables, 14)
