"""Shared-prefix decode attention against a plain implementation in 64 bits.

Tolerance (derived, per value): with u the unit roundoff of the cache dtype (2^-8 bf16, 2^-11
fp16, 2^-24 fp32), vmax the largest |v| and n the longest sequence,
  |out - exact| <= vmax (u + E) + u |exact|,
u vmax for rounding the probabilities, u |exact| for the output, and E the float32 work: a
score's error 2 (D + 4) 2^-24 max sum|q_i k_i| / sqrt(D) (the numerator's and the denominator's),
the exponent's argument and ex2 (|x| <= 2^7: 2^-16), summation (n + 8) 2^-24, and half-precision
probabilities below the normal range, n 2^-25.
"""

from __future__ import annotations

import math

import pytest
import torch

import augur_b200 as ab
from augur_b200 import _lib, _ops, attention
from augur_b200.attention import SharedPrefixTables, paged_decode_attention, paged_shared_prefix_attention
from tests.conftest import poison_

pytestmark = pytest.mark.gpu

_UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


@pytest.fixture(autouse=True)
def every_run_counts(monkeypatch):
    """Runs are taken apart however little reading they spare, so that small cases reach the shared kernels."""
    monkeypatch.setattr(attention, "_MIN_SAVED_BYTES", 0)


class Case:
    """A pool whose unwritten rows are NaN, and sequences given as (parent, blocks kept, length):
    each takes its parent's first blocks and fills its other positions with rows of its own."""

    def __init__(self, cuda, dtype, heads, kv_heads, dim, bs, seqs, seed=0, q_scale=1.0, rising=False, row_pad=0):
        g = torch.Generator().manual_seed(seed)
        need = sum(-(-n // bs) - kept for _, kept, n in seqs) + 4
        shape = (2, need, kv_heads, bs, dim + row_pad)
        keys, values = (poison_(torch.empty(shape, dtype=dtype, device=cuda))[..., :dim] for _ in range(2))
        ids = torch.randperm(need, generator=g).tolist()
        self.pool = ab.PagedKVCache(keys=keys, values=values, block_size=bs, allocator=ab.BlockAllocator(need))
        self.tables, self.layer = [], 1
        for parent, kept, n in seqs:
            mine = self.tables[parent].block_ids[:kept] if kept else []
            fresh = [ids.pop() for _ in range(-(-n // bs) - kept)]
            table = ab.SequenceBlockTable(block_ids=mine + fresh, block_size=bs, seq_len=n)
            at = torch.arange(kept * bs, n)
            if at.numel():
                blk, row = torch.tensor(table.block_ids)[at // bs].to(cuda), (at % bs).to(cuda)
                k = torch.randn(at.numel(), kv_heads, dim, generator=g)
                if rising:  # every tile's maximum passes the last one's
                    k = k * (0.05 + 4.0 * at.view(-1, 1, 1) / max(1, n))
                keys[self.layer][blk, :, row] = k.to(dtype).to(cuda)
                values[self.layer][blk, :, row] = torch.randn(at.numel(), kv_heads, dim, generator=g).to(dtype).to(cuda)
            self.tables.append(table)
        self.q = (torch.randn(len(seqs), heads, 1, dim, generator=g) * q_scale).to(dtype).to(cuda)

    def exact(self):
        keys, values = self.pool.keys[self.layer], self.pool.values[self.layer]
        heads, dim, bs = self.q.shape[1], self.q.shape[3], self.pool.block_size
        out, vmax, score = torch.zeros(self.q.shape, dtype=torch.float64, device=self.q.device), 0.0, 0.0
        for b, t in enumerate(self.tables):
            if t.seq_len == 0:
                continue
            at = torch.arange(t.seq_len, device=keys.device)
            blk = torch.tensor(t.block_ids, device=keys.device)[at // bs]
            k, v = keys[blk, :, at % bs].double(), values[blk, :, at % bs].double()  # [n, kv heads, dim]
            rep = heads // k.shape[1]
            k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
            q = self.q[b, :, 0].double()
            p = torch.softmax(torch.einsum("hd,nhd->hn", q, k) / math.sqrt(dim), dim=1)
            out[b, :, 0] = torch.einsum("hn,nhd->hd", p, v)
            vmax = max(vmax, float(v.abs().max()))
            score = max(score, float(torch.einsum("hd,nhd->hn", q.abs(), k.abs()).max()) / math.sqrt(dim))
        return out, vmax, score

    def check(self, out):
        want, vmax, score = self.exact()
        n, dim, unit = max(t.seq_len for t in self.tables), self.q.shape[3], _UNIT[self.q.dtype]
        extra = 2 * (dim + 4) * 2.0 ** -24 * score + 2.0 ** -16 + (n + 8) * 2.0 ** -24 + n * 2.0 ** -25
        assert out.shape == self.q.shape and out.dtype == self.q.dtype
        err = (out.double() - want).abs()
        assert torch.isfinite(out).all()
        over = err - (vmax * (unit + extra) + unit * want.abs())
        assert float(over.max()) <= 0, f"worst error {float(err.max()):.3e}, over by {float(over.max()):.3e}"
        assert _ops.read_status(out.device) == _lib.OK


def forks(n, prefix, bs, own):
    """n samples of one prompt: full blocks shared, then own(i) positions each."""
    kept = prefix // bs
    return [(0, kept if i else 0, kept * bs + prefix % bs + own(i)) for i in range(n)]


_HEADS = [(14, 2, 64), (32, 8, 128), (16, 16, 64), (16, 1, 128), (24, 2, 64)]


@pytest.mark.parametrize("heads,kv_heads,dim", _HEADS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("prefix,n,bs", [(500, 4, 16), (1024, 40, 16), (129 * 8, 9, 8), (2000, 3, 32), (700, 20, 64),
                                         (1300, 5, 128), (1800, 6, 256)])
def test_forks_on_the_tensor_cores(cuda, dtype, heads, kv_heads, dim, prefix, n, bs):
    case = Case(cuda, dtype, heads, kv_heads, dim, bs, forks(n, prefix, bs, lambda i: 1 + 7 * i % 61), seed=n)
    case.check(paged_shared_prefix_attention(case.q, case.pool, case.layer, case.tables, kernel="tcgen05"))


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,bs", [
    (torch.float32, 14, 2, 64, 16), (torch.float32, 8, 1, 128, 32), (torch.float32, 6, 3, 80, 12),
    (torch.bfloat16, 6, 2, 80, 16), (torch.float16, 14, 2, 64, 12), (torch.bfloat16, 20, 1, 64, 16),
    (torch.float32, 4, 4, 33, 5), (torch.bfloat16, 4, 2, 256, 16), (torch.float32, 64, 1, 128, 16)])
def test_other_types_and_shapes(cuda, dtype, heads, kv_heads, dim, bs):
    case = Case(cuda, dtype, heads, kv_heads, dim, bs, forks(7, 600, bs, lambda i: 1 + 13 * i), seed=dim)
    case.check(paged_shared_prefix_attention(case.q, case.pool, case.layer, case.tables))


_BATCHES = {
    "one sequence": [(0, 0, 300)],
    "one token each": [(0, 0, 1), (0, 0, 1)],
    "nothing shared": [(0, 0, 400), (0, 0, 77), (0, 0, 1000)],
    "an empty sequence": [(0, 0, 640), (0, 0, 0), (0, 40, 641), (0, 40, 700)],
    "no keys of their own": [(0, 0, 640), (0, 40, 640), (0, 40, 640)],
    "a shorter holder": [(0, 0, 640), (0, 20, 320), (0, 40, 660)],
    "nested runs": [(0, 0, 640)] + [(0, 40, 1200)] + [(1, 75, 1201 + i) for i in range(6)] + [(0, 40, 641 + 9 * i)
                                                                                             for i in range(5)],
    "long answers": [(0, 0, 700), (0, 40, 4700), (0, 40, 3333)],
    "many rows": [(0, 0, 520)] + [(0, 32, 513 + i % 50) for i in range(90)],
    "one long run": [(0, 0, 20000)] + [(0, 1249, 19985 + i) for i in range(5)],
}


@pytest.mark.parametrize("n", [2, 3, 5, 9, 17, 33, 70])  # rows of a run: all divisions of a CTA's warps into rows and keys
@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [
    (torch.float32, 2, 2, 64), (torch.float32, 6, 2, 128), (torch.float32, 4, 4, 256), (torch.bfloat16, 3, 1, 100), (torch.float16, 5, 1, 30)])
def test_rows_and_keys_divided_among_warps(cuda, n, dtype, heads, kv_heads, dim):
    case = Case(cuda, dtype, heads, kv_heads, dim, 8, forks(n, 777, 8, lambda i: 1 + 13 * (i % 11)), seed=n)
    case.check(paged_shared_prefix_attention(case.q, case.pool, case.layer, case.tables, kernel="generic"))


@pytest.mark.parametrize("heads", [1, 9, 24, 33, 64])  # of one KV head: one warp's, and more than all warps take at once
def test_many_heads_of_one_kv_head(cuda, heads):
    case = Case(cuda, torch.float32, heads, 1, 64, 16, forks(4, 333, 16, lambda i: 1 + 100 * i), seed=heads)
    case.check(paged_shared_prefix_attention(case.q, case.pool, case.layer, case.tables))


@pytest.mark.parametrize("kernel", ["tcgen05", "generic"])
@pytest.mark.parametrize("name", _BATCHES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(14, 2, 64), (8, 2, 128)])
def test_batches(cuda, name, kernel, heads, kv_heads, dim):
    case = Case(cuda, torch.bfloat16, heads, kv_heads, dim, 16, _BATCHES[name], seed=3)
    case.check(paged_shared_prefix_attention(case.q, case.pool, case.layer, case.tables, kernel=kernel))


@pytest.mark.parametrize("kernel", ["tcgen05", "generic"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [3, 45])
def test_rising_scores_rescale(cuda, kernel, dtype, dim, n):
    """Scores that grow along the sequence by far more than 2^8 in the exponent."""
    case = Case(cuda, dtype, 14, 2, dim, 16, forks(n, 3000, 16, lambda i: 40 + i), seed=1, q_scale=2.0, rising=True)
    case.check(paged_shared_prefix_attention(case.q, case.pool, case.layer, case.tables, kernel=kernel))


def test_strides_streams_and_out(cuda):
    case = Case(cuda, torch.bfloat16, 14, 2, 64, 16, forks(6, 900, 16, lambda i: 1 + i), row_pad=64)
    want = paged_shared_prefix_attention(case.q, case.pool, case.layer, case.tables)
    case.check(want)
    fused = torch.randn(6, 18, 1, 64, device=cuda).to(torch.bfloat16)
    fused[:, :14] = case.q
    plan = SharedPrefixTables(case.pool, case.tables, 14)
    assert torch.equal(paged_shared_prefix_attention(fused[:, :14], case.pool, case.layer, plan), want)
    odd = torch.empty(6, 14, 1, 65, device=cuda, dtype=torch.bfloat16)[..., 1:]  # rows not 16-byte aligned
    odd.copy_(case.q)
    case.check(paged_shared_prefix_attention(odd, case.pool, case.layer, plan))
    out = torch.zeros(6, 20, 1, 64, device=cuda, dtype=torch.bfloat16)
    got = paged_shared_prefix_attention(case.q, case.pool, case.layer, plan, out=out[:, 3:17])
    assert got.data_ptr() == out[:, 3:17].data_ptr() and torch.equal(out[:, 3:17], want)
    assert not out[:, :3].any() and not out[:, 17:].any()
    flat = paged_shared_prefix_attention(case.q[:, :, 0], case.pool, case.layer, plan)
    assert flat.shape == (6, 14, 64) and torch.equal(flat, want[:, :, 0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        assert torch.equal(paged_shared_prefix_attention(case.q, case.pool, case.layer, plan), want)  # prepared call
        with torch.cuda.stream(side):
            assert torch.equal(paged_shared_prefix_attention(case.q, case.pool, case.layer, plan), want)
    got = paged_shared_prefix_attention(case.q, case.pool, case.layer, plan, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    # the prepared call follows a cache whose tensors were replaced, and refuses what it was not prepared for
    other = Case(cuda, torch.bfloat16, 14, 2, 64, 16, forks(6, 900, 16, lambda i: 1 + i), seed=9, row_pad=64)
    case.pool.keys, case.pool.values = other.pool.keys, other.pool.values
    other.tables, other.pool = case.tables, case.pool
    other.q = case.q
    with pytest.raises(ValueError, match="layer_idx"):
        paged_shared_prefix_attention(case.q, case.pool, 2, plan)
    with pytest.raises(ValueError, match="dtypes differ"):
        paged_shared_prefix_attention(case.q.half(), case.pool, case.layer, plan)


def test_captured_in_a_graph_and_repeatable(cuda):
    case = Case(cuda, torch.bfloat16, 14, 2, 64, 16, _BATCHES["long answers"], seed=5)
    plan = SharedPrefixTables(case.pool, case.tables, 14)
    want = paged_shared_prefix_attention(case.q, case.pool, case.layer, plan)
    case.check(want)
    for _ in range(20):  # the last part to arrive joins them in their order
        assert torch.equal(paged_shared_prefix_attention(case.q, case.pool, case.layer, plan), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged_shared_prefix_attention(case.q, case.pool, case.layer, plan)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = paged_shared_prefix_attention(case.q, case.pool, case.layer, plan)
    torch.cuda.current_stream().wait_stream(side)
    case.q.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    case.check(out)


def test_a_graph_has_scratch_of_its_own(cuda):
    case = Case(cuda, torch.bfloat16, 14, 2, 64, 16, _BATCHES["long answers"], seed=6)
    plan = SharedPrefixTables(case.pool, case.tables, 14)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):  # its first use: nothing is there from an eager call
        out = paged_shared_prefix_attention(case.q, case.pool, case.layer, plan)
    other = Case(cuda, torch.bfloat16, 14, 2, 64, 16, _BATCHES["long answers"], seed=7)
    for _ in range(3):
        graph.replay()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            got = paged_shared_prefix_attention(other.q, other.pool, other.layer, other.tables)
    torch.cuda.synchronize()
    case.check(out)
    other.check(got)


def test_values_replaced_between_layers(cuda):
    case = Case(cuda, torch.bfloat16, 14, 2, 64, 16, _BATCHES["long answers"], seed=8)
    plan = SharedPrefixTables(case.pool, case.tables, 14)
    first = paged_shared_prefix_attention(case.q, case.pool, case.layer, plan)
    case.pool.values = case.pool.values * 2  # exact in the type: twice the output
    again = paged_shared_prefix_attention(case.q, case.pool, case.layer, plan)
    assert torch.equal(again, first * 2)


def test_agrees_with_paged_decode_attention(cuda):
    case = Case(cuda, torch.bfloat16, 14, 2, 64, 16, forks(32, 1024, 16, lambda i: 1 + 3 * i))
    got = paged_shared_prefix_attention(case.q, case.pool, case.layer, case.tables)
    want = paged_decode_attention(case.q, case.pool, case.layer, case.tables)
    torch.testing.assert_close(got.float(), want.float(), rtol=1e-2, atol=1e-2)  # the decode attention's own tolerance


@pytest.mark.parametrize("kernel", ["tcgen05", "generic"])
def test_a_block_outside_the_pool_is_recorded(cuda, kernel):
    case = Case(cuda, torch.bfloat16, 14, 2, 64, 16, forks(4, 800, 16, lambda i: 5))
    case.pool.values.nan_to_num_()
    case.pool.keys.nan_to_num_()
    for t in case.tables:  # in the shared run
        t.block_ids[7] = case.pool.keys.shape[1] + 3
    out = paged_shared_prefix_attention(case.q, case.pool, case.layer, case.tables, kernel=kernel)
    assert torch.isfinite(out).all()
    assert _ops.read_status(cuda) == _lib.EBOUNDS
    case = Case(cuda, torch.bfloat16, 14, 2, 64, 16, forks(4, 800, 16, lambda i: 5))
    case.pool.values.nan_to_num_()
    case.pool.keys.nan_to_num_()
    case.tables[2].block_ids[-1] = -7  # in a sequence's own part
    out = paged_shared_prefix_attention(case.q, case.pool, case.layer, case.tables, kernel=kernel)
    assert torch.isfinite(out).all()
    assert _ops.read_status(cuda) == _lib.EBOUNDS


def test_refusals(cuda):
    case = Case(cuda, torch.float32, 14, 2, 64, 16, forks(3, 400, 16, lambda i: 5))
    with pytest.raises(ab.KVLibraryError, match="needs bf16/fp16"):
        paged_shared_prefix_attention(case.q, case.pool, case.layer, case.tables, kernel="tcgen05")
    with pytest.raises(ValueError, match="one block table per sequence"):
        paged_shared_prefix_attention(case.q, case.pool, case.layer, case.tables[:2])
    with pytest.raises(ValueError, match="another cache"):
        paged_shared_prefix_attention(case.q, case.pool, case.layer, SharedPrefixTables(case.pool, case.tables, 28))
    with pytest.raises(ValueError, match="out must have"):
        paged_shared_prefix_attention(case.q, case.pool, case.layer, case.tables, out=torch.empty_like(case.q).half())
    wide = Case(cuda, torch.float32, 65, 1, 8, 16, forks(3, 400, 16, lambda i: 5))
    with pytest.raises(ab.KVLibraryError, match="at most 64 query heads"):
        paged_shared_prefix_attention(wide.q, wide.pool, wide.layer, wide.tables)
    empty = paged_shared_prefix_attention(case.q[:0], case.pool, case.layer, [])
    assert empty.shape == (0, 14, 1, 64)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [(torch.bfloat16, 14, 2, 64), (torch.float16, 32, 8, 128), (torch.float32, 14, 2, 64),
                                                      (torch.float32, 20, 4, 36), (torch.bfloat16, 64, 1, 80)])
@pytest.mark.parametrize("name", _BATCHES)
def test_runs_that_spare_little_are_read_by_each_sequence(cuda, monkeypatch, name, dtype, heads, kv_heads, dim):
    """The plan without runs: every key is a sequence's own, long ones in several parts."""
    monkeypatch.setattr(attention, "_MIN_SAVED_BYTES", 1 << 62)
    case = Case(cuda, dtype, heads, kv_heads, dim, 16, _BATCHES[name], seed=4)
    plan = SharedPrefixTables(case.pool, case.tables, heads)
    assert plan.n_items == 0 and not plan.runs
    case.check(paged_shared_prefix_attention(case.q, case.pool, case.layer, plan))
