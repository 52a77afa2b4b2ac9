"""The example that runs several-axis RoPE with the append, shared-prefix attention and sampling
together, and the decode step behind it."""

from __future__ import annotations

import importlib.util
import os

import pytest
import torch

import augur_b200 as ab
from augur_b200 import _lib, _ops, attention
from augur_b200.attention import paged_decode_attention, paged_shared_prefix_attention
from augur_b200.batched import write_paged_kv_batch
from augur_b200.sequences import PagedSequences

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location("parallel_samples", os.path.join(ROOT, "examples", "parallel_samples.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("least", [0, 1 << 62])
def test_example(cuda, monkeypatch, least):
    """With the prompt's blocks read once for all samples, and with each sample reading them."""
    monkeypatch.setattr(attention, "_MIN_SAVED_BYTES", least)
    example = _example()
    args = dict(samples=9, steps=20, text=70, grid=(2, 9, 11), layers=2, vocab=5003)
    tokens, logprobs = example.generate(**args)
    assert tokens.shape == logprobs.shape == (20, 9) and int(tokens.min()) >= 0 and int(tokens.max()) < 5003
    assert (logprobs <= 0).all() and torch.isfinite(logprobs).all()
    assert len({tuple(t) for t in tokens.t().tolist()}) > 1  # the samples differ
    again, same = example.generate(**args)
    assert torch.equal(tokens, again) and torch.equal(logprobs, same)
    greedy, _ = example.generate(**args, temperature=0.0)
    assert (greedy == greedy[:, :1]).all()  # from one prompt, greedily: one answer


def test_shared_prefix_step_grows_and_copies(cuda, monkeypatch):
    """Forks of a prompt that ends inside a block: the first step copies that block for all but one of
    them; attention over the grown tables is the one-sequence kernels'."""
    monkeypatch.setattr(attention, "_MIN_SAVED_BYTES", 0)
    cfg = ab.QwenConfig(num_hidden_layers=1)
    pool = ab.new_paged_kv_cache(cfg, num_blocks=200, block_size=16, device=cuda, dtype=torch.bfloat16)
    seqs = PagedSequences(pool)
    g = torch.Generator(device=cuda).manual_seed(0)

    def kv(n):
        return (torch.randn(1, n, 2, 64, generator=g, device=cuda).to(torch.bfloat16) for _ in range(2))

    adm = seqs.admit(list(range(1000)))
    k, v = kv(1000)
    write_paged_kv_batch(pool, k, v, torch.from_numpy(adm.slots).to(cuda))
    batch = [adm.seq_id, *seqs.fork(adm.seq_id, 6)]
    for step in range(30):
        slots, plan = seqs.shared_prefix_step(batch, 14)
        assert seqs.last_cow_blocks == (6 if step == 0 else 0)
        assert plan.runs == [(list(range(7)), 0, 992)]
        assert [seqs.tables[s].seq_len for s in batch] == [1001 + step] * 7 and slots.unique().numel() == 7
        k, v = kv(7)
        write_paged_kv_batch(pool, k, v, slots)
        q = torch.randn(7, 14, 1, 64, generator=g, device=cuda).to(torch.bfloat16)
        got = paged_shared_prefix_attention(q, pool, 0, plan)
        want = paged_decode_attention(q, pool, 0, [seqs.tables[s] for s in batch])
        torch.testing.assert_close(got.float(), want.float(), rtol=1e-2, atol=1e-2)
    assert _ops.read_status(cuda) == _lib.OK
