"""Several-axis rotary positions with the cache append, against 64 bits.

The angle is defined in float32 (position times inv_freq, one rounding); from it on, the exact
value is 64-bit. Tolerance, per value and with u the dtype's unit roundoff: u |exact| for the
output (2^-25 below fp16's normal range, where its steps are 2^-24), and (|a| + |b|) 2^-22 for
float32 sin, cos (2 ulp) and the two products.
"""

from __future__ import annotations

import pytest
import torch

import augur_b200 as ab
from augur_b200 import _lib, _ops
from augur_b200.rope import RopeAxes, write_paged_kv_batch_rope, write_paged_kv_batch_rope_axes
from tests.conftest import bits, poison_

pytestmark = pytest.mark.gpu

_UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def exact(x, positions, axes):
    half = x.shape[-1] // 2
    angle = positions.float()[axes.axis.long()].t() * axes.inv_freq  # float32 [tokens, frequencies]
    cos, sin = angle.double().cos().unsqueeze(1), angle.double().sin().unsqueeze(1)
    a, b = x[..., :half].double(), x[..., half:].double()
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def close(got, x, positions, axes):
    want = exact(x, positions, axes)
    half = x.shape[-1] // 2
    size = (x[..., :half].abs().double() + x[..., half:].abs().double()).repeat(1, 1, 2)
    low = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    over = (got.double() - want).abs() - (_UNIT[x.dtype] * want.abs() + size * 2.0 ** -22 + low)
    assert got.dtype == x.dtype and float(over.max()) <= 0, float(over.max())


def make(cuda, dtype, tokens, heads, kv_heads, dim, bs, n_axes=3, seed=0, high=40000):
    g = torch.Generator(device=cuda).manual_seed(seed)
    q, k, v = (torch.randn(tokens, h, dim, generator=g, device=cuda).to(dtype) for h in (heads, kv_heads, kv_heads))
    positions = torch.randint(0, high, (n_axes, tokens), generator=g, device=cuda)
    blocks = -(-tokens // bs) + 3
    slots = torch.randperm(blocks * bs, generator=g, device=cuda)[:tokens]
    shape = (2, blocks, kv_heads, bs, dim)
    pool = ab.PagedKVCache(keys=poison_(torch.empty(shape, dtype=dtype, device=cuda)),
                           values=poison_(torch.empty(shape, dtype=dtype, device=cuda)), block_size=bs,
                           allocator=ab.BlockAllocator(blocks))
    return q, k, v, positions, slots, pool


def check(pool, q, k, v, slots, positions, axes, layer=1):
    before = [bits(t).clone() for t in (pool.keys, pool.values)]
    out = write_paged_kv_batch_rope_axes(pool, q, k, v, slots, positions, axes, layer)
    assert _ops.read_status(q.device) == _lib.OK
    close(out, q, positions, axes)
    bs = pool.block_size
    written = slots >= 0
    blk, row = slots[written] // bs, slots[written] % bs
    if int(written.sum()):
        close(pool.keys[layer][blk, :, row], k[written], positions[:, written], axes)
        assert torch.equal(bits(pool.values[layer][blk, :, row]), bits(v[written]))
    for t, old in zip((pool.keys, pool.values), before):  # and nothing else
        now = bits(t).clone()
        now[layer][blk, :, row] = old[layer][blk, :, row]
        assert torch.equal(now, old)
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,dim,bs", [(14, 2, 64, 16), (32, 8, 128, 32), (5, 5, 80, 12), (3, 1, 10, 5), (2, 1, 256, 16)])
@pytest.mark.parametrize("tokens", [1, 48, 2500])
@pytest.mark.parametrize("layout", ["runs", "dealt"])
def test_rotation_and_append(cuda, dtype, heads, kv_heads, dim, bs, tokens, layout):
    half = dim // 2
    side = half * 3 // 8
    axes = getattr(RopeAxes, layout)((half - 2 * side, side, side), 1e6, cuda)
    q, k, v, positions, slots, pool = make(cuda, dtype, tokens, heads, kv_heads, dim, bs)
    check(pool, q, k, v, slots, positions, axes)


@pytest.mark.parametrize("sections", [(32,), (0, 32), (16, 16), (8, 8, 8, 8), (20, 0, 12)])
def test_axis_counts(cuda, sections):
    q, k, v, positions, slots, pool = make(cuda, torch.float16, 300, 14, 2, 64, 16, n_axes=max(len(sections), 2), high=1 << 24)
    axes = RopeAxes.runs(sections, 1e4, cuda)
    assert axes.axis.tolist() == [a for a, n in enumerate(sections) for _ in range(n)]
    check(pool, q, k, v, slots, positions, axes)


def test_dealt_frequencies():
    assert RopeAxes.dealt((6, 4, 2), 1e4, torch.device("cpu")).axis.tolist() == [0, 1, 2, 0, 1, 2, 0, 1, 0, 0, 1, 0]


def test_one_axis_agrees_with_the_one_position_rotation(cuda):
    q, k, v, positions, slots, pool = make(cuda, torch.bfloat16, 700, 14, 2, 64, 16, n_axes=1)
    out = check(pool, q, k, v, slots, positions, RopeAxes.runs((32,), 1e6, cuda))
    one = write_paged_kv_batch_rope(pool, q, k, v, slots, positions[0], 1e6, 0)
    torch.testing.assert_close(out.float(), one.float(), rtol=3e-2, atol=3e-2)  # which rounds after each of three operations


def test_strides_skips_and_streams(cuda):
    axes = RopeAxes.runs((8, 12, 12), 1e6, cuda)
    q, k, v, positions, slots, pool = make(cuda, torch.bfloat16, 901, 14, 2, 64, 16)
    slots[::7] = -1
    want = check(pool, q, k, v, slots, positions, axes)
    fused = torch.cat([q, k, v], dim=1)
    assert torch.equal(check(pool, fused[:, :14], fused[:, 14:16], fused[:, 16:], slots, positions, axes), want)
    odd = torch.zeros(901, 18, 67, dtype=torch.bfloat16, device=cuda)[..., 1:65]  # rows not 16-byte aligned
    odd.copy_(fused)
    assert torch.equal(check(pool, odd[:, :14], odd[:, 14:16], odd[:, 16:], slots, positions, axes), want)
    apart = torch.zeros(901, 3, 2, dtype=torch.int64, device=cuda)
    apart[:, :, 1] = positions.t()
    two = slots.repeat_interleave(2)
    assert torch.equal(check(pool, q, k, v, two[::2], apart[:, :, 1].t(), axes), want)
    assert torch.equal(check(pool, q, k, v, slots.int(), positions.int(), axes), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = write_paged_kv_batch_rope_axes(pool, q, k, v, slots, positions, axes, 1, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = write_paged_kv_batch_rope_axes(pool, q, k, v, slots, positions, axes, 1)
    torch.cuda.current_stream().wait_stream(side)
    positions.add_(5)
    graph.replay()
    torch.cuda.synchronize()
    close(got, q, positions, axes)


def test_a_slot_or_axis_outside_is_recorded(cuda):
    axes = RopeAxes.runs((8, 12, 12), 1e6, cuda)
    q, k, v, positions, slots, pool = make(cuda, torch.bfloat16, 20, 14, 2, 64, 16)
    slots[3] = pool.keys.shape[1] * 16
    old = bits(pool.keys).clone()
    write_paged_kv_batch_rope_axes(pool, q, k, v, slots, positions, axes, 1)
    assert _ops.read_status(cuda) == _lib.EBOUNDS
    assert int((bits(pool.keys) != old).any(-1).sum()) == 19 * 2
    axes.axis[5] = 9
    write_paged_kv_batch_rope_axes(pool, q, k, v, slots.clamp(max=0), positions, axes, 1)
    assert _ops.read_status(cuda) == _lib.EBOUNDS


def test_refusals(cuda):
    axes = RopeAxes.runs((8, 12, 12), 1e6, cuda)
    q, k, v, positions, slots, pool = make(cuda, torch.bfloat16, 20, 14, 2, 64, 16)
    call = write_paged_kv_batch_rope_axes
    with pytest.raises(ValueError, match="positions must have shape"):
        call(pool, q, k, v, slots, positions[:2], axes, 0)
    with pytest.raises(ValueError, match="slot_mapping"):
        call(pool, q, k, v, slots[:5], positions, axes, 0)
    with pytest.raises(ValueError, match="head_dim / 2 frequencies"):
        call(pool, q, k, v, slots, positions, RopeAxes.runs((8, 8, 8), 1e6, cuda), 0)
    with pytest.raises(ValueError, match="layer range"):
        call(pool, q, k, v, slots, positions, axes, 2)
    with pytest.raises(ValueError, match="one dtype"):
        call(pool, q.half(), k, v, slots, positions, axes, 0)
    with pytest.raises(ValueError, match="does not match cache"):
        call(pool, q[..., :32], k, v, slots, positions, axes, 0)
    with pytest.raises(ValueError, match="no CPU fallback"):
        call(pool, q, k, v, slots, positions, RopeAxes.runs((8, 12, 12), 1e6, torch.device("cpu")), 0)
    with pytest.raises(ValueError, match="axis number"):
        RopeAxes([0, -1], torch.ones(2))
    with pytest.raises(ValueError, match="inv_freq"):
        RopeAxes([0, 1], torch.ones(3))
    assert call(pool, q[:0], k[:0], v[:0], slots[:0], positions[:, :0], axes, 0).shape == (0, 14, 64)
