"""The serving operators' workloads: several samples decoded from shared prompts.

Three operators run together when many samples are drawn from the same prompts:

* ``shared_attention``: one decode token per sequence attends over its paged cache; the
  sequences of one prompt share that prompt's full blocks, which are read once for all.
* ``rope_axes``: rotary positions with several axes (time, height, width), fused with the
  append of keys and values to the paged cache.
* ``sample``: temperature, top-k, top-p and min-p sampling from one given random number a row.

Each case has a plain form (elementary torch operations in 32 bits, rounded once) and the
framework's own call, chosen by the module's ``own``; ``exact`` evaluates the definition in
64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_AXES = 3  # time, height, width
_THETA = 1_000_000.0
_UNIT = float(2 ** 31)  # sampling weights are whole multiples of 2^-31 of the row's largest


def listed():
    return [
        # four samples of a short chat prompt, a few tokens in: one layer's call is all latency
        _attention("attn_4_samples", "bf16", 14, 2, 64, 16, 1, 4, 500, 500, 24),
        # 256 samples forked from one 1,024-token prompt (the repository's prefix-fork workload)
        _attention("attn_256_forks", "bf16", 14, 2, 64, 16, 1, 256, 1024, 1024, 128),
        # a batch of 24 prompts of unlike, odd lengths with 9 samples each, long answers
        _attention("attn_24_prompts", "fp16", 32, 8, 128, 32, 24, 9, 37, 2345, 700),
        # 64 questions about one long document
        _attention("attn_long_document", "bf16", 32, 8, 128, 16, 1, 64, 98304, 98304, 250),
        # the float32 cache
        _attention("attn_fp32", "fp32", 14, 2, 64, 16, 2, 12, 333, 1000, 60),
        # appending one decode token a sequence
        _rope("rope_decode", "bf16", 14, 2, 64, 16, 48, False),
        # an image and its question, prefilled
        _rope("rope_image_prompt", "bf16", 14, 2, 64, 16, 8191, False),
        # a video clip with wide heads, frequencies dealt to the axes in turn
        _rope("rope_video_prompt", "fp16", 32, 8, 128, 32, 40001, True),
        # the next token of one sequence
        _sample("sample_1_row", "bf16", 1, 151936),
        # a batch with an odd vocabulary
        _sample("sample_33_rows", "fp16", 33, 32003),
        # the 256 forks' next tokens from float32 logits
        _sample("sample_256_rows", "fp32", 256, 151936),
    ]


def _attention(name, dtype, heads, kv_heads, head_dim, block, prompts, samples, prefix_min, prefix_max, answer_max):
    return {"name": name, "op": "shared_attention", "dtype": dtype, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "block": block, "prompts": prompts, "samples": samples,
            "prefix_min": prefix_min, "prefix_max": prefix_max, "answer_max": answer_max}


def _rope(name, dtype, heads, kv_heads, head_dim, block, tokens, interleaved):
    return {"name": name, "op": "rope_axes", "dtype": dtype, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "block": block, "tokens": tokens, "interleaved": interleaved}


def _sample(name, dtype, rows, vocab):
    return {"name": name, "op": "sample", "dtype": dtype, "rows": rows, "vocab": vocab}


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    kind = rng.choice(["shared_attention", "shared_attention", "rope_axes", "sample"])
    if kind == "sample":
        rows, vocab = _log_int(rng, 1, 256), _log_int(rng, 4000, 160000)
        case = _sample("", rng.choice(["bf16", "fp16", "fp32"]), rows, vocab)
    elif kind == "rope_axes":
        heads, kv_heads, head_dim = rng.choice([(14, 2, 64), (32, 8, 128), (16, 16, 64), (8, 1, 128)])
        case = _rope("", rng.choice(["bf16", "fp16", "fp32"]), heads, kv_heads, head_dim, rng.choice([8, 16, 32]),
                     _log_int(rng, 1, 20000), rng.random() < 0.5)
    else:
        heads, kv_heads, head_dim = rng.choice([(14, 2, 64), (32, 8, 128), (16, 16, 64), (8, 1, 128)])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp16", "fp32"])
        block = rng.choice([8, 16, 32, 64])
        prompts, samples = _log_int(rng, 1, 24), _log_int(rng, 2, 200)
        # the scores of one pass, and the pool, stay well below the long document's
        most = 60_000_000 // (prompts * samples * heads) if dtype != "fp32" else 6_000_000 // (prompts * samples * heads)
        most = max(40, min(most, 60_000_000 // (prompts * kv_heads * head_dim)))
        longest = _log_int(rng, 33, most)
        case = _attention("", dtype, heads, kv_heads, head_dim, block, prompts, samples,
                          rng.randint(1, longest), longest, _log_int(rng, 1, min(600, max(2, most))))
    del case["name"]
    return case


def work(case):
    size = _BYTES[case["dtype"]]
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (4 * 5 + 12), "flops": 4.0 * n}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "rope_axes":
        n = case["tokens"]
        moved = 2 * (heads + 2 * kv_heads) * dim * size + (_AXES + 1) * 8
        return {"bytes": n * moved, "flops": 3.0 * n * (heads + kv_heads) * dim}
    prefixes, answers = _lengths(case)
    shared = [p // case["block"] * case["block"] for p in prefixes]
    tokens = sum(shared) + sum(p - s + a for p, s, row in zip(prefixes, shared, answers) for a in row)
    seen = sum(p + a for p, row in zip(prefixes, answers) for a in row)
    rows = case["prompts"] * case["samples"] * heads * dim * size
    return {"bytes": tokens * 2 * kv_heads * dim * size + 2 * rows, "flops": 4.0 * heads * dim * seen}


def prepare(case, seed):
    return {"shared_attention": _prepare_attention, "rope_axes": _prepare_rope,
            "sample": _prepare_sample}[case["op"]](case, seed)


def run(state):
    return state["run_own" if own else "run_plain"](state)


def exact(case, seed):
    return {"shared_attention": _exact_attention, "rope_axes": _exact_rope,
            "sample": _exact_sample}[case["op"]](case, prepare(case, seed))


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


# ---------------------------------------------------------------- decode attention over shared prompts


def _lengths(case):
    """Each prompt's length, and each sample's answer so far (the new token included): the case's own."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    prefixes = [r.randint(case["prefix_min"], case["prefix_max"]) for _ in range(case["prompts"])]
    return prefixes, [[r.randint(1, case["answer_max"]) for _ in range(case["samples"])] for _ in prefixes]


def _prepare_attention(case, seed):
    bs, dtype = case["block"], _DTYPES[case["dtype"]]
    prefixes, answers = _lengths(case)
    shared = [p // bs for p in prefixes]  # whole blocks: a partly filled one is each sample's own copy
    own_tokens = [p % bs + a for p, row in zip(prefixes, answers) for a in row]
    own_blocks = [-(-n // bs) for n in own_tokens]
    total = sum(shared) + sum(own_blocks)
    r = random.Random(seed)
    ids = list(range(total + 3))
    r.shuffle(ids)
    g = _generator(seed)
    shape = (1, total + 3, case["kv_heads"], bs, case["head_dim"])
    keys, values = _randn(g, *shape, dtype=dtype), _randn(g, *shape, dtype=dtype)
    batch = case["prompts"] * case["samples"]
    q = _randn(g, batch, case["heads"], 1, case["head_dim"], dtype=dtype) * 1.5
    at, common, private = 0, [], []
    for n in shared:
        common.append(ids[at:at + n])
        at += n
    for n in own_blocks:
        private.append(ids[at:at + n])
        at += n

    def padded(rows):
        width = max(1, max(len(x) for x in rows))
        return torch.tensor([x + [0] * (width - len(x)) for x in rows], dtype=torch.int64).cuda()

    state = {"run_own": _own_attention, "run_plain": _plain_attention, "q": q, "keys": keys, "values": values,
             "samples": case["samples"], "common": padded(common), "private": padded(private),
             "common_len": torch.tensor([n * bs for n in shared]).cuda(),
             "private_len": torch.tensor(own_tokens).cuda()}
    if own:
        import augur_b200 as ab
        from augur_b200.attention import SharedPrefixTables

        pool = ab.PagedKVCache(keys=keys, values=values, block_size=bs, allocator=ab.BlockAllocator(total + 3))
        tables = [ab.SequenceBlockTable(block_ids=common[b // case["samples"]] + private[b], block_size=bs,
                                        seq_len=shared[b // case["samples"]] * bs + own_tokens[b])
                  for b in range(batch)]
        state["pool"] = pool
        state["tables"] = SharedPrefixTables(pool, tables, n_q_heads=case["heads"])  # once a step, for all layers
    return state


def _own_attention(state):
    from augur_b200.attention import paged_shared_prefix_attention

    return paged_shared_prefix_attention(state["q"], state["pool"], 0, state["tables"])


def _rows_of(pool, blocks):
    """[n, kv heads, width * block, head_dim] in 32 bits: the rows of these blocks, in order."""
    n, width = blocks.shape
    heads, bs, dim = pool.shape[2:]
    return pool[0][blocks].float().permute(0, 2, 1, 3, 4).reshape(n, heads, width * bs, dim)


def _plain_attention(state):
    q, n = state["q"], state["samples"]
    batch, heads, _, dim = q.shape
    kv_heads = state["keys"].shape[2]
    groups, prompts = heads // kv_heads, batch // n
    q = q.float().reshape(prompts, n, kv_heads, groups, dim) / math.sqrt(dim)
    # the prompt's keys against all its samples' queries, each sample's own keys against its own
    ahead = q.transpose(1, 2).reshape(prompts, kv_heads, n * groups, dim) @ _rows_of(
        state["keys"], state["common"]).transpose(2, 3)
    behind = q.reshape(batch, kv_heads, groups, dim) @ _rows_of(state["keys"], state["private"]).transpose(2, 3)
    at = torch.arange(ahead.shape[3], device=q.device)
    ahead = ahead.masked_fill(at >= state["common_len"].view(-1, 1, 1, 1), -math.inf)
    at = torch.arange(behind.shape[3], device=q.device)
    behind = behind.masked_fill(at >= state["private_len"].view(-1, 1, 1, 1), -math.inf)
    behind = behind.reshape(prompts, n, kv_heads, groups, -1).transpose(1, 2).reshape(prompts, kv_heads, n * groups, -1)
    most = torch.maximum(ahead.amax(3, keepdim=True), behind.amax(3, keepdim=True))
    ahead, behind = (ahead - most).exp(), (behind - most).exp()
    total = ahead.sum(3, keepdim=True) + behind.sum(3, keepdim=True)
    out = ahead @ _rows_of(state["values"], state["common"])
    behind = behind.reshape(prompts, kv_heads, n, groups, -1).transpose(1, 2).reshape(batch, kv_heads, groups, -1)
    own_part = behind @ _rows_of(state["values"], state["private"])
    out = out + own_part.reshape(prompts, n, kv_heads, groups, dim).transpose(1, 2).reshape(out.shape)
    out = (out / total).reshape(prompts, kv_heads, n, groups, dim).transpose(1, 2)
    return out.reshape(batch, heads, 1, dim).to(state["q"].dtype)


def _exact_attention(case, state):
    batch, heads, _, dim = state["q"].shape
    kv_heads = case["kv_heads"]
    out = torch.empty(batch, heads, 1, dim, dtype=torch.float64, device="cuda")
    common_len, private_len = state["common_len"].tolist(), state["private_len"].tolist()
    for b in range(batch):
        p = b // case["samples"]
        rows = []
        for pool in (state["keys"], state["values"]):
            own_rows = pool[0][state["private"][b]].transpose(0, 1).reshape(kv_heads, -1, dim)[:, :private_len[b]]
            first = pool[0][state["common"][p]].transpose(0, 1).reshape(kv_heads, -1, dim)[:, :common_len[p]]
            rows.append(torch.cat([first, own_rows], dim=1).double())
        q = state["q"][b, :, 0].double().view(kv_heads, heads // kv_heads, dim)
        s = torch.einsum("hgd,hld->hgl", q, rows[0]) / math.sqrt(dim)
        out[b, :, 0] = torch.einsum("hgl,hld->hgd", torch.softmax(s, dim=-1), rows[1]).reshape(heads, dim)
    return out


# ---------------------------------------------------------------- rotary positions with several axes, cache append


def _axis_of_frequency(case):
    """Which axis turns each of the head_dim / 2 frequencies: a quarter is time's, the rest is halved
    between height and width; in runs, or dealt in turn until height and width have theirs."""
    half = case["head_dim"] // 2
    side = half * 3 // 8
    if not case["interleaved"]:
        return [0] * (half - 2 * side) + [1] * side + [2] * side
    return [j % 3 if j < 3 * side else 0 for j in range(half)]


def _prepare_rope(case, seed):
    n, bs, dim, dtype = case["tokens"], case["block"], case["head_dim"], _DTYPES[case["dtype"]]
    heads, kv_heads = case["heads"], case["kv_heads"]
    g = _generator(seed)
    qkv = _randn(g, n, heads + 2 * kv_heads, dim, dtype=dtype)  # one projection's output
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    at = torch.arange(n, device="cuda")
    if n >= 256:  # a prompt: text, then frames of a grid of patches, then text again
        lead, side = n // 10, 24
        patch = at - lead
        grid = torch.stack([patch // (side * side), patch % (side * side) // side, patch % side]) + lead
        tail = at - (n - lead) + int((n - 2 * lead) // (side * side)) + lead + side
        text = torch.where(at < lead, at, tail)
        positions = torch.where((at >= lead) & (at < n - lead), grid, text)
        blocks = -(-n // bs)
        table = torch.randperm(blocks + 2, generator=g, device="cuda")
        slots = table[at // bs] * bs + at % bs
        total = blocks + 2
    else:  # one token of each of n sequences, each in a block of its own
        positions = torch.randint(0, 30000, (1, n), generator=g, device="cuda").expand(_AXES, n)
        total = n + 2
        slots = torch.randperm(total, generator=g, device="cuda")[:n] * bs
        slots = slots + torch.randint(0, bs, (n,), generator=g, device="cuda")
    pool_shape = (1, total, kv_heads, bs, dim)
    keys, values = torch.zeros(pool_shape, dtype=dtype, device="cuda"), torch.zeros(pool_shape, dtype=dtype, device="cuda")
    inv_freq = torch.tensor([_THETA ** (-2.0 * j / dim) for j in range(dim // 2)], dtype=torch.float32).cuda()
    axis = _axis_of_frequency(case)
    state = {"run_own": _own_rope, "run_plain": _plain_rope, "q": q, "k": k, "v": v, "keys": keys, "values": values,
             "positions": positions.contiguous(), "slots": slots, "inv_freq": inv_freq,
             "axis": torch.tensor(axis).cuda()}
    if own:
        import augur_b200 as ab
        from augur_b200.rope import RopeAxes

        state["pool"] = ab.PagedKVCache(keys=keys, values=values, block_size=bs, allocator=ab.BlockAllocator(total))
        state["axes"] = RopeAxes(axis, inv_freq)
    return state


def _own_rope(state):
    from augur_b200.rope import write_paged_kv_batch_rope_axes

    q = write_paged_kv_batch_rope_axes(state["pool"], state["q"], state["k"], state["v"], state["slots"],
                                       state["positions"], state["axes"], 0)
    return q, state["keys"], state["values"]


def _plain_rope(state):
    keys, values = state["keys"], state["values"]
    half, bs = keys.shape[4] // 2, keys.shape[3]
    angle = state["positions"].float()[state["axis"]].transpose(0, 1) * state["inv_freq"]  # [tokens, frequencies]
    cos, sin = angle.cos().unsqueeze(1), angle.sin().unsqueeze(1)

    def turned(x):
        a, b = x.float()[..., :half], x.float()[..., half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1).to(x.dtype)

    block, row = state["slots"] // bs, state["slots"] % bs
    keys[0][block, :, row] = turned(state["k"])
    values[0][block, :, row] = state["v"]
    return turned(state["q"]), keys, values


def _exact_rope(case, state):
    half, bs = case["head_dim"] // 2, case["block"]
    angle = torch.stack([state["positions"][a].double() * f.double()
                         for a, f in zip(_axis_of_frequency(case), state["inv_freq"])], dim=1)
    turn = torch.polar(torch.ones_like(angle), angle).unsqueeze(1)

    def turned(x):
        z = torch.complex(x[..., :half].double(), x[..., half:].double()) * turn
        return torch.cat([z.real, z.imag], dim=-1)

    keys, values = torch.zeros_like(state["keys"], dtype=torch.float64), torch.zeros_like(state["values"], dtype=torch.float64)
    for pool, rows in ((keys, turned(state["k"])), (values, state["v"].double())):
        flat = torch.zeros(pool.shape[1] * bs, *rows.shape[1:], dtype=torch.float64, device="cuda")
        flat[state["slots"]] = rows
        pool[0] = flat.view(pool.shape[1], bs, *rows.shape[1:]).transpose(1, 2)
    return turned(state["q"]), keys, values


# ---------------------------------------------------------------- sampling


def _prepare_sample(case, seed):
    rows, vocab = case["rows"], case["vocab"]
    g = _generator(seed)
    logits = _randn(g, rows, vocab) * 2.0
    likely = torch.randint(0, vocab, (rows, 24), generator=g, device="cuda")  # what the model leans to
    logits.scatter_add_(1, likely, 4.0 + 8.0 * torch.rand(rows, 24, generator=g, device="cuda"))
    if rows >= 8:
        logits[1, : vocab // 2] = -math.inf  # a grammar's mask
        logits[2] = torch.where(torch.rand(vocab, generator=g, device="cuda") < 0.999, -65504.0, logits[2])
        logits[3] = -math.inf  # and one that leaves nothing
    logits = logits.to(_DTYPES[case["dtype"]])

    def pick(values, dtype):
        at = torch.randint(0, len(values), (rows,), generator=g, device="cuda")
        return torch.tensor(values, dtype=dtype, device="cuda")[at]

    return {"run_own": _own_sample, "run_plain": _plain_sample, "logits": logits,
            "uniform": torch.rand(rows, generator=g, device="cuda"),
            "temperature": pick([0.6, 0.8, 1.0, 1.3, 0.0 if rows > 4 else 0.7], torch.float32),
            "top_k": pick([0, 20, 50, 1000], torch.int32),
            "top_p": pick([1.0, 0.95, 0.9, 0.8], torch.float32),
            "min_p": pick([0.0, 0.0, 0.02, 0.1], torch.float32)}


def _own_sample(state):
    from augur_b200.sampling import sample_tokens

    return sample_tokens(state["logits"], state["uniform"], temperature=state["temperature"], top_k=state["top_k"],
                         top_p=state["top_p"], min_p=state["min_p"])


def _plain_sample(state):
    """Weights are whole numbers, exp((x - max) / temperature) in steps of 2^-31, so every sum is exact
    and the token does not hang on the order of the additions. The draw: the first token, by index,
    at which the kept weights' running sum passes uniform * their total."""
    x = state["logits"].float()
    vocab = x.shape[1]
    most = x.amax(1, keepdim=True)
    temperature = state["temperature"].unsqueeze(1)
    greedy = temperature <= 0
    z = (x - most) * (1.0 / torch.where(greedy, 1.0, temperature))
    z = torch.where(x == most, 0.0, torch.where(greedy, -math.inf, z))
    share = z.exp()
    weight = (share * _UNIT).floor().long()
    top_k = state["top_k"].unsqueeze(1)
    top_k = torch.where(greedy, 1, torch.where((top_k <= 0) | (top_k > vocab), vocab, top_k))
    down, order = z.sort(dim=1, descending=True, stable=True)  # ties: the lowest index first
    rank = torch.arange(vocab, device=x.device)
    sorted_weight = weight.gather(1, order) * (rank < top_k)
    running = sorted_weight.cumsum(1)
    total = running[:, -1:]
    needed = (state["top_p"].double().unsqueeze(1) * total.double()).ceil().long().clamp(min=1)
    kept = (running - sorted_weight < needed) & (rank < top_k) & (down.exp() >= state["min_p"].unsqueeze(1))
    keep = torch.zeros_like(kept).scatter_(1, order, kept)
    running = (weight * keep).cumsum(1)
    total = running[:, -1:]
    target = (state["uniform"].double().unsqueeze(1) * total.double()).floor().long()
    target = torch.minimum(target, total - 1)
    token = (running <= target).sum(1, keepdim=True).clamp(max=vocab - 1)
    logprob = z.gather(1, token) - (total.double() / _UNIT).float().log()
    nothing = most == -math.inf
    token = torch.where(nothing, -1, token)
    logprob = torch.where(nothing, -math.inf, logprob)
    return token.squeeze(1), logprob.squeeze(1)


def _exact_sample(case, state):
    tokens, logprobs = [], []
    for b in range(case["rows"]):
        x = state["logits"][b].double()
        most, t = x.max(), float(state["temperature"][b])
        if most == -math.inf:
            tokens.append(-1)
            logprobs.append(-math.inf)
            continue
        if t <= 0:
            tokens.append(int((x == most).nonzero()[0]))
            logprobs.append(0.0)
            continue
        p = torch.exp((x - most) / t)
        order = torch.argsort(p, descending=True, stable=True)
        k = int(state["top_k"][b])
        order = order[:k] if 0 < k < order.numel() else order
        mass = p[order].cumsum(0)
        order = order[(mass - p[order] < float(state["top_p"][b]) * mass[-1]) & (p[order] >= float(state["min_p"][b]))]
        order = order.sort().values
        mass = p[order].cumsum(0)
        at = min(int((mass <= float(state["uniform"][b]) * mass[-1]).sum()), order.numel() - 1)
        tokens.append(int(order[at]))
        logprobs.append(float(torch.log(p[order[at]] / mass[-1])))
    return torch.tensor(tokens), torch.tensor(logprobs, dtype=torch.float64)
