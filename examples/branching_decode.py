"""Prompts over the 8-bit K/V cache, then several continuations of each, all pages kept by the library.

    python -m examples.branching_decode [int8|e4m3]

One attention layer with random weights stands in for a model. Per prompt: pages (kv_extend), one append with scaled rotary
positions (rotary_kv_append), causal attention (attn_prefill), then `width` branches that share the prompt's pages (kv_fork).
Per step: a page where a branch needs one, the append and the attention of one token of every branch. Half the branches are
then dropped (kv_release), what is left moves together into a smaller pool (kv_compact), and decoding goes on there.
Everything runs on the context's stream without reading anything back; the sizes of the pools are the caller's choice.
"""
import sys

import torch

import nibble_b200 as nb

HEADS, KV_HEADS, HEAD_DIM, VOCAB, PAGE = 8, 2, 64, 128, 16


class Layer:
    """Embedding, Q/K/V projections and an output projection to logits, seeded."""

    def __init__(self, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        width = HEADS * HEAD_DIM
        weight = lambda *shape: torch.randn(shape, device="cuda", generator=g) / shape[0] ** 0.5  # noqa: E731
        self.embed, self.out = torch.randn((VOCAB, width), device="cuda", generator=g), weight(width, VOCAB)
        self.q, self.k, self.v = (weight(width, h * HEAD_DIM) for h in (HEADS, KV_HEADS, KV_HEADS))

    def qkv(self, tokens, dtype=torch.float32):
        x = self.embed[tokens]
        return [(x @ w).to(dtype).reshape(len(tokens), -1, HEAD_DIM) for w in (self.q, self.k, self.v)]


class Cache:
    """A pool, its page tables, row lengths and page reference counts, all on the device."""

    def __init__(self, ctx, kind, n_pages, rows, max_len):
        self.pool = ctx.kv_pool(n_pages, KV_HEADS, HEAD_DIM, dtype=kind)
        self.table = torch.full((rows, -(-max_len // PAGE)), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")

    @property
    def book(self):
        return self.pool, self.table, self.lens, self.refs


def ints(values):
    return torch.tensor(list(values), dtype=torch.int32, device="cuda")


def decode_step(ctx, layer, cache, rows, tokens, rotary, max_len):
    """Appends tokens[i] to row rows[i] of the cache; the attention's output [n, HEADS, HEAD_DIM]."""
    n = len(rows)
    pos = cache.lens[rows.long()]
    ctx.kv_extend(*cache.book, rows, pos + 1)
    table = cache.table[rows.long()]
    q, k, v = layer.qkv(tokens)
    start, one = torch.arange(n, dtype=torch.int32, device="cuda"), torch.ones(n, dtype=torch.int32, device="cuda")
    ctx.rotary_kv_append(cache.pool, q, k, v, q, start, one, pos, table, 1, rotary)
    out = torch.empty_like(q)
    ctx.attn_decode(cache.pool, q, table, pos + 1, max_len, out)
    return out


def run(ctx, kind, prompts=(37, 200, 5), width=4, steps=20, seed=0):
    """The continuations' tokens [branches, steps], the last step's attention outputs, and the cache at the end."""
    layer, n = Layer(seed), len(prompts)
    rotary = nb.RotarySpec(10000.0, True, rotary_dim=48, scaling="yarn", factor=4.0, original_ctx=64)
    rows, max_len = n * width, max(prompts) + steps + 1
    cache = Cache(ctx, kind, sum(-(-p // PAGE) for p in prompts) + rows * (-(-steps // PAGE) + 2), rows, max_len)

    # the prompts: prompt i in row i * width, packed one behind another
    first = ints(range(0, rows, width))
    length, start = ints(prompts), ints(sum(prompts[:i]) for i in range(n))
    zero = torch.zeros(n, dtype=torch.int32, device="cuda")
    tokens = torch.randint(VOCAB, (sum(prompts),), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
    ctx.kv_extend(*cache.book, first, length)
    q, k, v = layer.qkv(tokens, torch.bfloat16)
    table = cache.table[first.long()]
    ctx.rotary_kv_append(cache.pool, q, k, v, q, start, length, zero, table, max(prompts), rotary)
    out = torch.empty_like(q)
    ctx.attn_prefill(cache.pool, q, start, length, zero, table, max(prompts), out)
    logits = out[(start + length - 1).long()].float().reshape(n, -1) @ layer.out

    # the branches: rows i * width + 1.. share row i * width's pages; branch j starts with the j-th likeliest token
    ctx.kv_fork(*cache.book, ints(r - r % width for r in range(rows) if r % width), ints(r for r in range(rows) if r % width))
    next_tokens = logits.topk(width).indices.reshape(-1)
    rows_now, chosen = ints(range(rows)), []
    for step in range(steps):
        if step == steps // 2:  # every other branch is dropped, the rest move together
            ctx.kv_release(*cache.book, rows_now[1::2].contiguous())
            rows_now, next_tokens = rows_now[::2].contiguous(), next_tokens[::2]
            chosen = [c[::2] for c in chosen]
            small = Cache(ctx, kind, cache.pool.n_pages, rows, max_len)
            used = torch.zeros(1, dtype=torch.int32, device="cuda")
            ctx.kv_compact(cache.pool, small.pool, cache.table, cache.lens, small.table, small.refs, used)
            small.lens.copy_(cache.lens)
            ctx.check()  # waits, so that the old pool can go
            cache.pool.close()
            cache = small
        chosen.append(next_tokens)
        out = decode_step(ctx, layer, cache, rows_now, next_tokens, rotary, max_len)
        next_tokens = (out.reshape(len(rows_now), -1) @ layer.out).argmax(-1)
    ctx.check()
    return torch.stack(chosen, 1), out, cache, rows_now


if __name__ == "__main__":
    with_kind = nb.E4M3 if sys.argv[1:] == ["e4m3"] else nb.I8
    context = nb.Context(0)
    context.set_stream(torch.cuda.current_stream().cuda_stream)
    for branch in run(context, with_kind)[0].tolist():
        print(*branch)
