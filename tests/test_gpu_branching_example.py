"""examples/branching_decode.py: the continuations over the 8-bit cache, against the same layer computed plainly in float64 on
the cache's own contents, and against itself.

Tolerance, derived before the first run: the last step's attention reads codes whose values kv_read gives exactly (code * scale
in float32, one rounding: 2^-24 relative), so what differs is the decode kernel's fp32 arithmetic: 2e-5 of sum p |v|, as for the
decode tests."""
import importlib.util
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "branching_decode.py")
    spec = importlib.util.spec_from_file_location("branching_decode", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("kind", ["I8", "E4M3"])
@pytest.mark.parametrize("prompts,width,steps", [((37, 200, 5), 4, 20), ((16,), 2, 3), ((1, 700), 3, 34)])
def test_branching_decode(nbl_ctx, example, kind, prompts, width, steps):
    import torch
    import nibble_b200 as nb
    tokens, out, cache, rows = example.run(nbl_ctx, getattr(nb, kind), prompts, width, steps)
    branches = -(-len(prompts) * width // 2)
    assert tokens.shape == (branches, steps) and len(rows) == branches
    lens = cache.lens.cpu().numpy()
    kept = rows.cpu().numpy()
    assert (lens[kept] == np.repeat(prompts, width)[kept] + steps).all()
    assert (np.delete(lens, kept) == 0).all()
    # every page that a table names is counted, shared ones as often as they are named
    table = cache.table.cpu().numpy()
    assert (np.bincount(table[table >= 0], minlength=cache.pool.n_pages) == cache.refs.cpu().numpy()).all()

    # the last step again, plainly: the last token's query over what the cache holds
    layer = example.Layer(0)
    H, KV, D = example.HEADS, example.KV_HEADS, example.HEAD_DIM
    n = int(lens[kept].sum())
    k, v = (torch.empty((n, KV, D), device="cuda") for _ in range(2))
    start = np.cumsum(lens[kept]) - lens[kept]
    zero = torch.zeros(len(kept), dtype=torch.int32, device="cuda")
    nbl_ctx.kv_read(cache.pool, example.ints(start), example.ints(lens[kept]), zero, cache.table[rows.long()].contiguous(),
                    int(lens.max()), k_out=k, v_out=v)
    pool = nbl_ctx.kv_pool(len(kept) * (int(lens.max()) // 16 + 1), KV, D, dtype=getattr(nb, kind))  # only for its rotation
    own = torch.arange(pool.n_pages, dtype=torch.int32, device="cuda").reshape(len(kept), -1)
    q, k0, v0 = layer.qkv(tokens[:, -1])
    rotary = nb.RotarySpec(10000.0, True, rotary_dim=48, scaling="yarn", factor=4.0, original_ctx=64)
    nbl_ctx.rotary_kv_append(pool, q, k0, v0, q, example.ints(range(len(kept))), example.ints([1] * len(kept)),
                             example.ints(lens[kept] - 1), own, 1, rotary)
    nbl_ctx.check()
    q, k, v = (t.cpu().numpy().astype(np.float64) for t in (q, k, v))
    for i in range(len(kept)):
        part = slice(start[i], start[i] + lens[kept[i]])
        for h in range(H):
            s = k[part, h // (H // KV)] @ q[i, h] / D ** 0.5
            p = np.exp(s - s.max())
            p /= p.sum()
            want, size = p @ v[part, h // (H // KV)], p @ np.abs(v[part, h // (H // KV)])
            assert np.abs(out[i, h].cpu().numpy() - want).max() <= 2e-5 * size.max()
    pool.close()
    cache.pool.close()


def test_branching_decode_repeats(nbl_ctx, example):
    import nibble_b200 as nb
    runs = [example.run(nbl_ctx, nb.I8, (100, 3), 2, 6) for _ in range(2)]
    assert (runs[0][0] == runs[1][0]).all() and (runs[0][1] == runs[1][1]).all()
    for r in runs:
        r[2].pool.close()
