"""Calls on the 8-bit K/V cache that are at or past their bounds: what is out of them is flagged and left out, what is empty is
no work, what is large is not refused. Values are compared with the 64-bit forms and tolerances of test_gpu_kv8.py."""
import numpy as np
import pytest

from nibble_b200.workloads import make_page_tables
from test_gpu_kv8 import (QMAX, PlainCache, append_both, attend, check_decode, dev, export, ints, np_of, random_pool,
                          rows_of)

pytestmark = pytest.mark.gpu
NAN = float("nan")


def check_rows(got, qf, values, table_row, start, pos0, count, dtype, every=1):
    """Rows start .. start + count of got against attention over the pool's values, within test_gpu_kv8.check_prefill's bounds."""
    k, v = rows_of(values, table_row, pos0 + count)
    weight, last = (0.0, 0.0) if dtype == "float32" else (2.0 ** -11, 2.0 ** -11 if dtype == "float16" else 2.0 ** -8)
    for t in range(0, count, every):
        ro, _, size = attend(qf[start + t], k, v, pos0 + t + 1)
        tol = weight * size + last * np.abs(ro) + 2e-5 * size.max(-1, keepdims=True)
        assert (np.abs(got[start + t] - ro) <= tol).all(), f"row {t}"


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("stride", [40, 200])  # narrow tables: whole works; wide ones: their keys split, the parts joined
def test_prefill_item_longer_than_max_q_len_is_left_out(nbl_ctx, D, dtype, stride):
    import torch
    import nibble_b200 as nb
    H, KV, items = 6, 2, [(3, 290), (0, 150), (100, 420), (1, 0)]  # the third exceeds 300
    table, n_pages = make_page_tables([p + m for p, m in items], shuffle_seed=1, stride=stride)
    kv, values = random_pool(nbl_ctx, "int8", n_pages, KV, D, 2, spread=0.5)
    starts = np.cumsum([0] + [m for _, m in items])[:-1]
    n = sum(m for _, m in items)
    q, qf = np_of(np.random.default_rng(1).standard_normal((n, H, D)).astype(np.float32), getattr(torch, dtype))
    out = torch.full_like(q, NAN)
    nbl_ctx.attn_prefill(kv, q, ints(starts), ints([m for _, m in items]), ints([p for p, _ in items]), dev(table), 300, out)
    with pytest.raises(nb.NibbleError, match="length"):
        nbl_ctx.check()
    got = out.float().cpu().numpy()
    assert np.isnan(got[starts[2]:starts[2] + 420]).all()
    for i in (0, 1):
        check_rows(got, qf, values, table[i], starts[i], *items[i], dtype, every=13)
    kv.close()


def spoil(q, rng, bad):
    """A copy of q with bad in one element of some (row, head)s, and which."""
    import torch
    n, H, D = q.shape
    at = rng.random((n, H)) < 0.3
    at[0, 0] = True
    r, h = np.nonzero(at)
    x = q.clone()
    x[torch.from_numpy(r), torch.from_numpy(h), torch.from_numpy(rng.integers(0, D, len(r)))] = bad
    return x, torch.from_numpy(at).cuda()


@pytest.mark.parametrize("bad", [NAN, float("inf"), float("-inf")])
@pytest.mark.parametrize("kind,D", [("int8", 64), ("e4m3", 128)])
def test_decode_of_queries_that_are_not_finite(nbl_ctx, kind, D, bad):
    """Their heads' outputs and lse are NaN (a row without keys stays 0 and -inf); all others are the same bits as without them."""
    import torch
    lens, H, KV = [1, 40, 0, 900, 9000], 6, 2  # the last one's parts are joined
    table, n_pages = make_page_tables(lens, shuffle_seed=1)
    kv, _ = random_pool(nbl_ctx, kind, n_pages, KV, D, 3)
    rng = np.random.default_rng(7)
    q = dev(rng.standard_normal((5, H, D)).astype(np.float32))
    x, at = spoil(q, rng, bad)
    got = []
    for t in (q, x):
        out, lse = torch.empty_like(q), torch.empty((5, H), device="cuda")
        nbl_ctx.attn_decode(kv, t, dev(table), ints(lens), max(lens), out, lse)
        got.append((out, lse))
    nbl_ctx.check()
    (out, lse), (bad_out, bad_lse) = got
    keys = ints(lens) > 0
    nan = at & keys[:, None]
    assert bad_out[nan].isnan().all() and bad_lse[nan].isnan().all()
    assert torch.equal(bad_out[~nan], out[~nan]) and torch.equal(bad_lse[~nan], lse[~nan])
    assert (bad_out[~keys] == 0).all() and (bad_lse[~keys] == float("-inf")).all()
    kv.close()


@pytest.mark.parametrize("bad", [NAN, float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("kind,D,items,stride", [
    ("int8", 64, [(0, 5), (3001, 4)], None),           # few tokens: the warp-level kernel
    ("e4m3", 128, [(0, 3), (40, 2)], None),
    ("int8", 64, [(0, 300), (70, 150)], 30),           # whole works
    ("e4m3", 64, [(0, 300), (3000, 150)], None),       # joined parts
    ("int8", 128, [(0, 200), (3000, 130)], None),
    ("e4m3", 128, [(0, 200), (100, 130)], 20)])
def test_prefill_of_queries_that_are_not_finite(nbl_ctx, kind, D, items, stride, dtype, bad):
    import torch
    H, KV = 6, 2
    table, n_pages = make_page_tables([p + m for p, m in items], shuffle_seed=1, stride=stride)
    kv, _ = random_pool(nbl_ctx, kind, n_pages, KV, D, 3)
    starts = np.cumsum([0] + [m for _, m in items])[:-1]
    rng = np.random.default_rng(8)
    q = dev(rng.standard_normal((sum(m for _, m in items), H, D)).astype(np.float32)).to(getattr(torch, dtype))
    x, at = spoil(q, rng, bad)
    got = []
    for t in (q, x):
        out = torch.empty_like(q)
        nbl_ctx.attn_prefill(kv, t, ints(starts), ints([m for _, m in items]), ints([p for p, _ in items]), dev(table),
                             max(m for _, m in items), out)
        got.append(out)
    nbl_ctx.check()
    assert not got[0].isnan().any()
    assert got[1][at].isnan().all()
    assert torch.equal(got[1][~at], got[0][~at])
    kv.close()


@pytest.mark.parametrize("how", ["loud_page_not_attended", "spread", "zero_pages"])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("D,H,items,stride", [
    (64, 8, [(0, 300), (70, 150)], 30),     # four heads a block, whole works
    (64, 4, [(0, 300), (3000, 150)], None),  # two, joined parts
    (128, 8, [(0, 200), (100, 130)], 20),
    (128, 4, [(0, 200), (3000, 130)], None)])
def test_prefill_of_uneven_value_scales(nbl_ctx, how, kind, D, H, items, stride):
    """Value scales far apart among a row's pages: errors are measured by what the row attends (sum p |v|), however loud the rest.
    loud_page_not_attended: an item's first page is 2^30 times as loud as the others and has weights near e^-96 of theirs."""
    import torch
    KV = 2
    table, n_pages = make_page_tables([p + m for p, m in items], shuffle_seed=1, stride=stride)
    kv, _ = random_pool(nbl_ctx, kind, n_pages, KV, D, 3)
    codes, scales = export(nbl_ctx, kv)
    rng = np.random.default_rng(11)
    n = sum(m for _, m in items)
    x = rng.standard_normal((n, H, D))
    scales[:, 0] = np.float32(2.0 / QMAX[kind])
    scales[:, 1] = np.float32(2.0 / QMAX[kind])
    if how == "loud_page_not_attended":
        x += 6 * (64 / D) ** 0.5  # a common sign, and keys of the other one in the first page
        for row in table:
            codes[row[0], 0], scales[row[0], 1] = -QMAX[kind], scales[row[0], 1] * np.float32(2.0 ** 30)
    elif how == "spread":
        scales[:, 1] *= np.exp2(rng.integers(-40, 41, (n_pages, KV))).astype(np.float32)
    else:
        for row in table:  # the leading pages, one in the middle
            for page in (row[0], row[1], row[5]):
                codes[page, 1], scales[page, 1] = 0, 0
        scales[:, 1] *= np.float32(1e-20)
    c = dev(codes).to(torch.int8 if kind == "int8" else torch.float8_e4m3fn)
    nbl_ctx.kv_import(kv, ints(np.arange(n_pages)), c, dev(scales))
    values = codes.astype(np.float64) * scales.astype(np.float64)[..., None, None]
    q, qf = np_of(x.astype(np.float32), torch.float16)
    out = torch.full((n, H, D), NAN, device="cuda")
    starts = np.cumsum([0] + [m for _, m in items])[:-1]
    nbl_ctx.attn_prefill(kv, q, ints(starts), ints([m for _, m in items]), ints([p for p, _ in items]), dev(table),
                         max(m for _, m in items), out)
    nbl_ctx.check()
    got = out.double().cpu().numpy()
    for i, (p, m) in enumerate(items):
        k, v = rows_of(values, table[i], p + m)
        for t in range(0, m, 7):
            if how == "loud_page_not_attended" and p + t < 40:
                continue  # rows that see little but the loud page
            ro, _, size = attend(qf[starts[i] + t], k, v, p + t + 1)
            assert (np.abs(got[starts[i] + t] - ro) <= 2.0 ** -11 * size + 2e-5 * size.max(-1, keepdims=True)).all(), f"item {i} row {t}"
    kv.close()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("mean", [1.0, -4.0])
def test_attention_of_queries_of_one_sign(nbl_ctx, kind, D, mean):
    """Queries with a common part (a projection's bias): scores are still good to fp32 accuracy. Decode, and fp32 and 16-bit
    queries of few tokens. |score| stays below 60, whose fp32 error is 2^-24 * 60 = 4e-6, so test_gpu_kv8's 2e-5 holds."""
    import torch
    lens, H, KV = [1, 33, 700, 3000], 8, 2
    table, n_pages = make_page_tables(lens, shuffle_seed=4)
    kv, values = random_pool(nbl_ctx, kind, n_pages, KV, D, 5, spread=0.3)
    rng = np.random.default_rng(6)
    q = (rng.standard_normal((len(lens), H, D)) + mean).astype(np.float32)
    check_decode(nbl_ctx, kv, values, table, lens, H, q)
    for dtype in ("float32", "float16"):
        x, xf = np_of(q, getattr(torch, dtype))
        out = torch.full((len(lens), H, D), NAN, device="cuda")
        nbl_ctx.attn_prefill(kv, x, ints(np.arange(4)), ints([1] * 4), ints(np.array(lens) - 1), dev(table), 1, out)
        nbl_ctx.check()
        got = out.cpu().numpy()
        for r, n in enumerate(lens):
            k, v = rows_of(values, table[r], n)
            ro, _, size = attend(xf[r], k, v, n)
            assert (np.abs(got[r] - ro) <= (0 if dtype == "float32" else 2.0 ** -11) * size + 2e-5 * size.max(-1, keepdims=True)).all()
    kv.close()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("mean", [4.0, -16.0])
def test_decode_scores_of_queries_of_one_sign(nbl_ctx, D, mean):
    """A score is a sum of D products q_d k_d, whose fp32 error is a small multiple of 2^-24 of sum |q_d k_d| / sqrt(D), whatever the
    products' signs; lse, over rows of one length and many keys, carries what the scores have in common. Allowed: 2^-21 of the
    largest such sum (2^-22 for the two fp16 terms of q, as much for the sums)."""
    import torch
    lens, H, KV = [2000, 2000, 1999], 16, 4
    table, n_pages = make_page_tables(lens, shuffle_seed=4)
    kv, values = random_pool(nbl_ctx, "int8", n_pages, KV, D, 5, spread=0.1)
    q = (np.random.default_rng(6).standard_normal((len(lens), H, D)) + mean).astype(np.float32)
    out, lse = torch.empty((len(lens), H, D), device="cuda"), torch.empty((len(lens), H), device="cuda")
    nbl_ctx.attn_decode(kv, dev(q), dev(table), ints(lens), max(lens), out, lse)
    nbl_ctx.check()
    got = lse.double().cpu().numpy()
    for r, n in enumerate(lens):
        k, v = rows_of(values, table[r], n)
        _, want, _ = attend(q[r], k, v, n)
        size = np.einsum("hd,jhd->hj", np.abs(q[r].astype(np.float64)), np.abs(np.repeat(k, H // KV, 1))).max(1) / np.sqrt(D)
        assert (np.abs(got[r] - want) <= 2.0 ** -21 * size).all(), f"row {r}"
    kv.close()


@pytest.mark.parametrize("items", [[(4000, 128)], [(3000, 70), (0, 130), (2900, 100)]])
def test_split_prefill_inside_a_large_buffer(nbl_ctx, items):
    """Few tokens of a long buffer of activations: the scratch goes by the tokens that the call can have."""
    import torch
    import nibble_b200 as nb
    H, KV, D, n = 8, 2, 128, 32768
    table, n_pages = make_page_tables([p + m for p, m in items], shuffle_seed=1)
    ctx = nb.Context(0)  # no scratch yet
    try:
        kv, values = random_pool(ctx, "int8", n_pages, KV, D, 3, spread=0.5)
        starts = [n - 1000 * (i + 1) for i in range(len(items))]
        q, qf = np_of(np.random.default_rng(2).standard_normal((n, H, D)).astype(np.float32), torch.float16)
        out = torch.full((n, H, D), NAN, device="cuda", dtype=torch.float16)
        args = (ints(starts), ints([m for _, m in items]), ints([p for p, _ in items]), dev(table), max(m for _, m in items), out)
        torch.cuda.synchronize()
        before = torch.cuda.mem_get_info()[0]
        ctx.attn_prefill(kv, q, *args)
        ctx.check()
        assert before - torch.cuda.mem_get_info()[0] < 64 << 20
        got = out.float().cpu().numpy()
        written = np.zeros(n, bool)
        for i, (p, m) in enumerate(items):
            check_rows(got, qf, values, table[i], starts[i], p, m, "float16", every=9)
            written[starts[i]:starts[i] + m] = True
        assert np.isnan(got[~written]).all() and not np.isnan(got[written]).any()
        kv.close()
    finally:
        ctx.close()


def test_empty_calls_are_no_work(nbl_ctx):
    """No rows, no items, no pages, empty lists: nothing is refused, nothing changes."""
    import torch
    import nibble_b200 as nb
    lens = [40, 17]
    table, n_pages = make_page_tables(lens, shuffle_seed=1)
    kv, _ = random_pool(nbl_ctx, "int8", n_pages, 2, 64, 3)
    before = export(nbl_ctx, kv)
    book = dev(table), ints(lens), ints(np.ones(n_pages))
    kept = [t.clone() for t in book]
    none, no_rows = ints([]), ints(np.zeros((0, table.shape[1])))

    def empty(heads, dtype=torch.float32):
        return torch.zeros((0, heads, 64), device="cuda", dtype=dtype)

    assert none.data_ptr() == 0
    nbl_ctx.rotary_kv_append(kv, empty(4), empty(2), empty(2), empty(4), none, none, none, no_rows, 0, nb.RotarySpec(1e4, True))
    nbl_ctx.rotary_kv_append(kv, empty(4), empty(2), empty(2), empty(4), none, none, none, no_rows, 7, nb.RotarySpec(1e4, True))
    nbl_ctx.kv_read(kv, none, none, none, no_rows, 7, empty(2), empty(2))
    nbl_ctx.attn_decode(kv, empty(4), no_rows, none, 0, empty(4), torch.zeros((0, 4), device="cuda"))
    for dtype in (torch.float32, torch.half):
        nbl_ctx.attn_prefill(kv, empty(4, dtype), none, none, none, no_rows, 7, empty(4, dtype))
    for call in (nbl_ctx.kv_import, nbl_ctx.kv_export):
        call(kv, none, torch.zeros((0, 2, 2, 16, 64), device="cuda", dtype=torch.int8), torch.zeros((0, 2, 2), device="cuda"))
    nbl_ctx.kv_copy_pages(kv, none, none)
    nbl_ctx.kv_fork(kv, *book, none, none)
    nbl_ctx.kv_extend(kv, *book, none, none)
    nbl_ctx.kv_release(kv, *book, none)
    # items without tokens among the rows
    out = torch.full((3, 4, 64), NAN, device="cuda")
    q, k = torch.ones((3, 4, 64), device="cuda"), torch.ones((3, 2, 64), device="cuda")
    zero, start = ints([0, 0]), ints([0, 3])
    nbl_ctx.rotary_kv_append(kv, q, k, k, out, start, zero, zero, dev(table), 3, nb.RotarySpec(1e4, True))
    nbl_ctx.attn_prefill(kv, q, start, zero, zero, dev(table), 3, out)
    nbl_ctx.kv_read(kv, start, zero, zero, dev(table), 3, out[:, :2].contiguous())
    nbl_ctx.check()
    assert out.isnan().all()
    assert all(torch.equal(a, b) for a, b in zip(book, kept))
    assert all(np.array_equal(a, b) for a, b in zip(export(nbl_ctx, kv), before))
    # a table without rows
    small = nbl_ctx.kv_pool(3, 2, dtype=nb.I8)
    refs, used = ints([5, 5, 5]), ints([9])
    nbl_ctx.kv_compact(kv, small, no_rows, none, no_rows.clone(), refs, used)
    nbl_ctx.check()
    assert refs.tolist() == [0, 0, 0] and used.item() == 0
    kv.close()
    small.close()


@pytest.mark.parametrize("width,items", [(170_000, [(3, 1000), (0, 40), (500, 900)]), (4_000_000, [(70, 1000)])])
def test_prefill_with_a_wide_page_table(nbl_ctx, width, items):
    """A table row's width is no work: fp32 queries whose tiles times the width pass 2^31 are attended in several launches."""
    import torch
    H, KV, D = 32, 8, 64
    narrow, n_pages = make_page_tables([p + m for p, m in items], shuffle_seed=1)
    table = np.full((len(items), width), -1, np.int32)
    table[:, :narrow.shape[1]] = narrow
    kv, values = random_pool(nbl_ctx, "int8", n_pages, KV, D, 3, spread=0.5)
    starts = np.cumsum([0] + [m for _, m in items])[:-1]
    q, qf = np_of(np.random.default_rng(1).standard_normal((sum(m for _, m in items), H, D)).astype(np.float32), torch.float32)
    out = torch.full_like(q, NAN)
    nbl_ctx.attn_prefill(kv, q, ints(starts), ints([m for _, m in items]), ints([p for p, _ in items]), dev(table), 1000, out)
    nbl_ctx.check()
    got = out.cpu().numpy()
    assert not np.isnan(got).any()
    for i, (p, m) in enumerate(items):
        check_rows(got, qf, values, table[i], starts[i], p, m, "float32", every=29)
    kv.close()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("most", [150, 10_000, 2 ** 31 - 1])
def test_prefill_with_a_loose_max_q_len(nbl_ctx, dtype, most):
    """max_q_len only bounds the items: any larger one gives the same."""
    import torch
    items, H, KV, D = [(900, 150), (0, 60)], 4, 2, 64
    table, n_pages = make_page_tables([p + m for p, m in items], shuffle_seed=1)
    kv, values = random_pool(nbl_ctx, "e4m3", n_pages, KV, D, 3, spread=0.5)
    q, qf = np_of(np.random.default_rng(1).standard_normal((210, H, D)).astype(np.float32), getattr(torch, dtype))
    out = torch.full_like(q, NAN)
    nbl_ctx.attn_prefill(kv, q, ints([0, 150]), ints([150, 60]), ints([900, 0]), dev(table), most, out)
    nbl_ctx.check()
    for i, (p, m) in enumerate(items):
        check_rows(out.float().cpu().numpy(), qf, values, table[i], (0, 150)[i], p, m, dtype, every=11)
    kv.close()


def test_decode_is_captured_at_its_first_call_and_outlives_scratch_growth(nbl_ctx):
    """A graph of the decode: nothing is allocated at its first call, and a later call that grows the context's scratch leaves
    what the graph uses where it is."""
    import torch
    import nibble_b200 as nb
    ctx = nb.Context(0)
    try:
        lens, H, KV, D = [9000, 3, 0, 4100], 8, 2, 128
        table, n_pages = make_page_tables(lens, shuffle_seed=1)
        kv, values = random_pool(ctx, "int8", n_pages, KV, D, 3)
        qs = np.random.default_rng(2).standard_normal((3, 4, H, D)).astype(np.float32)
        q, t, n = dev(qs[0]), dev(table), ints(lens)
        out, lse = torch.zeros((4, H, D), device="cuda"), torch.zeros((4, H), device="cuda")
        torch.cuda.synchronize()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=side):
            ctx.set_stream(side.cuda_stream)
            ctx.attn_decode(kv, q, t, n, max(lens), out, lse)
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        x = torch.randn((300, H, D), device="cuda").half()  # few works over many keys: parts in the context's scratch
        free = torch.cuda.mem_get_info()[0]
        ctx.attn_prefill(kv, x, ints([0]), ints([300]), ints([8700]), t, 300, torch.empty_like(x))
        ctx.check()
        assert torch.cuda.mem_get_info()[0] < free
        for k in (1, 2):
            q.copy_(dev(qs[k]))
            graph.replay()
            ctx.check()
            for r, m in enumerate(lens):
                keys, vals = rows_of(values, table[r], m)
                ro, rl, size = attend(qs[k][r], keys, vals, m)
                assert (np.abs(out[r].cpu().numpy() - ro) <= 2e-5 * size.max(-1, keepdims=True)).all()
                got = lse[r].cpu().numpy()
                assert np.isneginf(got).all() if m == 0 else np.abs(got - rl).max() <= 2e-5 * max(1.0, np.abs(rl).max())
        del graph
        kv.close()
    finally:
        ctx.close()


def test_rotary_tables_of_many_parameters_do_not_pile_up(nbl_ctx):
    """A scaling factor that changes with every call: old tables go, and one that is made again gives the same bits."""
    import torch
    import nibble_b200 as nb
    ctx = nb.Context(0)
    try:
        kv = ctx.kv_pool(4, 1, 64, dtype=nb.I8)
        width = 16384  # a table of 262144 positions x 32 pairs x 8 bytes: 64 MB
        table = torch.full((1, width), -1, device="cuda", dtype=torch.int32)
        table[0, :4] = ints([0, 1, 2, 3])
        q, k = torch.randn((40, 2, 64), device="cuda"), torch.randn((40, 1, 64), device="cuda")

        def rotated(factor):
            out = torch.empty_like(q)
            ctx.rotary_kv_append(kv, q, k, k, out, ints([0]), ints([40]), ints([7]), table, 40,
                                 nb.RotarySpec(1e4, True, scaling="linear", factor=factor))
            return out

        first = rotated(1.0)
        ctx.check()
        free = torch.cuda.mem_get_info()[0]
        outs = [rotated(1.0 + i / 8) for i in range(40)]
        ctx.check()
        assert free - torch.cuda.mem_get_info()[0] < 18 * (width * 16 * 32 * 8)
        assert torch.equal(outs[0], first) and torch.equal(rotated(1.0), first) and torch.equal(rotated(5.75), outs[38])
        assert not torch.equal(outs[1], first)
        ctx.check()
        kv.close()
    finally:
        ctx.close()


def test_extend_by_more_pages_than_32_bits_count(nbl_ctx):
    """Rows that want 2^31 pages together: there are not so many, so no row gets any."""
    import torch
    import nibble_b200 as nb
    kv = nbl_ctx.kv_pool(64, 1)
    width, rows = 2 ** 27 - 1, 17
    table = torch.full((rows, width), -1, device="cuda", dtype=torch.int32)  # 9 GB
    lens, refs = ints([0] * rows), ints([0] * 64)
    nbl_ctx.kv_extend(kv, table, lens, refs, ints(range(rows)), ints([width * 16] * rows))
    with pytest.raises(nb.NibbleError, match="no free page"):
        nbl_ctx.check()
    assert lens.tolist() == [0] * rows and refs.tolist() == [0] * 64 and (table[:, :64] == -1).all()
    nbl_ctx.kv_extend(kv, table, lens, refs, ints([3]), ints([33]))
    nbl_ctx.check()
    assert table[3, :4].tolist() == [0, 1, 2, -1] and lens[3].item() == 33
    kv.close()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("offset", [1, 2, 4])
def test_attention_off_alignment(nbl_ctx, dtype, D, offset):
    """q and out that begin off a 16-byte boundary: many query tokens, and the decode."""
    import torch
    items, H, KV = [(700, 100), (0, 33)], 6, 2
    table, n_pages = make_page_tables([p + m for p, m in items], shuffle_seed=1)
    kv, values = random_pool(nbl_ctx, "int8", n_pages, KV, D, 3, spread=0.5)
    dt = getattr(torch, dtype)
    q, qf = np_of(np.random.default_rng(1).standard_normal((133, H, D)).astype(np.float32), dt)

    def moved(t):
        flat = torch.full((t.numel() + offset,), NAN, device="cuda", dtype=t.dtype)
        flat[offset:] = t.reshape(-1)
        return flat[offset:].view(t.shape)

    out = moved(torch.full_like(q, NAN))
    nbl_ctx.attn_prefill(kv, moved(q), ints([0, 100]), ints([100, 33]), ints([700, 0]), dev(table), 100, out)
    nbl_ctx.check()
    for i, (p, m) in enumerate(items):
        check_rows(out.float().cpu().numpy(), qf, values, table[i], (0, 100)[i], p, m, dtype, every=7)
    if dtype == "float32":
        got = moved(torch.full_like(q[:2], NAN))
        nbl_ctx.attn_decode(kv, moved(q[:2]), dev(table), ints([800, 33]), 800, got)
        nbl_ctx.check()
        for r, n in enumerate((800, 33)):
            k, v = rows_of(values, table[r], n)
            ro, _, size = attend(qf[r], k, v, n)
            assert (np.abs(got[r].cpu().numpy() - ro) <= 2e-5 * size.max(-1, keepdims=True)).all()
    kv.close()


@pytest.mark.parametrize("count", [256, 257, 400])
def test_append_and_read_of_many_items(nbl_ctx, count):
    """More items than a warp of every block adds up (and as many): page u is then page u % most of item u / most."""
    import torch
    import nibble_b200 as nb
    rng = np.random.default_rng(count)
    items = [(int(rng.integers(0, 40)), int(rng.integers(0, 35))) for _ in range(count)]
    table, n_pages = make_page_tables([p + m for p, m in items], shuffle_seed=5)
    kv = nbl_ctx.kv_pool(n_pages, 1, dtype=nb.I8)
    plain = PlainCache("int8", n_pages, 1, 64)
    q, want = append_both(nbl_ctx, kv, plain, table, items, 2, nb.RotarySpec(1e4, True), torch.float16, rng)
    nbl_ctx.check()
    codes, scales = export(nbl_ctx, kv)
    assert np.array_equal(scales, plain.scales) and np.array_equal(codes, plain.codes)
    assert (np.abs(q.float().cpu().numpy() - want) <= np.abs(want).max(-1, keepdims=True) * 4 * 2.0 ** -24 + np.abs(want) * 2.0 ** -11 + 2.0 ** -25).all()
    starts = np.cumsum([0] + [m for _, m in items])[:-1]
    n = sum(m for _, m in items)
    k, v = (torch.full((n, 1, 64), NAN, device="cuda") for _ in range(2))
    nbl_ctx.kv_read(kv, ints(starts), ints([m for _, m in items]), ints([p for p, _ in items]), dev(table), 34, k, v)
    nbl_ctx.check()
    values = codes.astype(np.float64) * scales.astype(np.float64)[..., None, None]
    for i, (p, m) in enumerate(items):
        for got, ref in zip((k, v), rows_of(values, table[i], p + m)):
            assert np.array_equal(got[starts[i]:starts[i] + m].cpu().numpy(), ref[p:p + m].astype(np.float32))
    kv.close()
