"""The 8-bit K/V cache and the page bookkeeping on the GPU, against plain 64-bit (float64) forms written here.

Tolerances, derived before the first run:
  * codes and scales: equal. Quantization is fp32 IEEE steps in a fixed order, restated here in numpy float32; the
    rotation table is float64 cos / sin rounded to float32 on both sides, so an angle's float32 may differ by an ulp
    where the float64 values straddle a rounding boundary (probability < 1e-3 per entry at these positions). Such an ulp
    moves a code only if the value lies within 2^-23 of a boundary: at the sizes here fewer than 1e-3 codes are
    expected to move, and none is allowed.
  * q_out: fp32 within 4 ulp of its row's largest element (the table's ulp; the products are rounded alike); 16-bit types
    one rounding of that.
  * decode and fp32-query attention: max |error| <= 2e-5 of the row's max |value| bound sum p |v|: scores carry an error
    of 2^-22 * sum|q c| (two-term fp16 queries) plus fp32 accumulation, below 1e-5 for |score| up to ~30, and weights
    one of 2^-22.
  * 16-bit queries: weights rounded to fp16, so at most 2^-11 * sum p |v| (each term off by 2^-11 at most), plus one
    rounding of the output type (2^-11 fp16, 2^-8 bf16), plus the fp32 part above.
"""
import math

import numpy as np
import pytest

from nibble_b200.workloads import make_page_tables

pytestmark = pytest.mark.gpu
PAGE = 16
QMAX = {"int8": 127.0, "e4m3": 448.0}


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def ints(v):
    return dev(np.asarray(v, np.int32))


def kind_of(kind):
    import nibble_b200 as nb
    return nb.I8 if kind == "int8" else nb.E4M3


def e4m3(x):
    """Nearest e4m3 value (ties to even) of float32 x, saturating, as float32."""
    import torch
    return torch.from_numpy(np.ascontiguousarray(np.clip(x, -448, 448), dtype=np.float32)).to(torch.float8_e4m3fn).float().numpy()


def export(ctx, kv, n_pages=None):
    """(code values float32 [pages, 2, KV, 16, D], scales [pages, 2, KV]) of the whole pool."""
    import torch
    import nibble_b200 as nb
    n = kv.n_pages if n_pages is None else n_pages
    i8 = kv.dtype == nb.I8
    codes = torch.empty((n, 2, kv.n_kv_heads, PAGE, kv.head_dim), device="cuda", dtype=torch.int8 if i8 else torch.uint8)
    scales = torch.empty((n, 2, kv.n_kv_heads), device="cuda")
    ctx.kv_export(kv, ints(np.arange(n)), codes, scales)
    codes = codes if i8 else codes.view(torch.float8_e4m3fn)
    return codes.float().cpu().numpy(), scales.cpu().numpy()


def random_pool(ctx, kind, n_pages, KV, D, seed, spread=1.0):
    """A pool of random codes and scales (imported), and its values in float64 [pages, 2, KV, 16, D]."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    kv = ctx.kv_pool(n_pages, KV, D, dtype=kind_of(kind))
    x = torch.randn((n_pages, 2, KV, PAGE, D), generator=g, device="cuda") * (QMAX[kind] / 3.5)
    codes = x.round().clamp(-127, 127).to(torch.int8) if kind == "int8" else x.clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = torch.exp(torch.randn((n_pages, 2, KV), generator=g, device="cuda") * spread) * (2.0 / QMAX[kind])
    ctx.kv_import(kv, ints(np.arange(n_pages)), codes, scales)
    return kv, codes.double().cpu().numpy() * scales.double().cpu().numpy()[..., None, None]


def rows_of(values, table_row, n):
    """K and V [n, KV, D] float64 of the first n positions of a page-table row."""
    pages = values[table_row[: -(-n // PAGE)]]  # [p, 2, KV, 16, D]
    x = pages.transpose(1, 0, 3, 2, 4).reshape(2, -1, values.shape[2], values.shape[4])[:, :n]
    return x[0], x[1]


def attend(q, k, v, n_keys):
    """q [H, D] over the first n_keys rows of k, v [n, KV, D] -> out [H, D], lse [H], sum p |v| [H, D]; float64."""
    H, D = q.shape
    if n_keys == 0:
        return np.zeros((H, D)), np.full(H, -np.inf), np.zeros((H, D))
    G = H // k.shape[1]
    kk, vv = np.repeat(k[:n_keys], G, 1), np.repeat(v[:n_keys], G, 1)
    s = np.einsum("hd,jhd->hj", q.astype(np.float64), kk) / math.sqrt(D)
    m = s.max(1, keepdims=True)
    p = np.exp(s - m)
    L = p.sum(1, keepdims=True)
    p /= L
    return np.einsum("hj,jhd->hd", p, vv), (m + np.log(L))[:, 0], np.einsum("hj,jhd->hd", p, np.abs(vv))


# ------------------------------------------------------------------------------------------------ rotary + append
def frequencies(spec, D):
    n = spec.rotary_dim or D
    i = np.arange(n // 2, dtype=np.float64)
    base, mul = float(np.float32(spec.freq_base)), 1.0
    if spec.scaling == "ntk":
        base *= spec.factor ** (n / (n - 2))
    f = base ** (-2 * i / n)
    if spec.scaling == "linear":
        f = f / spec.factor
    elif spec.scaling == "yarn":
        at = lambda b: n * math.log(spec.original_ctx / (b * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(at(spec.beta_fast)), 0), min(math.ceil(at(spec.beta_slow)), n - 1)
        r = np.clip((i - low) / max(high - low, 0.001), 0, 1)
        f = f / spec.factor * r + f * (1 - r)
        mul = 0.1 * math.log(spec.factor) + 1
    elif spec.scaling == "wavelength":
        sm = np.clip((spec.original_ctx * f / (2 * math.pi) - spec.low_freq_factor) / (spec.high_freq_factor - spec.low_freq_factor), 0, 1)
        f = (1 - sm) * f / spec.factor + sm * f
    if spec.attn_factor:
        mul = float(np.float32(spec.attn_factor))
    if spec.freq_factors:
        f = f / np.array(spec.freq_factors, np.float32).astype(np.float64)
    return f, mul


def rotate(x, pos, spec):
    """x [n, heads, D] float32 rotated at pos [n], every product and sum rounded to float32."""
    D = x.shape[-1]
    f, mul = frequencies(spec, D)
    ang = np.asarray(pos, np.float64)[:, None] * f
    c, s = (np.cos(ang) * mul).astype(np.float32)[:, None], (np.sin(ang) * mul).astype(np.float32)[:, None]
    m = f.size
    y = x.astype(np.float32).copy()
    ia, ib = (slice(0, m), slice(m, 2 * m)) if spec.neox else (slice(0, 2 * m, 2), slice(1, 2 * m, 2))
    a, b = x[..., ia], x[..., ib]
    y[..., ia] = a * c - b * s
    y[..., ib] = a * s + b * c
    return y


class PlainCache:
    """Codes and scales of a pool, appended to the plain way."""

    def __init__(self, kind, n_pages, KV, D):
        self.kind = kind
        self.codes = np.zeros((n_pages, 2, KV, PAGE, D), np.float32)
        self.scales = np.zeros((n_pages, 2, KV), np.float32)

    def encode(self, x):
        return np.clip(np.rint(x), -127, 127).astype(np.float32) if self.kind == "int8" else e4m3(x)

    def append(self, table_row, pos0, k, v):
        n = len(k)
        one = np.float32(1)
        for b in range(pos0 // PAGE, -(-(pos0 + n) // PAGE) if n else 0):
            page, lo, hi = table_row[b], max(pos0, b * PAGE), min(pos0 + n, (b + 1) * PAGE)
            if page < 0:
                continue
            s0, s1 = lo - b * PAGE, hi - b * PAGE
            for w, x in enumerate((k, v)):
                new = x[lo - pos0:hi - pos0].transpose(1, 0, 2)  # [KV, tokens, D]
                amax = np.abs(new).max((1, 2)).astype(np.float32)
                want = np.where(amax >= np.float32(1e-30), amax * (np.float32(1) / np.float32(QMAX[self.kind])), 0).astype(np.float32)
                old = self.scales[page, w] if s0 else np.zeros_like(want)
                s = np.maximum(old, want)
                inv = np.divide(one, s, out=np.zeros_like(s), where=s > 0)
                codes = np.zeros_like(self.codes[page, w])
                codes[:, :s0] = self.encode(self.codes[page, w][:, :s0] * (old * inv)[:, None, None])
                codes[:, s0:s1] = self.encode(new * inv[:, None, None])
                self.codes[page, w], self.scales[page, w] = codes, s


def np_of(x, dtype):
    """x float32 -> (device tensor of dtype, the float32 values it holds)."""
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda().to(dtype)
    return t, t.float().cpu().numpy()


def append_both(ctx, kv, plain, table, items, H, spec, dtype, rng, bias=False, offset=0, out_dtype=None):
    """Appends random tokens to the pool and to the plain cache; returns (q_out, expected q). items: (pos0, len)."""
    import torch
    KV, D = kv.n_kv_heads, kv.head_dim
    n = sum(m for _, m in items)
    arrs = [rng.standard_normal((n, h, D)).astype(np.float32) * sc for h, sc in ((H, 1), (KV, 3), (KV, 0.7))]
    tens = []
    for i, a in enumerate(arrs):
        t, arrs[i] = np_of(a, dtype)
        flat = torch.zeros(t.numel() + offset, device="cuda", dtype=dtype)  # rows that start off a 16-byte boundary
        flat[offset:] = t.reshape(-1)
        tens.append(flat[offset:].view(t.shape))
    bs = [rng.standard_normal(h * D).astype(np.float32) if bias else None for h in (H, KV, KV)]
    q_out = torch.full((n, H, D), float("nan"), device="cuda", dtype=out_dtype or dtype)
    starts = np.cumsum([0] + [m for _, m in items])[:-1]
    ctx.rotary_kv_append(kv, *tens, q_out, ints(starts), ints([m for _, m in items]), ints([p for p, _ in items]), dev(table),
                         max(m for _, m in items), spec, **{f"b{x}": None if b is None else dev(b) for x, b in zip("qkv", bs)})
    biased = [a if b is None else a + b.reshape(1, -1, D) for a, b in zip(arrs, bs)]
    want_q = np.empty_like(arrs[0])
    for i, (p, m) in enumerate(items):
        part = slice(starts[i], starts[i] + m)
        pos = np.arange(p, p + m)
        want_q[part] = rotate(biased[0][part], pos, spec)
        plain.append(table[i], p, rotate(biased[1][part], pos, spec), biased[2][part])
    return q_out, want_q


def specs():
    import nibble_b200 as nb
    return {
        "adjacent": nb.RotarySpec(1e4, False),
        "half_apart": nb.RotarySpec(1e6, True),
        "part_half_apart": nb.RotarySpec(1e4, True, rotary_dim=32),
        "part_adjacent_2": nb.RotarySpec(1e4, False, rotary_dim=2),
        "linear": nb.RotarySpec(1e4, False, scaling="linear", factor=4.0),
        "ntk_part": nb.RotarySpec(1e4, True, rotary_dim=48, scaling="ntk", factor=2.0),
        "yarn": nb.RotarySpec(1e6, True, scaling="yarn", factor=4.0, original_ctx=32768),
        "yarn_attn": nb.RotarySpec(1e4, False, rotary_dim=16, scaling="yarn", factor=8.0, original_ctx=64, attn_factor=1.25),
        "wavelength": nb.RotarySpec(5e5, False, scaling="wavelength", factor=8.0, original_ctx=8192),
        "factors": nb.RotarySpec(5e5, False, rotary_dim=8, freq_factors=(1.0, 2.0, 3.0, 8.0)),
    }


@pytest.mark.parametrize("name", ["adjacent", "half_apart", "part_half_apart", "part_adjacent_2", "linear", "ntk_part", "yarn",
                                  "yarn_attn", "wavelength", "factors"])
@pytest.mark.parametrize("kind,D,dtype", [("int8", 64, "float32"), ("e4m3", 128, "bfloat16")])
def test_append_rotary_forms(nbl_ctx, name, kind, D, dtype):
    import torch
    rng = np.random.default_rng(sum(map(ord, name)))
    items = [(0, 37), (5, 1), (16, 16), (31, 2), (999, 18)]
    table, n_pages = make_page_tables([p + m for p, m in items], shuffle_seed=3)
    kv = nbl_ctx.kv_pool(n_pages, 2, D, dtype=kind_of(kind))
    plain = PlainCache(kind, n_pages, 2, D)
    dt = getattr(torch, dtype)
    q, want = append_both(nbl_ctx, kv, plain, table, items, 6, specs()[name], dt, rng)
    nbl_ctx.check()
    codes, scales = export(nbl_ctx, kv)
    assert np.array_equal(scales, plain.scales)
    assert np.array_equal(codes, plain.codes)
    got = q.float().cpu().numpy()
    top = np.abs(want).max(-1, keepdims=True)
    tol = top * 4 * 2.0 ** -24 + (0 if dtype == "float32" else np.abs(want) * 2.0 ** -8)
    assert (np.abs(got - want) <= tol).all()
    kv.close()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("D,KV,H", [(64, 1, 1), (64, 8, 32), (128, 2, 14), (128, 4, 4)])
def test_append_fills_pages_in_steps(nbl_ctx, kind, D, KV, H):
    """Prompts, then single tokens and short runs into part-filled pages: the scale grows and old codes are rounded again."""
    import torch
    rng = np.random.default_rng(D + KV)
    lens = [0, 15, 16, 33]
    table, n_pages = make_page_tables([x + 40 for x in lens], shuffle_seed=9)
    kv = nbl_ctx.kv_pool(n_pages, KV, D, dtype=kind_of(kind))
    plain = PlainCache(kind, n_pages, KV, D)
    spec = specs()["half_apart"]
    append_both(nbl_ctx, kv, plain, table, [(0, x) for x in lens], H, spec, torch.float16, rng, bias=True)
    at = list(lens)
    for step in ([1, 1, 1, 1], [1, 0, 1, 1], [7, 1, 3, 2], [0, 2, 0, 17], [1, 1, 1, 1]):
        append_both(nbl_ctx, kv, plain, table, list(zip(at, step)), H, spec, torch.float16, rng, bias=True)
        at = [a + s for a, s in zip(at, step)]
    nbl_ctx.check()
    codes, scales = export(nbl_ctx, kv)
    assert np.array_equal(scales, plain.scales)
    assert np.array_equal(codes, plain.codes)
    kv.close()


@pytest.mark.parametrize("offset", [1, 2, 3, 4])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_append_off_alignment_and_in_place(nbl_ctx, offset, dtype):
    import torch
    rng = np.random.default_rng(offset)
    items = [(3, 30), (0, 5)]
    table, n_pages = make_page_tables([33, 5], shuffle_seed=1)
    kv = nbl_ctx.kv_pool(n_pages, 2, dtype=kind_of("int8"))
    plain = PlainCache("int8", n_pages, 2, 64)
    q, want = append_both(nbl_ctx, kv, plain, table, items, 4, specs()["adjacent"], getattr(torch, dtype), rng, offset=offset,
                          out_dtype=torch.float32)
    nbl_ctx.check()
    codes, scales = export(nbl_ctx, kv)
    assert np.array_equal(scales, plain.scales) and np.array_equal(codes, plain.codes)
    assert (np.abs(q.cpu().numpy() - want) <= np.abs(want).max(-1, keepdims=True) * 4 * 2.0 ** -24).all()
    # q_out may be q_in
    x = torch.randn((5, 4, 64), device="cuda")
    y = torch.empty_like(x)
    k = torch.randn((5, 2, 64), device="cuda")
    args = (ints([0]), ints([5]), ints([0]), dev(table[1:]), 5, specs()["adjacent"])
    nbl_ctx.rotary_kv_append(kv, x, k, k, y, *args)
    nbl_ctx.rotary_kv_append(kv, x, k, k, x, *args)
    assert torch.equal(x, y)
    kv.close()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_append_zeros_tiny_huge_and_non_finite(nbl_ctx, kind):
    import torch
    import nibble_b200 as nb
    kv = nbl_ctx.kv_pool(4, 1, dtype=kind_of(kind))
    table = ints([[0], [1], [2], [3]])
    k = torch.zeros((4, 1, 64), device="cuda")
    k[1] = 1e-38  # below the smallest scale: stored as zeros
    k[2] = 2e38
    k[3, 0, 5], k[3, 0, 6], k[3, 0, 7] = float("nan"), float("inf"), 1.0
    v = torch.ones((4, 1, 64), device="cuda")
    q = torch.ones((4, 1, 64), device="cuda")
    spec = nb.RotarySpec(1e4, True)
    one = ints([1, 1, 1])
    nbl_ctx.rotary_kv_append(kv, q[:3], k[:3], v[:3], q[:3].clone(), ints([0, 1, 2]), one, ints([0, 0, 0]), table, 1, spec)
    nbl_ctx.check()
    out = torch.empty((4, 1, 64), device="cuda")
    nbl_ctx.kv_read(kv, ints([0, 1, 2]), one, ints([0, 0, 0]), table, 1, k_out=out[:3])
    got = out[:3].cpu().numpy()
    assert (got[:2] == 0).all() and np.allclose(got[2], 2e38, rtol=0.07)
    nbl_ctx.rotary_kv_append(kv, q[3:], k[3:], v[3:], q[3:].clone(), ints([0]), ints([1]), ints([0]), table[3:], 1, spec)
    with pytest.raises(nb.NibbleError, match="infinity or NaN"):
        nbl_ctx.check()
    _, scales = export(nbl_ctx, kv)
    assert np.isfinite(scales).all()
    nbl_ctx.kv_read(kv, ints([3]), ints([1]), ints([0]), table, 1, k_out=out)  # row 0's table entry is page 0: other data
    assert torch.isfinite(out[3]).all()
    kv.close()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("out", ["float32", "float16", "bfloat16"])
def test_read_export_import(nbl_ctx, kind, D, out):
    import torch
    KV, lens = 3, [1, 16, 50, 7]
    table, n_pages = make_page_tables(lens, shuffle_seed=4)
    kv, values = random_pool(nbl_ctx, kind, n_pages, KV, D, 5)
    pos0 = [0, 3, 11, 2]
    count = [1, 13, 39, 0]
    starts = np.cumsum([0] + count)[:-1]
    dt = getattr(torch, out)
    k, v = (torch.full((sum(count), KV, D), float("nan"), device="cuda", dtype=dt) for _ in range(2))
    nbl_ctx.kv_read(kv, ints(starts), ints(count), ints(pos0), dev(table), max(count), k, v)
    nbl_ctx.check()
    for i in range(4):
        rk, rv = rows_of(values, table[i], lens[i])
        for got, ref in ((k, rk), (v, rv)):
            g = got[starts[i]:starts[i] + count[i]].float().cpu().numpy()
            r = torch.from_numpy(ref[pos0[i]:pos0[i] + count[i]].astype(np.float32)).to(dt).float().numpy()
            assert np.array_equal(g, r)
    codes, scales = export(nbl_ctx, kv)
    assert np.array_equal(codes.astype(np.float64) * scales[..., None, None], values)
    kv.close()


# ------------------------------------------------------------------------------------------------ attention
def check_decode(nbl_ctx, kv, values, table, lens, H, q, n_splits=0, q_scale=1.0, max_len=None, tol=2e-5):
    import torch
    D = kv.head_dim
    out = torch.full((len(lens), H, D), float("nan"), device="cuda")
    lse = torch.full((len(lens), H), float("nan"), device="cuda")
    nbl_ctx.attn_decode(kv, dev(q), dev(table), ints(lens), max(lens) if max_len is None else max_len, out, lse, n_splits)
    nbl_ctx.check()
    o, l = out.cpu().numpy(), lse.cpu().numpy()
    for r, n in enumerate(lens):
        k, v = rows_of(values, table[r], n)
        ro, rl, size = attend(q[r], k, v, n)
        assert (np.abs(o[r] - ro) <= tol * size.max(-1, keepdims=True)).all(), f"row {r}"
        if n:
            assert np.abs(l[r] - rl).max() <= tol * max(1.0, np.abs(rl).max()), f"row {r} lse"
        else:
            assert (o[r] == 0).all() and np.isneginf(l[r]).all()


DECODE_LENS = [1, 15, 16, 0, 17, 31, 32, 33, 100, 257, 1000, 2049]


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,KV", [(14, 2), (32, 8), (8, 8), (7, 1), (20, 2), (33, 1)])
@pytest.mark.parametrize("n_splits", [0, 1, 3])
def test_decode(nbl_ctx, kind, D, H, KV, n_splits):
    table, n_pages = make_page_tables(DECODE_LENS, shuffle_seed=H + D)
    kv, values = random_pool(nbl_ctx, kind, n_pages, KV, D, H)
    q = np.random.default_rng(H * D).standard_normal((len(DECODE_LENS), H, D)).astype(np.float32)
    check_decode(nbl_ctx, kv, values, table, DECODE_LENS, H, q, n_splits)
    kv.close()


@pytest.mark.parametrize("kind,D,KV,H", [("int8", 64, 8, 32), ("e4m3", 128, 1, 4)])
def test_decode_long_rows_split(nbl_ctx, kind, D, KV, H):
    lens = [20011, 65536]
    table, n_pages = make_page_tables(lens, shuffle_seed=2)
    kv, values = random_pool(nbl_ctx, kind, n_pages, KV, D, 1)
    q = np.random.default_rng(5).standard_normal((2, H, D)).astype(np.float32)
    check_decode(nbl_ctx, kv, values, table, lens, H, q)
    check_decode(nbl_ctx, kv, values, table, lens, H, q, n_splits=37)
    kv.close()


@pytest.mark.parametrize("mag", [1e-12, 1e-3, 1e3, 1e20])
def test_decode_magnitudes(nbl_ctx, mag):
    """Queries and value scales far from 1 (key scales the other way, so scores stay ordinary)."""
    import torch
    lens, KV, H, D = [100, 33], 2, 8, 64
    table, n_pages = make_page_tables(lens, shuffle_seed=2)
    kv, values = random_pool(nbl_ctx, "int8", n_pages, KV, D, 1)
    codes, scales = export(nbl_ctx, kv)
    scales[:, 0] /= np.float32(mag)
    scales[:, 1] *= np.float32(mag)
    nbl_ctx.kv_import(kv, ints(np.arange(n_pages)), dev(codes.astype(np.int8)), dev(scales))
    values = codes.astype(np.float64) * scales.astype(np.float64)[..., None, None]
    q = (np.random.default_rng(5).standard_normal((2, H, D)) * mag).astype(np.float32)
    check_decode(nbl_ctx, kv, values, table, lens, H, q)
    kv.close()


def test_decode_sharp_and_uneven_scales(nbl_ctx):
    """Large scores (one key takes nearly all the weight) and value scales that differ by 1e6 between pages."""
    lens, KV, H, D = [500, 47], 2, 8, 128
    table, n_pages = make_page_tables(lens, shuffle_seed=2)
    kv, values = random_pool(nbl_ctx, "int8", n_pages, KV, D, 1, spread=3.0)
    q = np.random.default_rng(5).standard_normal((2, H, D)).astype(np.float32) * 2
    # scores reach a few hundred: their fp32 error is 2^-22 of that, so weights are good to about 1e-4
    check_decode(nbl_ctx, kv, values, table, lens, H, q, tol=5e-4)
    kv.close()


def test_places_past_the_end_do_not_count(nbl_ctx):
    """What stands in a page past a row's length is another sequence's, or old: same results whatever it is."""
    import torch
    lens, KV, H, D = [21, 5], 1, 4, 64
    table, n_pages = make_page_tables(lens, shuffle_seed=2)
    kv, values = random_pool(nbl_ctx, "e4m3", n_pages, KV, D, 1)
    codes, scales = export(nbl_ctx, kv)
    q = dev(np.random.default_rng(5).standard_normal((2, H, D)).astype(np.float32))
    got = []
    for fill in (0.0, 448.0, -448.0):
        c = codes.copy()
        for r, n in enumerate(lens):
            c[table[r, (n - 1) // PAGE], :, :, (n - 1) % PAGE + 1:] = fill
        nbl_ctx.kv_import(kv, ints(np.arange(n_pages)), dev(c).to(torch.float8_e4m3fn), dev(scales))
        out = torch.empty((2, H, D), device="cuda")
        nbl_ctx.attn_decode(kv, q, dev(table), ints(lens), 21, out)
        got.append(out)
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    kv.close()


PREFILL_ITEMS = [(0, 1), (0, 130), (40, 3), (15, 17), (16, 0), (300, 33), (1, 257), (700, 8)]  # (pos0, len)


def check_prefill(nbl_ctx, kv, values, table, items, H, dtype, seed, out_dtype=None, stride=1):
    import torch
    D = kv.head_dim
    dt = getattr(torch, dtype)
    n = sum(m for _, m in items)
    q, qf = np_of(np.random.default_rng(seed).standard_normal((n, H, D)).astype(np.float32), dt)
    odt = getattr(torch, out_dtype or dtype)
    out = torch.full((n, H, D), float("nan"), device="cuda", dtype=odt)
    starts = np.cumsum([0] + [m for _, m in items])[:-1]
    nbl_ctx.attn_prefill(kv, q, ints(starts), ints([m for _, m in items]), ints([p for p, _ in items]), dev(table),
                         max(m for _, m in items), out)
    nbl_ctx.check()
    got = out.float().cpu().numpy()
    last = {"float32": 0.0, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}[str(odt).replace("torch.", "")]
    weight = 0.0 if dtype == "float32" else 2.0 ** -11
    for i, (p, m) in enumerate(items):
        k, v = rows_of(values, table[i], p + m)
        for t in range(0, m, stride):
            ro, _, size = attend(qf[starts[i] + t], k, v, p + t + 1)
            tol = weight * size + last * np.abs(ro) + 2e-5 * size.max(-1, keepdims=True)
            assert (np.abs(got[starts[i] + t] - ro) <= tol).all(), f"item {i} row {t}"


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,KV", [(14, 2), (8, 8), (9, 1), (32, 4)])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
def test_prefill(nbl_ctx, kind, D, H, KV, dtype):
    table, n_pages = make_page_tables([p + m for p, m in PREFILL_ITEMS], shuffle_seed=H + D)
    kv, values = random_pool(nbl_ctx, kind, n_pages, KV, D, H, spread=0.5)
    check_prefill(nbl_ctx, kv, values, table, PREFILL_ITEMS, H, dtype, H, stride=5)
    kv.close()


@pytest.mark.parametrize("dtype,out_dtype", [("bfloat16", "float32"), ("float16", "float32"), ("bfloat16", None)])
@pytest.mark.parametrize("D", [64, 128])
def test_prefill_few_and_long(nbl_ctx, dtype, out_dtype, D):
    """A few drafted tokens over a long cache (split), and a prompt of several query tiles over one."""
    for items in ([(5001, 4), (4000, 2)], [(3001, 300)]):
        table, n_pages = make_page_tables([p + m for p, m in items], shuffle_seed=1)
        kv, values = random_pool(nbl_ctx, "int8", n_pages, 2, D, 3, spread=0.5)
        check_prefill(nbl_ctx, kv, values, table, items, 6, dtype, 4, out_dtype, stride=7 if items[0][1] > 9 else 1)
        kv.close()


@pytest.mark.parametrize("H,KV", [(4, 2), (5, 1), (12, 2), (3, 1)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("items", [[(2500, 40), (0, 130), (3000, 257), (10, 1), (5, 0), (0, 400)], [(9001, 300)],
                                   [(2000, 290), (0, 0), (2300, 150)], [(0, 2600)]])
def test_prefill_few_ragged_items(nbl_ctx, H, KV, D, items):
    """Fewer query tiles than SMs, of unlike lengths, groups that do not fill a CTA's heads: tiles dealt over the CTAs."""
    table, n_pages = make_page_tables([p + m for p, m in items], shuffle_seed=H)
    kv, values = random_pool(nbl_ctx, "e4m3", n_pages, KV, D, H, spread=0.5)
    check_prefill(nbl_ctx, kv, values, table, items, H, "float16", H, stride=37)
    kv.close()


@pytest.mark.parametrize("H,KV,D", [(10, 2, 64), (6, 2, 128), (2, 2, 64)])
def test_prefill_many_short_items(nbl_ctx, H, KV, D):
    """More works than CTAs, most of one to three tiles."""
    items = [(7 * i % 90, 65 + 17 * i % 130) for i in range(150)]
    table, n_pages = make_page_tables([p + m for p, m in items], shuffle_seed=H)
    kv, values = random_pool(nbl_ctx, "int8", n_pages, KV, D, H, spread=0.5)
    check_prefill(nbl_ctx, kv, values, table, items, H, "bfloat16", H, stride=61)
    kv.close()


def test_attention_on_another_stream(nbl_ctx):
    import torch
    import nibble_b200 as nb
    side = torch.cuda.Stream()
    ctx = nb.Context(0)
    ctx.set_stream(side.cuda_stream)
    try:
        lens = [300, 40]
        table, n_pages = make_page_tables(lens, shuffle_seed=1)
        with torch.cuda.stream(side):
            kv, values = random_pool(ctx, "int8", n_pages, 2, 64, 3)
            q = np.random.default_rng(0).standard_normal((2, 4, 64)).astype(np.float32)
            check_decode(ctx, kv, values, table, lens, 4, q)
            kv.close()
    finally:
        ctx.close()


def test_repeated_calls_give_the_same_bits(nbl_ctx):
    import torch
    lens, H, D = [4000, 1], 8, 64
    table, n_pages = make_page_tables(lens, shuffle_seed=1)
    kv, _ = random_pool(nbl_ctx, "int8", n_pages, 2, D, 3)
    q = dev(np.random.default_rng(0).standard_normal((2, H, D)).astype(np.float32))
    outs = [torch.empty((2, H, D), device="cuda") for _ in range(5)]
    for o in outs:
        nbl_ctx.attn_decode(kv, q, dev(table), ints(lens), 4000, o)
    assert all(torch.equal(outs[0], o) for o in outs)
    kv.close()


def test_append_items_out_of_bounds_are_flagged(nbl_ctx):
    """Items longer than max_len, past the rows or the table, and so many that share rows that their pages exceed the launch."""
    import torch
    import nibble_b200 as nb
    kv = nbl_ctx.kv_pool(64, 1, dtype=nb.I8)
    x = torch.ones((160, 1, 64), device="cuda")
    spec = nb.RotarySpec(1e4, True)
    table = ints(np.arange(60).reshape(3, 20))
    for start, length, pos0, most in [([0, 0, 0], [160, 160, 160], [0, 0, 0], 160), ([0, 0, 0], [1, 30, 1], [0, 0, 0], 20),
                                      ([0, 150, 0], [1, 20, 1], [0, 0, 0], 20), ([0, 0, 0], [1, 20, 1], [0, 310, 0], 20),
                                      ([0, -1, 0], [1, 20, 1], [0, 0, 0], 20), ([0, 0, 0], [1, 20, 1], [0, -1, 0], 20)]:
        nbl_ctx.rotary_kv_append(kv, x, x, x, x.clone(), ints(start), ints(length), ints(pos0), table, most, spec)
        with pytest.raises(nb.NibbleError):
            nbl_ctx.check()
    kv.close()


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals(nbl_ctx):
    import torch
    import nibble_b200 as nb
    INV, UNSUP = 1, 4

    def refused(status, f, *a, **k):
        with pytest.raises(nb.NibbleError) as e:
            f(*a, **k)
        assert e.value.status == status, str(e.value)

    refused(UNSUP, nbl_ctx.kv_pool, 4, 1, 96, dtype=nb.I8)
    refused(UNSUP, nbl_ctx.kv_pool, 4, 1, 64, 32, dtype=nb.E4M3)
    refused(UNSUP, nbl_ctx.kv_pool, 4, 1, 128)
    refused(INV, nbl_ctx.kv_pool, 0, 1, dtype=nb.I8)
    kv, f16 = nbl_ctx.kv_pool(4, 2, dtype=nb.I8), nbl_ctx.kv_pool(4, 2)
    with pytest.raises(ValueError):
        kv.tensor()
    table, one, zero = ints([[0, 1]]), ints([1]), ints([0])
    q, k = torch.zeros((1, 4, 64), device="cuda"), torch.zeros((1, 2, 64), device="cuda")

    def append(pool=kv, spec=None, heads=4, max_len=1):
        nbl_ctx.rotary_kv_append(pool, q[:, :heads].contiguous(), k, k, q[:, :heads].contiguous(), zero, one, zero, table, max_len,
                                 spec or nb.RotarySpec(1e4, False))

    append()
    refused(INV, append, f16)
    refused(INV, append, heads=3)
    refused(INV, append, max_len=33)
    for bad in (dict(rotary_dim=3), dict(rotary_dim=66), dict(rotary_dim=-2), dict(scaling="linear", factor=0.5),
                dict(scaling="yarn", factor=2.0), dict(scaling="wavelength", factor=2.0),
                dict(scaling="yarn", factor=2.0, original_ctx=64, beta_fast=0.5), dict(attn_factor=-1.0)):
        refused(INV, append, spec=nb.RotarySpec(1e4, False, **bad))
    refused(INV, append, spec=nb.RotarySpec(0.5, False))
    with pytest.raises(ValueError):
        append(spec=nb.RotarySpec(1e4, False, scaling="sideways"))
    with pytest.raises(ValueError):
        append(spec=nb.RotarySpec(1e4, False, freq_factors=(1.0,)))
    with pytest.raises(ValueError):
        nbl_ctx.rotary_kv_append(kv, q, k[:, :1].contiguous(), k, q, zero, one, zero, table, 1, nb.RotarySpec(1e4, False))
    refused(INV, nbl_ctx.kv_read, f16, zero, one, zero, table, 1, k)
    refused(INV, nbl_ctx.kv_import, f16, one, k, q)
    refused(INV, nbl_ctx.rope_kv_append, kv, q, k, k, q, zero, zero, table, 4, nb.RopeSpec(1e4, False))
    refused(INV, nbl_ctx.attn_decode, kv, q[:, :3].contiguous(), table, one, 1, q)
    refused(INV, nbl_ctx.attn_decode, kv, q, table, one, 33, q)
    refused(INV, nbl_ctx.attn_prefill, kv, q, zero, one, zero, table, 1, q.half())
    refused(INV, nbl_ctx.attn_prefill, kv, q.half(), zero, one, zero, table, 1, q.bfloat16())
    other = nb.Context(0)
    refused(INV, other.attn_decode, kv, q, table, one, 1, q)
    other.close()
    # device-side: bad page ids and lengths are skipped and flagged
    for call in (lambda: nbl_ctx.attn_decode(kv, q, ints([[9, 1]]), one, 1, q.clone()),
                 lambda: nbl_ctx.attn_decode(kv, q, table, ints([-3]), 1, q.clone()),
                 lambda: nbl_ctx.attn_decode(kv, q, table, ints([99]), 1, q.clone()),
                 lambda: nbl_ctx.attn_prefill(kv, q, zero, ints([2]), zero, table, 2, q.clone()),
                 lambda: nbl_ctx.attn_prefill(kv, q, ints([-1]), one, zero, table, 2, q.clone()),
                 lambda: nbl_ctx.attn_prefill(kv, q, zero, one, ints([32]), table, 2, q.clone()),
                 lambda: nbl_ctx.rotary_kv_append(kv, q, k, k, q.clone(), zero, one, ints([-1]), table, 1, nb.RotarySpec(1e4, False)),
                 lambda: nbl_ctx.rotary_kv_append(kv, q, k, k, q.clone(), zero, one, zero, ints([[-1, 1]]), 1, nb.RotarySpec(1e4, False)),
                 lambda: nbl_ctx.kv_read(kv, zero, ints([2]), zero, table, 2, k.clone()),
                 lambda: nbl_ctx.kv_import(kv, ints([4]), torch.zeros((1, 2, 2, 16, 64), dtype=torch.int8, device="cuda"),
                                           torch.zeros((1, 2, 2), device="cuda")),
                 lambda: nbl_ctx.kv_import(kv, ints([0]), torch.zeros((1, 2, 2, 16, 64), dtype=torch.int8, device="cuda"),
                                           torch.full((1, 2, 2), -1.0, device="cuda"))):
        call()
        refused(5, nbl_ctx.check)
    nbl_ctx.check()
    kv.close()
    f16.close()


def test_zero_rows_are_no_work(nbl_ctx):
    import torch
    import nibble_b200 as nb
    kv = nbl_ctx.kv_pool(4, 2, dtype=nb.I8)
    q, table, none = torch.zeros((0, 4, 64), device="cuda"), ints(np.zeros((0, 2))), ints([])
    nbl_ctx.attn_decode(kv, torch.zeros((1, 4, 64), device="cuda"), ints([[0]]), ints([0]), 0, torch.zeros((1, 4, 64), device="cuda"))
    nbl_ctx.check()
    assert q.numel() == 0 and none.numel() == 0 and table.numel() == 0
    kv.close()
