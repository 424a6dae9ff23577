"""The operators of the 8-bit K/V cache on real sizes: what each is given, its plain form, and its 64-bit definition.

Four operators share one cache of 16-token pages:

* ``append``   rotary positions on queries and keys (whole head or part of it, adjacent or half-apart pairs, scaled for
               long contexts), keys and values quantized to 8 bits with one scale per (page, K/V, head), written into
               the sequences' pages; the pass then reads the touched pages' rows back as 16-bit rows.
* ``decode``   attention of one query token per row over such a cache, with its log-sum-exp.
* ``prefill``  causal attention of several query tokens per sequence over such a cache.
* ``fork`` / ``compact``  page sharing with copy of the unfinished page, and the move of live pages into another pool.
"""
import math
import weakref

import torch

own = False

PAGE = 16
QMAX = {"int8": 127.0, "e4m3": 448.0}
TINY = 1e-30  # a block whose largest magnitude is below this is stored as zeros with scale 0
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------- the cases
def _rotary(base=1e4, half=False, rotary_dim=0, scaling="none", factor=1.0, original=0):
    return {"base": base, "half": half, "rotary_dim": rotary_dim, "scaling": scaling, "factor": factor,
            "original": original}


def listed():
    return [
        # one decode step's append: 64 sequences get one token each, most of them into a part-filled page
        {"name": "append_step", "op": "append", "items": 64, "len_lo": 1, "len_hi": 1, "pos_lo": 1, "pos_hi": 4096,
         "heads": 32, "kv_heads": 8, "head_dim": 64, "kind": "int8", "dtype": "float32", "bias": False,
         **_rotary(5e5)},
        # a batch of ragged prompts entering the cache
        {"name": "append_prompts", "op": "append", "items": 24, "len_lo": 97, "len_hi": 2047, "pos_lo": 0, "pos_hi": 0,
         "heads": 32, "kv_heads": 4, "head_dim": 64, "kind": "int8", "dtype": "bfloat16", "bias": False,
         **_rotary(1e4)},
        # one chunk of a long document: half the head rotated, context stretched four times, with biases
        {"name": "append_long_scaled", "op": "append", "items": 1, "len_lo": 8191, "len_hi": 8191, "pos_lo": 24571,
         "pos_hi": 24571, "heads": 28, "kv_heads": 4, "head_dim": 128, "kind": "e4m3", "dtype": "float16", "bias": True,
         **_rotary(1e6, True, 64, "yarn", 4.0, 32768)},
        # one short conversation: latency only
        {"name": "decode_one_short", "op": "decode", "rows": 1, "len_lo": 257, "len_hi": 257, "empty": False,
         "heads": 14, "kv_heads": 2, "head_dim": 64, "kind": "int8"},
        # the ordinary batch: 16 sequences x 16 layers of 4k tokens
        {"name": "decode_batch", "op": "decode", "rows": 256, "len_lo": 4097, "len_hi": 4097, "empty": False,
         "heads": 32, "kv_heads": 8, "head_dim": 64, "kind": "int8"},
        # ragged serving batch, one slot of it empty
        {"name": "decode_ragged", "op": "decode", "rows": 48, "len_lo": 511, "len_hi": 16384, "empty": True,
         "heads": 28, "kv_heads": 4, "head_dim": 128, "kind": "e4m3"},
        # few rows of a very long context: the split axis carries it
        {"name": "decode_long", "op": "decode", "rows": 4, "len_lo": 131073, "len_hi": 131073, "empty": False,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "kind": "int8"},
        # checking a few drafted tokens per sequence
        {"name": "prefill_drafts", "op": "prefill", "items": 8, "len_lo": 5, "len_hi": 5, "pos_lo": 777, "pos_hi": 2500,
         "heads": 14, "kv_heads": 2, "head_dim": 64, "kind": "int8", "dtype": "bfloat16"},
        # whole prompts
        {"name": "prefill_prompts", "op": "prefill", "items": 4, "len_lo": 2048, "len_hi": 2048, "pos_lo": 0,
         "pos_hi": 0, "heads": 32, "kv_heads": 4, "head_dim": 64, "kind": "int8", "dtype": "bfloat16"},
        # a chunk of a long prompt over what is already cached
        {"name": "prefill_chunk_long", "op": "prefill", "items": 1, "len_lo": 511, "len_hi": 511, "pos_lo": 16389,
         "pos_hi": 16389, "heads": 32, "kv_heads": 8, "head_dim": 128, "kind": "e4m3", "dtype": "float16"},
        # one search step: each of 8 sequences continues as 4 branches, whose old branches are dropped
        {"name": "fork_branches", "op": "fork", "groups": 8, "width": 4, "len_lo": 130, "len_hi": 2100, "kv_heads": 8},
        # the live pages of a half-empty pool move into a smaller one
        {"name": "compact_half", "op": "compact", "rows": 128, "len_lo": 500, "len_hi": 4096, "share": 4, "kv_heads": 8},
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["append", "append", "decode", "decode", "decode", "prefill", "prefill", "prefill", "fork", "compact"])
    kv_heads = rng.choice([1, 2, 4, 8])
    c = {"op": op, "kv_heads": kv_heads}
    if op in ("append", "decode", "prefill"):
        c |= {"heads": kv_heads * rng.randint(1, 8), "head_dim": rng.choice([64, 128]), "kind": rng.choice(["int8", "e4m3"])}
    if op == "append":
        items = log_int(1, 64)
        hi = log_int(1, max(1, min(8191, 24576 // items)))
        rd = rng.choice([0, 0, c["head_dim"] // 2, c["head_dim"] // 4])
        pos = log_int(1, 24576)
        c |= {"items": items, "len_lo": rng.randint(1, hi), "len_hi": hi, "pos_lo": rng.choice([0, pos // 3]), "pos_hi": pos,
              "dtype": rng.choice(["float32", "float16", "bfloat16"]), "bias": rng.random() < 0.5,
              **_rotary(rng.choice([1e4, 5e5, 1e6]), rng.random() < 0.5, rd, rng.choice(["none", "linear", "ntk", "yarn", "wavelength"]),
                        rng.choice([2.0, 4.0, 8.0]), rng.choice([4096, 8192, 32768]))}
    elif op == "decode":
        rows = log_int(1, 256)
        most = int(256 * 4097 * 8 * 64 / (rows * kv_heads * c["head_dim"]))
        hi = log_int(1, max(1, min(131073, most)))
        c |= {"rows": rows, "len_lo": log_int(1, hi), "len_hi": hi, "empty": rows > 1 and rng.random() < 0.3}
    elif op == "prefill":
        items = log_int(1, 8)
        hi = log_int(1, 2048)
        most = 1.3e11 / (4.0 * items * c["heads"] * c["head_dim"] * hi) - hi
        pos = max(0, min(log_int(1, 16389), int(most)))
        c |= {"items": items, "len_lo": rng.randint(1, hi), "len_hi": hi, "pos_lo": pos // 2, "pos_hi": pos,
              "dtype": rng.choice(["float16", "bfloat16"])}
    elif op == "fork":
        hi = log_int(1, 4096)
        c |= {"groups": log_int(1, 32), "width": rng.randint(1, 6), "len_lo": rng.randint(1, hi), "len_hi": hi}
    else:
        rows = log_int(1, 128)
        hi = log_int(1, 4096)
        c |= {"rows": rows, "len_lo": rng.randint(1, hi), "len_hi": hi, "share": rng.randint(1, 8)}
    return c


def _spread(n, lo, hi, turn=0.6180339887498949):
    """n lengths from lo to hi (the first is hi, the second lo), spread over the logarithm."""
    if n == 1 or lo == hi:
        return [hi] * n
    got = [hi, lo]
    base = max(lo, 1)
    for i in range(2, n):
        got.append(min(hi, max(lo, int(round(base * (hi / base) ** ((i * turn) % 1.0))))))
    return got


def _lens(case):
    """(query lengths, first positions) of append and prefill; (lengths,) of the others."""
    if case["op"] in ("append", "prefill"):
        n = case["items"]
        return _spread(n, case["len_lo"], case["len_hi"]), _spread(n, case["pos_lo"], case["pos_hi"], 0.7548776662466927)
    if case["op"] == "decode":
        lens = _spread(case["rows"], case["len_lo"], case["len_hi"])
        if case["empty"]:
            lens[-1] = 0
        return (lens,)
    return (_spread(case["groups" if case["op"] == "fork" else "rows"], case["len_lo"], case["len_hi"]),)


def _pages(n):
    return -(-n // PAGE)


def _page_bytes(case):
    return 2 * case["kv_heads"] * PAGE * 64 * 2  # the 16-bit pool's page, head_dim 64


def work(case):
    op = case["op"]
    if op in ("append", "decode", "prefill"):
        h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    if op == "append":
        lens, pos = _lens(case)
        wide = torch.empty((), dtype=TYPES[case["dtype"]]).element_size()
        n = sum(lens)
        old = sum(p % PAGE for p in pos)  # tokens of part-filled pages that the new scale may touch
        blocks = sum(_pages(p + m) - p // PAGE for p, m in zip(pos, lens))
        cells = kv * d
        moved = n * (2 * h * d + 2 * cells) * wide  # q in and out, k and v in
        moved += 2 * (old + n) * cells + 2 * old * cells + blocks * 2 * kv * 4  # codes out, old codes in, scales
        moved += 2 * (n + old) * cells * (1 + 2)  # the read back: codes in, 16-bit rows out
        return {"bytes": moved, "flops": 6 * n * (h + kv) * d + 4 * n * cells}
    if op == "decode":
        total = sum(_lens(case)[0])
        return {"bytes": total * 2 * kv * d + sum(_pages(x) for x in _lens(case)[0]) * 2 * kv * 4 + case["rows"] * h * (2 * d + 1) * 4,
                "flops": 4 * total * h * d}
    if op == "prefill":
        lens, pos = _lens(case)
        pairs = sum(m * p + m * (m + 1) // 2 for m, p in zip(lens, pos))
        return {"bytes": sum((p + m) * 2 * kv * d for m, p in zip(lens, pos)) + sum(lens) * 2 * h * d * 2, "flops": 4 * pairs * h * d}
    if op == "fork":
        lens = _lens(case)[0]
        w = case["width"]
        shared = sum(x // PAGE for x in lens) * w
        copied = sum(1 for x in lens if x % PAGE) * w
        return {"bytes": copied * 2 * _page_bytes(case) + shared * 4 * 3, "flops": 0}
    live = _live_pages(case)
    return {"bytes": live * 2 * _page_bytes(case) + sum(_pages(x) for x in _lens(case)[0]) * 4 * 2, "flops": 0}


def _live_pages(case):
    """Distinct pages of a compact case: every `share` rows have their first row's leading full pages in common."""
    lens = _lens(case)[0]
    live = 0
    for i, x in enumerate(lens):
        lead = lens[i - i % case["share"]]
        live += _pages(x) - (0 if i % case["share"] == 0 else min(lead // PAGE, x // PAGE))
    return live


# ---------------------------------------------------------------------------------------------------- the inputs
def _frequencies(case):
    """Angle per position of each rotated pair (float64), and the factor on cos and sin."""
    rd = case["rotary_dim"] or case["head_dim"]
    base, factor, original = case["base"], case["factor"], case["original"]
    i = torch.arange(0, rd // 2, dtype=torch.float64)
    if case["scaling"] == "ntk" and rd > 2:
        base = base * factor ** (rd / (rd - 2))
    f = base ** (-2.0 * i / rd)
    mul = 1.0
    if case["scaling"] == "linear":
        f = f / factor
    elif case["scaling"] == "yarn":
        def turns(beta):
            return rd * math.log(original / (beta * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(turns(32.0)), 0), min(math.ceil(turns(1.0)), rd - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        mul = 0.1 * math.log(factor) + 1.0
    elif case["scaling"] == "wavelength":
        wave = 2 * math.pi / f
        smooth = ((original / wave - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        f = (1 - smooth) * f / factor + smooth * f
    return f, mul


def _random(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)


def _tables(counts, seed, spare=3):
    """Rows of shuffled page ids (-1 past a row's pages), and the number of pages."""
    total, width = sum(counts) + spare, max(1, max(counts))
    ids = torch.randperm(total, generator=torch.Generator().manual_seed(int(seed) + 5)).to(torch.int32)
    table = torch.full((len(counts), width), -1, dtype=torch.int32)
    at = 0
    for r, c in enumerate(counts):
        table[r, :c] = ids[at:at + c]
        at += c
    return table.cuda(), total


def _codes(kind, shape, g):
    """Cache codes as a quantizer leaves them: the largest magnitudes of a block near the end of the range."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16).mul_(QMAX[kind] / 3.5)
    if kind == "int8":
        return x.round_().clamp_(-127, 127).to(torch.int8)
    return x.clamp_(-448, 448).to(torch.float8_e4m3fn)


def _cache(case, n_pages, seed):
    """Codes [pages + 1, 2, kv_heads, 16, head_dim] and scales [pages + 1, 2, kv_heads] (the last page is nobody's)."""
    g = _random(seed)
    kv, d = case["kv_heads"], case["head_dim"]
    codes = _codes(case["kind"], (n_pages + 1, 2, kv, PAGE, d), g)
    scales = torch.rand((n_pages + 1, 2, kv), generator=g, device="cuda").add_(0.5).mul_(3.5 / QMAX[case["kind"]])
    return codes, scales


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(lens):
    at, got = 0, []
    for x in lens:
        got.append(at)
        at += x
    return got


def _inputs(case, seed):
    op, g = case["op"], _random(seed + 1)
    s = {"case": dict(case)}
    if op in ("append", "prefill"):
        lens, pos = _lens(case)
        n, h, kv, d = sum(lens), case["heads"], case["kv_heads"], case["head_dim"]
        s["table"], n_pages = _tables([_pages(p + m) for p, m in zip(pos, lens)], seed)
        s["codes"], s["scales"] = _cache(case, n_pages, seed)
        s |= {"q_start": _ints(_starts(lens)), "q_len": _ints(lens), "pos0": _ints(pos), "max_len": max(lens)}
        t = TYPES[case["dtype"]]
        s["q"] = torch.randn((n, h, d), generator=g, device="cuda").to(t)
    if op == "append":
        # keys have channels that are larger than the others, values have not
        loud = 1.0 + 6.0 * (torch.rand((1, kv, d), generator=g, device="cuda") > 0.95)
        s["k"] = (torch.randn((n, kv, d), generator=g, device="cuda") * loud).to(t)
        s["v"] = torch.randn((n, kv, d), generator=g, device="cuda").to(t)
        for name, width in (("bq", h), ("bk", kv), ("bv", kv)):
            s[name] = torch.randn(width * d, generator=g, device="cuda") * 0.5 if case["bias"] else None
        f, mul = _frequencies(case)
        angle = torch.arange(max(p + m for p, m in zip(pos, lens)), dtype=torch.float64, device="cuda")[:, None] * f.cuda()
        s["cos"], s["sin"] = (angle.cos() * mul).float(), (angle.sin() * mul).float()
        s["q_out"] = torch.empty_like(s["q"])
        back = [p % PAGE + m for p, m in zip(pos, lens)]  # what is read back: whole pages from the first touched one
        s |= {"r_start": _ints(_starts(back)), "r_len": _ints(back), "r_pos0": _ints([p - p % PAGE for p in pos]),
              "r_max": max(back)}
        rt = torch.bfloat16 if case["dtype"] == "bfloat16" else torch.float16
        s["k_rows"] = torch.empty((sum(back), kv, d), dtype=rt, device="cuda")
        s["v_rows"] = torch.empty_like(s["k_rows"])
    elif op == "prefill":
        s["out"] = torch.empty_like(s["q"])
    elif op == "decode":
        lens = _lens(case)[0]
        s["table"], n_pages = _tables([_pages(x) for x in lens], seed)
        s["codes"], s["scales"] = _cache(case, n_pages, seed)
        s |= {"lens": _ints(lens), "max_len": max(lens)}
        s["q"] = torch.randn((len(lens), case["heads"], case["head_dim"]), generator=g, device="cuda")
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(s["q"].shape[:2], device="cuda")
    elif op == "fork":
        lens, w = _lens(case)[0], case["width"]
        src = [i for i in range(len(lens)) for _ in range(w)]
        dst = [len(lens) + i for i in range(len(src))]
        was = [max(1, lens[i] - 3) for i in src]  # the branches of the step before, dropped by this one
        s["table"], n_pages = _tables([_pages(x) for x in lens + was], seed, spare=len(src) + 7)
        wider = s["table"].shape[1]
        s |= {"lens": _ints(lens + was), "src": _ints(src), "dst": _ints(dst), "n_pages": n_pages, "wide": wider}
        s["refs"] = _counts(s["table"], n_pages)
        s["pool"] = torch.randn((n_pages, 2, case["kv_heads"], PAGE, 64), generator=g, device="cuda", dtype=torch.float16)
    else:
        lens, share = _lens(case)[0], case["share"]
        s["table"], n_pages = _tables([_pages(x) for x in lens], seed, spare=sum(_pages(x) for x in lens))
        for i in range(len(lens)):  # a shared prefix: the rows of a group have the first one's full pages
            lead = i - i % share
            common = min(lens[lead] // PAGE, lens[i] // PAGE)
            if i != lead and common:
                s["table"][i, :common] = s["table"][lead, :common]
        s |= {"lens": _ints(lens), "n_pages": n_pages, "n_out": _live_pages(case) + 2}
        s["pool"] = torch.randn((n_pages, 2, case["kv_heads"], PAGE, 64), generator=g, device="cuda", dtype=torch.float16)
        s["table_out"] = torch.full_like(s["table"], -1)
        s["refs_out"] = torch.zeros(s["n_out"], dtype=torch.int32, device="cuda")
        s["used"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        s["pool_out"] = torch.zeros((s["n_out"],) + tuple(s["pool"].shape[1:]), dtype=torch.float16, device="cuda")
    return s


def _counts(table, n_pages):
    return torch.bincount(table[table >= 0].long(), minlength=n_pages).to(torch.int32)


# ---------------------------------------------------------------------------------------------------- the framework
_contexts = []


def _context():
    """The process's one context, as a program keeps it."""
    if not _contexts:
        import nibble_b200 as nb
        _contexts.append(nb.Context(0))
    return _contexts[0]


class _Pool:
    """A pool of the framework that goes with the state that holds it."""

    def __init__(self, *args, **kw):
        self.kv = _context().kv_pool(*args, **kw)
        weakref.finalize(self, self.kv.close)


def prepare(case, seed):
    s = _inputs(case, seed)
    if not own:
        return s
    import nibble_b200 as nb
    if case["op"] in ("append", "decode", "prefill"):
        n_pages = s["codes"].shape[0] - 1
        s["held"] = _Pool(n_pages, case["kv_heads"], case["head_dim"], dtype=nb.I8 if case["kind"] == "int8" else nb.E4M3)
        ids = torch.arange(n_pages, dtype=torch.int32, device="cuda")
        _context().kv_import(s["held"].kv, ids, s.pop("codes")[:n_pages], s.pop("scales")[:n_pages])
    else:
        s["held"] = _Pool(s["n_pages"], case["kv_heads"])
        s["held"].kv.tensor().view(torch.float16).copy_(s.pop("pool"))
    if case["op"] == "append":
        s["spec"] = nb.RotarySpec(case["base"], neox=case["half"], rotary_dim=case["rotary_dim"], scaling=case["scaling"],
                                  factor=case["factor"], original_ctx=case["original"])
    if case["op"] == "compact":
        s["held_out"] = _Pool(s["n_out"], case["kv_heads"])
    return s


def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


def _own_append(s):
    ctx, kv = _context(), s["held"].kv
    ctx.rotary_kv_append(kv, s["q"], s["k"], s["v"], s["q_out"], s["q_start"], s["q_len"], s["pos0"], s["table"], s["max_len"],
                         s["spec"], bq=s["bq"], bk=s["bk"], bv=s["bv"])
    ctx.kv_read(kv, s["r_start"], s["r_len"], s["r_pos0"], s["table"], s["r_max"], s["k_rows"], s["v_rows"])
    return {"q": s["q_out"], "k": s["k_rows"], "v": s["v_rows"]}


def _own_decode(s):
    _context().attn_decode(s["held"].kv, s["q"], s["table"], s["lens"], s["max_len"], s["out"], s["lse"])
    return {"out": s["out"], "lse": s["lse"]}


def _own_prefill(s):
    _context().attn_prefill(s["held"].kv, s["q"], s["q_start"], s["q_len"], s["pos0"], s["table"], s["max_len"], s["out"])
    return s["out"]


def _own_fork(s):
    kv = s["held"].kv
    _context().kv_fork(kv, s["table"], s["lens"], s["refs"], s["src"], s["dst"])
    return {"table": s["table"], "lens": s["lens"], "refs": s["refs"], "pool": kv.tensor().view(torch.float16)}


def _own_compact(s):
    kv, to = s["held"].kv, s["held_out"].kv
    _context().kv_compact(kv, to, s["table"], s["lens"], s["table_out"], s["refs_out"], s["used"])
    return {"table": s["table_out"], "refs": s["refs_out"], "used": s["used"], "pool": to.tensor().view(torch.float16)}


# ---------------------------------------------------------------------------------------------------- the plain forms
def _rotate(x, cos, sin, half):
    """x [n, heads, head_dim] in float32, rotated in its leading 2 * cos.shape[-1] elements."""
    m = cos.shape[-1]
    a, b = (x[..., :m], x[..., m:2 * m]) if half else (x[..., 0:2 * m:2], x[..., 1:2 * m:2])
    c, d = cos[:, None, :], sin[:, None, :]
    ra, rb = a * c - b * d, a * d + b * c
    y = x.clone()
    if half:
        y[..., :m], y[..., m:2 * m] = ra, rb
    else:
        y[..., 0:2 * m:2], y[..., 1:2 * m:2] = ra, rb
    return y


def _to_codes(x, kind):
    if kind == "int8":
        return x.round().clamp(-127, 127).to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _plain_append(s):
    c = s["case"]
    kind, nobody = c["kind"], s["codes"].shape[0] - 1
    start, count, pos0 = (s[k].long() for k in ("q_start", "q_len", "pos0"))
    n = s["q"].shape[0]
    item = torch.repeat_interleave(torch.arange(len(start), device="cuda"), count, output_size=n)
    pos = torch.arange(n, device="cuda") - start[item] + pos0[item]
    x = [s[k].float() for k in ("q", "k", "v")]
    x = [t if b is None else t + b.view(1, -1, c["head_dim"]) for t, b in zip(x, (s["bq"], s["bk"], s["bv"]))]
    cos, sin = s["cos"][pos], s["sin"][pos]
    s["q_out"].copy_(_rotate(x[0], cos, sin, c["half"]))
    new = torch.stack([_rotate(x[1], cos, sin, c["half"]), x[2]], 1)  # [n, 2, kv, d]
    # the touched pages of each item, and what stands in each of their 16 places afterwards
    most = (s["max_len"] + PAGE - 2) // PAGE + 1
    block = pos0[:, None] // PAGE + torch.arange(most, device="cuda")
    live = block * PAGE < (pos0 + count)[:, None]
    page = torch.where(live, s["table"].long().gather(1, block.clamp(max=s["table"].shape[1] - 1)), nobody)
    place = block[..., None] * PAGE + torch.arange(PAGE, device="cuda")
    is_old = (place < pos0[:, None, None])[..., None, None, :, None]
    is_new = ((place >= pos0[:, None, None]) & (place < (pos0 + count)[:, None, None]))[..., None, None, :, None]
    token = (start[:, None, None] + place - pos0[:, None, None]).clamp(0, n - 1)
    fresh = new[token].permute(0, 1, 3, 4, 2, 5)  # [items, blocks, 2, kv, 16, d]
    largest = torch.where(is_new, fresh.abs(), 0.0).amax((-1, -2))
    wanted = torch.where(largest >= TINY, largest / QMAX[kind], 0.0)
    before = torch.where(is_old[..., 0].any(-1), s["scales"][page], 0.0)
    scale = torch.maximum(before, wanted)
    inverse = torch.where(scale > 0, 1.0 / scale, 0.0)
    kept = s["codes"][page].float() * (before * inverse)[..., None, None]
    value = torch.where(is_old, kept, torch.where(is_new, fresh * inverse[..., None, None], 0.0))
    if kind == "int8":
        s["codes"][page] = _to_codes(value, kind)
    else:
        s["codes"].view(torch.uint8)[page] = _to_codes(value, kind).view(torch.uint8)
    s["scales"][page] = scale
    # read back
    total = s["k_rows"].shape[0]
    start, count, pos0 = (s[k].long() for k in ("r_start", "r_len", "r_pos0"))
    item = torch.repeat_interleave(torch.arange(len(start), device="cuda"), count, output_size=total)
    pos = torch.arange(total, device="cuda") - start[item] + pos0[item]
    page = s["table"].long()[item, pos // PAGE]
    if kind == "int8":
        rows = s["codes"][page, :, :, pos % PAGE].float()
    else:
        rows = s["codes"].view(torch.uint8)[page, :, :, pos % PAGE].view(torch.float8_e4m3fn).float()
    rows = rows * s["scales"][page][..., None]
    s["k_rows"].copy_(rows[:, 0])
    s["v_rows"].copy_(rows[:, 1])
    return {"q": s["q_out"], "k": s["k_rows"], "v": s["v_rows"]}


def _gathered(s):
    """The rows' keys and values in float32: two of [rows, kv, places, d]."""
    page = s["table"].long().clamp(min=0)
    codes = s["codes"].view(torch.uint8)[page].view(s["codes"].dtype)
    x = codes.float().mul_(s["scales"][page][..., None, None])  # [rows, pages, 2, kv, 16, d]
    x = x.permute(2, 0, 3, 1, 4, 5).flatten(3, 4)
    return x[0], x[1]


def _attend(q, k, v, visible):
    """q [rows, kv, m, d], k and v [rows, kv, places, d], visible [rows, 1, m, places] -> outputs and log-sum-exp."""
    score = torch.matmul(q * (1.0 / math.sqrt(q.shape[-1])), k.transpose(-1, -2))
    score = torch.where(visible, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = (score - torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    return out, (top + total.log())[..., 0]


def _plain_decode(s):
    k, v = _gathered(s)
    rows, h, d = s["q"].shape
    kv = k.shape[1]
    visible = torch.arange(k.shape[2], device="cuda") < s["lens"][:, None]
    out, lse = _attend(s["q"].view(rows, kv, h // kv, d), k, v, visible[:, None, None, :])
    s["out"].copy_(out.reshape(rows, h, d))
    s["lse"].copy_(lse.reshape(rows, h))
    return {"out": s["out"], "lse": s["lse"]}


def _plain_prefill(s):
    k, v = _gathered(s)
    n, h, d = s["q"].shape
    items, kv, m = k.shape[0], k.shape[1], s["max_len"]
    start, count, pos0 = (s[x].long() for x in ("q_start", "q_len", "pos0"))
    token = (start[:, None] + torch.arange(m, device="cuda")).clamp(max=n - 1)
    q = s["q"].float()[token].view(items, m, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(items, kv, -1, d)
    seen = torch.arange(k.shape[2], device="cuda") <= (pos0[:, None] + torch.arange(m, device="cuda"))[..., None]
    out, _ = _attend(q, k, v, seen[:, None].repeat(1, 1, h // kv, 1))
    out = out.view(items, kv, h // kv, m, d).permute(0, 3, 1, 2, 4).reshape(items, m, h, d)
    item = torch.repeat_interleave(torch.arange(items, device="cuda"), count, output_size=n)
    s["out"].copy_(out[item, torch.arange(n, device="cuda") - start[item]])
    return s["out"]


def _plain_fork(s):
    table, lens, refs, pool = s["table"], s["lens"], s["refs"], s["pool"]
    src, dst = s["src"].long(), s["dst"].long()
    refs -= _counts(table[dst], s["n_pages"])
    full = (lens[src] // PAGE)[:, None]
    mine = torch.where(torch.arange(table.shape[1], device="cuda") < full, table[src], -1)
    refs += _counts(mine, s["n_pages"])
    part = lens[src] % PAGE > 0
    free = (refs == 0).nonzero()[:, 0]
    page = free[(part.cumsum(0) - 1).clamp(min=0)]  # the k-th part-filled page goes to the k-th free one
    here = part[:, None] & (torch.arange(table.shape[1], device="cuda") == full)
    source = table[src].gather(1, full.long().clamp(max=table.shape[1] - 1))[:, 0].long()
    table[dst] = torch.where(here, page[:, None].to(torch.int32), mine)
    lens[dst] = lens[src]
    pool[page[part]] = pool[source[part]]
    refs[page[part]] = 1
    return {"table": table, "lens": lens, "refs": refs, "pool": pool}


def _plain_compact(s):
    table = s["table"]
    held = torch.arange(table.shape[1], device="cuda") < ((s["lens"] + PAGE - 1) // PAGE)[:, None]
    flat = table[held].long()
    first = torch.full((s["n_pages"],), flat.numel(), dtype=torch.long, device="cuda")
    first.scatter_reduce_(0, flat, torch.arange(flat.numel(), device="cuda"), "amin")
    order = torch.sort(first).indices  # pages by their first appearance, the unused ones last
    new_id = torch.empty_like(order)
    new_id[order] = torch.arange(order.numel(), device="cuda")
    used = (first < flat.numel()).sum()
    s["used"].copy_(used)
    s["table_out"].fill_(-1)
    s["table_out"][held] = new_id[flat].to(torch.int32)
    s["refs_out"].copy_(torch.bincount(new_id[flat], minlength=s["n_out"])[:s["n_out"]])
    s["pool_out"][:used] = s["pool"][order[:used]]
    return {"table": s["table_out"], "refs": s["refs_out"], "used": s["used"], "pool": s["pool_out"]}


_plain = {"append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill, "fork": _plain_fork, "compact": _plain_compact}
_own = {"append": _own_append, "decode": _own_decode, "prefill": _own_prefill, "fork": _own_fork, "compact": _own_compact}


# ---------------------------------------------------------------------------------------------------- the definition
def _stored(s, page, places):
    """Keys and values of the first `places` places of a row's pages, in float64: two of [places, kv, d]."""
    x = s["codes"].view(torch.uint8)[page].view(s["codes"].dtype).double()
    x = x * s["scales"][page].double()[..., None, None]
    x = x.transpose(2, 3).permute(0, 2, 1, 3, 4).reshape(-1, 2, x.shape[2], x.shape[4])[:places]
    return x[:, 0], x[:, 1]


def exact(case, seed):
    op = case["op"]
    if op in ("fork", "compact"):
        return None  # whole numbers and copies
    s = _inputs(case, seed)
    lens = _lens(case)
    if op == "append":
        return _exact_append(case, s, *lens)
    out, lse = torch.zeros_like(s["q"], dtype=torch.float64), None
    if op == "decode":
        lse = torch.full_like(s["lse"], -math.inf, dtype=torch.float64)
    group, root, at = case["heads"] // case["kv_heads"], math.sqrt(case["head_dim"]), 0
    counts, pos = lens if op == "prefill" else ([1] * case["rows"], [x - 1 for x in lens[0]])
    for r, (m, p) in enumerate(zip(counts, pos)):
        if p + m > 0:
            k, v = _stored(s, s["table"][r, :_pages(p + m)].long(), p + m)
            later = torch.arange(p + m, device="cuda") > torch.arange(p, p + m, device="cuda")[:, None]
            for h in range(case["heads"]):
                score = (s["q"][at:at + m, h].double() @ k[:, h // group].T / root).masked_fill(later, -math.inf)
                out[at:at + m, h] = torch.softmax(score, -1) @ v[:, h // group]
                if op == "decode":
                    lse[at:at + m, h] = torch.logsumexp(score, -1)
        at += m
    return {"out": out, "lse": lse} if op == "decode" else out


def _exact_append(case, s, lens, pos):
    kind, d = case["kind"], case["head_dim"]
    f, mul = _frequencies(case)
    q, rows = torch.empty_like(s["q"], dtype=torch.float64), []
    at = 0
    for i, (m, p) in enumerate(zip(lens, pos)):
        part = slice(at, at + m)
        angle = torch.arange(p, p + m, dtype=torch.float64, device="cuda")[:, None] * f.cuda()
        turn = torch.polar(torch.full_like(angle, mul), angle)[:, None]
        got = []
        for x, b in ((s["q"], s["bq"]), (s["k"], s["bk"]), (s["v"], s["bv"])):
            x = x[part].double()
            got.append(x if b is None else x + b.double().view(1, -1, d))
        for x in got[:2]:
            w = f.numel()
            both = torch.complex(x[..., :w], x[..., w:2 * w]) if case["half"] else torch.complex(x[..., 0:2 * w:2], x[..., 1:2 * w:2])
            both = both * turn
            if case["half"]:
                x[..., :2 * w] = torch.cat([both.real, both.imag], -1)
            else:
                x[..., :2 * w] = torch.view_as_real(both).flatten(-2)
        q[part] = got[0]
        # whole pages from the first touched one: the tokens that were there, then the new ones
        old, pages = p % PAGE, s["table"][i, p // PAGE:_pages(p + m)].long()
        fresh = torch.stack(got[1:], 1)
        fresh = torch.cat([fresh.new_zeros((old,) + fresh.shape[1:]), fresh, fresh.new_zeros((-(p + m) % PAGE,) + fresh.shape[1:])])
        fresh = fresh.view(-1, PAGE, 2, case["kv_heads"], d).permute(0, 2, 3, 1, 4)
        scale = fresh.abs().amax((-1, -2)) / QMAX[kind]
        value = None
        if old:
            was = s["scales"][pages[0]].double()
            scale[0] = torch.maximum(scale[0], was)
            value = s["codes"].view(torch.uint8)[pages[0]].view(s["codes"].dtype).double()[..., :old, :] * was[..., None, None]
            fresh[0, ..., :old, :] = value
        code = fresh / scale.clamp(min=1e-300)[..., None, None]
        code = code.round() if kind == "int8" else code.clamp(-448, 448).to(torch.float8_e4m3fn).double()
        back = (code * scale[..., None, None]).permute(0, 3, 1, 2, 4).reshape(-1, 2, case["kv_heads"], d)
        rows.append(back[:old + m])
        at += m
    rows = torch.cat(rows)
    return {"q": q, "k": rows[:, 0].contiguous(), "v": rows[:, 1].contiguous()}
