"""What the Python calls of the 8-bit cache and of the page bookkeeping refuse before the library sees it: tensors of another type or
size than the kernels read and write. Without a GPU: the library is a stand-in that records which calls reach it."""
import copy
import pickle
import threading

import pytest
import torch

import nibble_b200 as nb

KV, D, PAGES = 2, 64, 9


class Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *args: self.calls.append(name) or 0


@pytest.fixture
def lib(monkeypatch):
    fake = Library()
    monkeypatch.setattr(nb._abi, "lib", fake, raising=False)
    monkeypatch.setattr(nb, "_ptr", lambda t: None if t is None else 1)
    return fake


@pytest.fixture
def ctx():
    c = object.__new__(nb.Context)
    c.handle, c.device, c._unviewed = 1, 0, []
    return c


def pool(dtype=nb.I8, n_pages=PAGES):
    kv = object.__new__(nb.KVPool)
    kv.handle, kv.n_pages, kv.n_kv_heads, kv.head_dim, kv.page_size, kv.dtype = 1, n_pages, KV, D, 16, dtype
    return kv


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def refused(lib, call, *args, **kw):
    lib.calls.clear()
    with pytest.raises(ValueError):
        call(*args, **kw)
    assert not lib.calls


def rows(n=5, heads=KV, dim=D, dtype=torch.float32):
    return torch.zeros((n, heads, dim), dtype=dtype)


def test_kv_read(ctx, lib):
    def read(k=None, v=None):
        ctx.kv_read(pool(), ints(3), ints(3), ints(3), ints(3, 4), 5, k, v)

    for k, v in ((rows(), rows()), (rows(), None), (None, rows()), (rows(dtype=torch.half), rows(dtype=torch.half))):
        read(k, v)
    read(rows().reshape(5, -1), rows())
    assert lib.calls == ["nbl_kv_read"] * 5
    refused(lib, read)
    refused(lib, read, rows(), rows(dtype=torch.half))  # v_out would be written as float32
    refused(lib, read, rows(), rows(4))
    refused(lib, read, rows(), rows(heads=1))
    refused(lib, read, rows(dim=32), rows(dim=32))
    refused(lib, read, None, rows(heads=4))
    refused(lib, read, rows().reshape(-1), None)


def test_append_outputs_biases_and_items(ctx, lib):
    spec = nb.RotarySpec(1e4, False)

    def append(q_out=None, items=(3, 3, 3), table=ints(3, 4), **biases):
        q, k = rows(heads=4), rows()
        ctx.rotary_kv_append(pool(), q, k, k, rows(heads=4) if q_out is None else q_out, *map(ints, items), table, 5, spec, **biases)

    append()
    append(bq=torch.zeros(4 * D), bk=torch.zeros(KV, D), bv=torch.zeros(KV * D))
    append(q_out=rows(heads=4, dtype=torch.bfloat16), table=ints(7, 4))
    append(q_out=rows(heads=4).reshape(5, -1))
    assert len(lib.calls) == 4
    refused(lib, append, q_out=rows(4, heads=4))
    refused(lib, append, q_out=rows(heads=3))
    for name, heads in (("bq", 4), ("bk", KV), ("bv", KV)):
        refused(lib, append, **{name: torch.zeros(heads * D, dtype=torch.bfloat16)})  # was read as float32
        refused(lib, append, **{name: torch.zeros(heads * D - 1)})
    refused(lib, append, items=(3, 2, 3))
    refused(lib, append, items=(3, 3, 2))
    refused(lib, append, items=(2, 3, 3))
    refused(lib, append, table=ints(2, 4))


def test_kv_read_items(ctx, lib):
    def read(items=(3, 3, 3), table=ints(3, 4)):
        ctx.kv_read(pool(), *map(ints, items), table, 5, rows())

    read()
    read(table=ints(4, 4))
    assert len(lib.calls) == 2
    refused(lib, read, (3, 2, 3))
    refused(lib, read, (3, 3, 1))
    refused(lib, read, table=ints(2, 4))


@pytest.mark.parametrize("name", ["kv_import", "kv_export"])
def test_import_and_export_pages(ctx, lib, name):
    def call(kind=nb.I8, n=3, codes=(3, 2, KV, 16, D), dtype=torch.int8, scales=(3, 2, KV), scale_dtype=torch.float32):
        getattr(ctx, name)(pool(kind), ints(n), torch.zeros(codes, dtype=dtype), torch.zeros(scales, dtype=scale_dtype))

    call()
    call(dtype=torch.uint8)
    call(nb.E4M3, dtype=torch.float8_e4m3fn)
    call(nb.E4M3)
    call(codes=(3, 2, KV, 16 * D), scales=(3, 2 * KV))  # (flat)
    assert len(lib.calls) == 5
    refused(lib, call, n=4)  # more pages than codes
    refused(lib, call, codes=(3, 2, KV, 16, 32))
    refused(lib, call, codes=(3, 2, 1, 16, D))
    refused(lib, call, codes=(3, 1, KV, 16, D))
    refused(lib, call, dtype=torch.half)
    refused(lib, call, dtype=torch.float8_e4m3fn)  # floats for a pool of integers
    refused(lib, call, nb.E4M3, dtype=torch.float8_e5m2)
    refused(lib, call, scales=(3, 2, 1))
    refused(lib, call, scales=(2, 2, KV))
    refused(lib, call, scale_dtype=torch.half)


@pytest.mark.parametrize("name", ["kv_fork", "kv_extend", "kv_release"])
def test_page_bookkeeping_arrays(ctx, lib, name):
    def call(table=(4, 6), lens=4, refs=PAGES, first=2, second=2):
        lists = [ints(first)] if name == "kv_release" else [ints(first), ints(second)]
        getattr(ctx, name)(pool(nb.F16), ints(*table), ints(lens), ints(refs), *lists)

    call()
    call(lens=5, refs=PAGES + 1)
    assert len(lib.calls) == 2
    refused(lib, call, refs=PAGES - 1)  # counts past the end were read and written
    refused(lib, call, lens=3)
    refused(lib, call, table=(24,))
    if name != "kv_release":
        refused(lib, call, second=1)
        refused(lib, call, first=1)


def test_copy_and_compact_arrays(ctx, lib):
    ctx.kv_copy_pages(pool(), ints(3), ints(3))

    def compact(out=(4, 6), lens=4, refs=12, used=1):
        ctx.kv_compact(pool(), pool(n_pages=12), ints(4, 6), ints(lens), ints(*out), ints(refs), ints(used))

    compact()
    assert lib.calls == ["nbl_kv_copy_pages", "nbl_kv_compact"]
    refused(lib, ctx.kv_copy_pages, pool(), ints(3), ints(2))
    refused(lib, compact, out=(6, 4))
    refused(lib, compact, lens=3)
    refused(lib, compact, refs=11)
    refused(lib, compact, used=0)


def test_indices_are_int32(ctx, lib):
    """64-bit tables, lengths or lists (what a torch index is by default) are refused wherever they come."""
    kv, x, spec = pool(), rows(), nb.RotarySpec(1e4, False)
    codes, scales = torch.zeros((3, 2, KV, 16, D), dtype=torch.int8), torch.zeros((3, 2, KV))
    book = (ints(4, 6), ints(4), ints(PAGES))
    calls = [  # (call, its index arguments)
        (lambda *i: ctx.rotary_kv_append(kv, x, x, x, x, *i, 5, spec), (ints(3), ints(3), ints(3), ints(3, 4))),
        (lambda *i: ctx.kv_read(kv, *i, 5, x), (ints(3), ints(3), ints(3), ints(3, 4))),
        (lambda i: ctx.kv_import(kv, i, codes, scales), (ints(3),)),
        (lambda i: ctx.kv_export(kv, i, codes, scales), (ints(3),)),
        (lambda *i: ctx.kv_copy_pages(kv, *i), (ints(3), ints(3))),
        (lambda *i: ctx.kv_fork(kv, *i), (*book, ints(2), ints(2))),
        (lambda *i: ctx.kv_extend(kv, *i), (*book, ints(2), ints(2))),
        (lambda *i: ctx.kv_release(kv, *i), (*book, ints(2))),
        (lambda *i: ctx.kv_compact(kv, pool(), *i), (ints(4, 6), ints(4), ints(4, 6), ints(PAGES), ints(1))),
    ]
    for call, args in calls:
        call(*args)
    assert len(lib.calls) == len(calls)
    for call, args in calls:
        for k in range(len(args)):
            for dtype in (torch.int64, torch.float32):
                refused(lib, call, *args[:k], args[k].to(dtype), *args[k + 1:])


def test_decode_queries_and_rows(ctx, lib):
    def decode(q=None, out=None, lse=None, lens=ints(5), table=ints(5, 4)):
        ctx.attn_decode(pool(), rows(heads=4) if q is None else q, table, lens, 60, rows(heads=4) if out is None else out, lse)

    decode()
    decode(lse=torch.zeros((5, 4)), lens=ints(6), table=ints(6, 4))
    decode(q=rows(1, heads=4), lens=ints(1), table=ints(4))  # a single row's table
    assert len(lib.calls) == 3
    refused(lib, decode, q=rows(heads=4, dtype=torch.half))  # was read as float32
    refused(lib, decode, out=rows(heads=4, dtype=torch.half))
    refused(lib, decode, out=rows(4, heads=4))
    refused(lib, decode, q=rows(heads=4, dim=128), out=rows(heads=4, dim=128))
    refused(lib, decode, lse=torch.zeros((5, 3)))
    refused(lib, decode, lse=torch.zeros((5, 4), dtype=torch.half))
    refused(lib, decode, lens=ints(4))
    refused(lib, decode, table=ints(4, 4))
    refused(lib, decode, lens=ints(5).long())
    refused(lib, decode, table=ints(5, 4).long())


def test_prefill_queries_and_items(ctx, lib):
    def prefill(q=None, out=None, items=(3, 3, 3), table=ints(3, 4), index=torch.int32):
        ctx.attn_prefill(pool(), rows(heads=4) if q is None else q, *(ints(n).to(index) for n in items), table, 5,
                         rows(heads=4) if out is None else out)

    prefill()
    prefill(rows(heads=4, dtype=torch.half), rows(heads=4, dtype=torch.half))
    assert len(lib.calls) == 2
    refused(lib, prefill, out=rows(4, heads=4))
    refused(lib, prefill, q=rows(heads=4, dim=32))
    refused(lib, prefill, items=(3, 2, 3))
    refused(lib, prefill, items=(3, 3, 2))
    refused(lib, prefill, table=ints(2, 4))
    refused(lib, prefill, index=torch.int64)
    refused(lib, prefill, table=ints(3, 4).long())


def test_attention_over_16_bit_pools_is_called_as_before(ctx, lib):
    q = rows(heads=4)
    ctx.attn_decode(pool(nb.F16), q, ints(5, 4), ints(5), 60, q)
    ctx.attn_prefill(pool(nb.F16), q.half(), ints(3), ints(3), ints(3), ints(3, 4), 5, q)
    assert lib.calls == ["nbl_attn_decode", "nbl_attn_prefill"]


@pytest.mark.parametrize("then", ["sync", "check"])
def test_a_closed_pools_last_view_may_go_on_another_thread(ctx, lib, then):
    """The library is not called from there: a context is one thread's at a time."""
    memory = nb._PoolMemory(ctx, 7)
    views = [nb._View(memory, {}), nb._View(memory, {})]
    memory.close()
    assert not lib.calls
    t = threading.Thread(target=views.clear)
    t.start()
    t.join()
    assert not views and not lib.calls
    getattr(ctx, then)()
    assert lib.calls == ["nbl_kv_destroy", "nbl_ctx_" + then]
    getattr(ctx, then)()
    memory.close()
    assert lib.calls.count("nbl_kv_destroy") == 1


def test_a_pool_without_views_goes_at_once(ctx, lib):
    memory = nb._PoolMemory(ctx, 7)
    view = nb._View(memory, {})
    del view
    memory.close()
    assert lib.calls == ["nbl_kv_destroy"]
    ctx.sync()
    other = nb._PoolMemory(ctx, 8)
    ctx.handle = None  # closed: its pools are gone
    other.close()
    assert lib.calls == ["nbl_kv_destroy", "nbl_ctx_sync"]


def test_a_closed_pool_gives_no_view(ctx, lib, monkeypatch):
    """tensor() of a closed pool would be a view of freed memory."""
    wrapped = []
    monkeypatch.setattr(nb, "_wrap_device_memory", lambda *a: wrapped.append(a) or torch.zeros(PAGES * 2 * KV * 16 * D, dtype=torch.int16))
    kv = pool(nb.F16)
    kv.ctx, kv.base, kv.nbytes, kv._memory, kv._tensor = ctx, 4096, PAGES * 2 * KV * 16 * D * 2, nb._PoolMemory(ctx, 1), None
    assert kv.tensor().shape == (PAGES, 2, KV, 16, D)
    kv.close()
    with pytest.raises(ValueError, match="closed"):
        kv.tensor()
    assert len(wrapped) == 1


def test_a_rotary_spec_copies_and_pickles_after_its_use():
    spec = nb.RotarySpec(5e5, True, rotary_dim=8, scaling="yarn", factor=4.0, original_ctx=64, freq_factors=(1.0, 2.0, 3.0, 8.0))
    first = spec._c()
    assert spec._c() is first
    for twin in (copy.copy(spec), copy.deepcopy(spec), pickle.loads(pickle.dumps(spec))):
        assert twin == spec and hash(twin) == hash(spec)
        made, factors = twin._c()
        assert made is not first[0] and list(factors) == [1.0, 2.0, 3.0, 8.0]
        assert (made.freq_base, made.neox, made.rotary_dim, made.scaling, made.factor) == (5e5, 1, 8, nb._abi.ROTARY_SCALING["yarn"], 4.0)
