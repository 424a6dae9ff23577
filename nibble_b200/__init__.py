"""nibble_b200: a B200 (sm_100a) attention backend for nibble, behind a C ABI (include/nibble_cuda.h).

The product is ``libnibble_cuda.so``: hand-written CUDA kernels for grouped-query attention (tcgen05/TMEM prefill,
split-K flash-decode over a paged fp16 K/V pool, fused bias+RoPE+append, LSE merge) and the drop-in fp32
operations of nibble's ``Backend`` interface. This package is the Python view of that ABI, used by the tests, the
benchmark and multi-GPU drivers; ``csrc/host/cuda_backend.h`` is the C++ view, mirroring ``nibble::Backend``.

Tensors passed here are torch CUDA tensors (torch is only the device-memory and stream plumbing); every compute
call goes through the C ABI. There is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

from . import _abi
from ._abi import BF16, E4M3, F16, F32, I8, Q4_0, Q4_K, Q5_0, Q5_1, Q5_K, Q6_K, Q8_0, NibbleError, check

__all__ = ["Context", "KVPool", "Weight", "NibbleError", "RopeSpec", "RotarySpec", "F32", "F16", "BF16", "I8", "E4M3", "Q4_0", "Q5_0", "Q8_0", "Q5_1",
           "Q4_K", "Q5_K", "Q6_K",
           "abi_version"]


def abi_version() -> int:
    return _abi.lib.nbl_abi_version()


@dataclass(frozen=True)
class RopeSpec:
    """nibble's RopeParams (src/backend/backend.h:16-20): base, NeoX pairing, optional per-pair factors."""
    freq_base: float
    neox: bool
    freq_factors: tuple | None = None

    def _c(self):
        ff = None
        ptr = None
        if self.freq_factors is not None:
            ff = (C.c_float * len(self.freq_factors))(*self.freq_factors)
            ptr = C.cast(ff, C.c_void_p)
        return _abi.RopeParams(self.freq_base, int(self.neox), ptr), ff


@dataclass(frozen=True)
class RotarySpec:
    """Rotary positions of part of a head, stretched for long contexts (nbl_rotary_params): the first rotary_dim elements
    (0: all) rotate, as pairs (i, i + n/2) with neox, else (2i, 2i + 1). scaling: "none", "linear", "ntk", "yarn" or
    "wavelength", for a context `factor` times the original one of original_ctx tokens."""
    freq_base: float
    neox: bool
    rotary_dim: int = 0
    scaling: str = "none"
    factor: float = 1.0
    original_ctx: int = 0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    low_freq_factor: float = 1.0
    high_freq_factor: float = 4.0
    attn_factor: float = 0.0
    freq_factors: tuple | None = None

    def _c(self):
        """The C struct and the factors that it points to (made once)."""
        made = self.__dict__.get("_made")
        if made is None:
            made = self._make()
            object.__setattr__(self, "_made", made)
        return made

    def __getstate__(self):
        """For copies and pickles: the fields, without the C struct and its pointers."""
        return {k: v for k, v in self.__dict__.items() if k != "_made"}

    def _make(self):
        if self.scaling not in _abi.ROTARY_SCALING:
            raise ValueError(f"unknown rotary scaling {self.scaling!r} (one of {', '.join(_abi.ROTARY_SCALING)})")
        ff = ptr = None
        if self.freq_factors is not None:
            ff = (C.c_float * len(self.freq_factors))(*self.freq_factors)
            ptr = C.cast(ff, C.c_void_p)
        return _abi.RotaryParams(self.freq_base, int(self.neox), self.rotary_dim, _abi.ROTARY_SCALING[self.scaling],
                                 self.factor, self.original_ctx, self.beta_fast, self.beta_slow, self.low_freq_factor,
                                 self.high_freq_factor, self.attn_factor, ptr), ff


_DT = {"float32": F32, "float16": F16, "bfloat16": BF16}


def torch_float32():
    import torch
    return torch.float32


def _ptr(t) -> int | None:
    if t is None:
        return None
    if isinstance(t, int):
        return t
    if not t.is_cuda:
        raise ValueError("expected a CUDA tensor")
    if not t.is_contiguous():
        raise ValueError("expected a contiguous tensor")
    return t.data_ptr()


_int32: set = set()  # torch.int32, once it has been seen


def _ints(t) -> int:
    """Pointer to an int32 tensor: positions, lengths, page ids (another type's elements would be read as pairs of int32)."""
    if t.dtype not in _int32:
        if str(t.dtype) != "torch.int32":
            raise ValueError(f"expected an int32 tensor, not {t.dtype}")
        _int32.add(t.dtype)
    if t.is_cuda and t.is_contiguous():
        return t.data_ptr()
    return _ptr(t)  # says what is wrong


_codes: dict = {}  # torch dtype -> element type code


def _dtype(t) -> int:
    code = _codes.get(t.dtype)
    if code is None:
        name = str(t.dtype).replace("torch.", "")
        if name not in _DT:
            raise ValueError(f"unsupported dtype {t.dtype}")
        code = _codes[t.dtype] = _DT[name]
    return code


def _new_rows(kv, q, k, v, q_out):
    """(rows, query heads) of tokens for kv: q [rows, heads, D], q_out as many elements, k and v [rows, kv heads, D]."""
    shape = q.shape
    n, heads, dim = shape
    if dim != kv.head_dim or q_out.numel() != n * heads * dim or k.shape != (n, kv.n_kv_heads, dim) or v.shape != k.shape:
        raise ValueError(f"expected q_in, q_out [rows, n_heads, {kv.head_dim}] and k_in, v_in [rows, {kv.n_kv_heads}, {kv.head_dim}]")
    return n, heads


def _items(first, second, third, page_table):
    """Pointers to an item's three entries and to the page table, which has a row for each; its stride, and the items. (One
    function for the four: the checks of a small call cost as much as its launch.)"""
    n, stride, dtype = first.numel(), page_table.shape[-1], first.dtype
    if second.numel() != n or third.numel() != n or page_table.numel() < n * stride:
        raise ValueError("expected one start, length and first position per item, and a page-table row for each")
    if (dtype in _int32 and second.dtype is dtype and third.dtype is dtype and page_table.dtype is dtype and
            first.is_cuda and second.is_cuda and third.is_cuda and page_table.is_cuda and first.is_contiguous() and
            second.is_contiguous() and third.is_contiguous() and page_table.is_contiguous()):
        return first.data_ptr(), second.data_ptr(), third.data_ptr(), page_table.data_ptr(), stride, n
    return _ints(first), _ints(second), _ints(third), _ints(page_table), stride, n


def _book(kv, page_table, seq_lens, ref_counts, first, second):
    """(table rows, stride, list entries): a length per table row, a count per page of the pool, lists of one length."""
    (n_rows, stride), n = page_table.shape, first.numel()
    if seq_lens.numel() < n_rows or ref_counts.numel() < kv.n_pages or second.numel() != n:
        raise ValueError("expected seq_lens for every table row, ref_counts for every page, and lists of one length")
    return n_rows, stride, n


def _check_bias(b, heads, dim):
    if _dtype(b) != F32 or b.numel() != heads * dim:
        raise ValueError(f"expected a float32 bias of {heads} * {dim} elements")


_EIGHT_BITS = (I8, E4M3)


def _check_pages(kv, page_ids, codes, scales):
    """Import and export: one byte a code, every page whole. (A pool of another type is refused by the library.)"""
    if kv.dtype not in _EIGHT_BITS:
        return
    want = (page_ids.numel(), 2, kv.n_kv_heads, kv.page_size, kv.head_dim)
    types = ("int8", "uint8", "float8_e4m3fn") if kv.dtype == E4M3 else ("int8", "uint8")
    if codes.numel() != want[0] * 2 * want[2] * want[3] * want[4] or str(codes.dtype).replace("torch.", "") not in types:
        raise ValueError(f"expected codes {list(want)} of {' or '.join(types)}")
    if scales.numel() != want[0] * 2 * want[2] or _dtype(scales) != F32:
        raise ValueError(f"expected float32 scales {list(want[:3])}")


class KVPool:
    """A paged K/V pool: pool[page][2][n_kv_heads][page_size][head_dim] (fp16 or bf16), or with dtype I8 / E4M3 8-bit
    codes with a scale per (page, K/V, head), in an order of the library's own (Context.kv_import / kv_export)."""

    def __init__(self, ctx: "Context", n_pages: int, n_kv_heads: int, head_dim: int = 64, page_size: int = 16,
                 dtype: int = F16):
        self.ctx = ctx
        cfg = _abi.KvConfig(n_pages, n_kv_heads, head_dim, page_size, dtype)
        h = C.c_void_p()
        check(_abi.lib.nbl_kv_create(ctx.handle, C.byref(cfg), C.byref(h)))
        self.handle = h
        self._memory, self._tensor = _PoolMemory(ctx, h), None
        self.n_pages, self.n_kv_heads, self.head_dim, self.page_size, self.dtype = (n_pages, n_kv_heads, head_dim,
                                                                                    page_size, dtype)
        base, nbytes = C.c_void_p(), C.c_int64()
        check(_abi.lib.nbl_kv_pool(h, C.byref(base), C.byref(nbytes)))
        self.base, self.nbytes = base.value, nbytes.value

    def tensor(self):
        """The pool's raw 16-bit elements as a torch int16 view [n_pages, 2, n_kv_heads, page_size, head_dim]
        (aliases the pool; no copy). Reinterpret with .view(torch.float16 / torch.bfloat16)."""
        import torch
        if self.dtype in (I8, E4M3):
            raise ValueError("an 8-bit pool has no plain view: use Context.kv_read, kv_export and kv_import")
        if self.handle is None:
            raise ValueError("the pool is closed")
        if self._tensor is None:
            t = _wrap_device_memory(self.base, self.nbytes // 2, torch.int16, self.ctx.device, self._memory)
            self._tensor = t.view(self.n_pages, 2, self.n_kv_heads, self.page_size, self.head_dim)
        return self._tensor.view(self._tensor.shape)

    def close(self):
        """Frees the pool; while tensors from tensor() are alive, at the context's next kv_pool(), sync() or check() after the
        last of them is gone."""
        self.handle = self._tensor = None
        self._memory.close()


class _PoolMemory:
    """A pool's device memory: freed when the pool is closed and no tensor views it any more, by a call of the context's user:
    the last view may go on any thread, at any point, where the library must not be called."""

    def __init__(self, ctx: "Context", handle):
        self.ctx, self.handle, self.views, self.closing = ctx, handle, [], False  # a list: its changes are atomic

    def close(self):
        self.closing = True
        if not self.views:
            self.free()

    def free(self):
        handle, self.handle = self.handle, None
        if handle and self.ctx.handle:  # a closed context has freed its pools
            check(_abi.lib.nbl_kv_destroy(handle))


class _View:
    """What a tensor over a pool's memory holds on to."""

    def __init__(self, memory: _PoolMemory, interface: dict):
        self.__cuda_array_interface__ = interface
        self.memory = memory
        memory.views.append(None)

    def __del__(self):
        memory = self.memory
        memory.views.pop()
        if memory.closing and not memory.views:
            memory.ctx._unviewed.append(memory)


class Weight:
    """A weight tensor uploaded to the device (nbl_weight): ne1 rows of ne0 elements, F32 or F16 -- the device form
    of nibble's Tensor view (src/tensor.h:57-70)."""

    def __init__(self, ctx: "Context", host, dtype: int | None = None, ne0: int | None = None):
        """host: a C-contiguous numpy float32 / float16 array, 1-D (a vector) or 2-D [ne1, ne0]; or, with dtype
        a quantized type (Q4_0 / Q5_0 / Q8_0 / Q5_1 / Q4_K / Q5_K / Q6_K) and ne0 given, the GGUF block bytes as
        uint8 [ne1, row bytes]."""
        import numpy as np
        a = np.ascontiguousarray(host)
        if dtype is None:
            dtype = {np.dtype(np.float32): F32, np.dtype(np.float16): F16}.get(a.dtype)
            if dtype is None:
                raise ValueError(f"weights must be float32 or float16, got {a.dtype}")
        if dtype in (Q4_0, Q5_0, Q8_0, Q5_1, Q4_K, Q5_K, Q6_K):
            if ne0 is None or a.ndim != 2:
                raise ValueError("quantized weights take uint8 blocks [ne1, row bytes] and ne0")
            ne1 = a.shape[0]
        else:
            ne1, ne0 = (1, a.shape[0]) if a.ndim == 1 else a.shape
        h = C.c_void_p()
        check(_abi.lib.nbl_weight_create(ctx.handle, a.ctypes.data, dtype, ne0, ne1, C.byref(h)))
        self.ctx, self.handle, self.ne0, self.ne1, self.dtype = ctx, h, ne0, ne1, dtype

    def close(self):
        if self.handle:
            check(_abi.lib.nbl_weight_destroy(self.handle))
            self.handle = None


def _wrap_device_memory(ptr: int, numel: int, dtype, device: int, memory: _PoolMemory):
    """A torch tensor aliasing `numel` elements of the pool's device memory at `ptr`."""
    import torch
    elsize = torch.empty((), dtype=dtype).element_size()
    view = _View(memory, {"shape": (numel,), "typestr": {torch.int16: "<i2", torch.float32: "<f4"}[dtype],
                          "data": (ptr, False), "version": 3, "strides": (elsize,)})
    with torch.cuda.device(device):
        return torch.as_tensor(view, device=f"cuda:{device}")


class Context:
    """An nbl_ctx on one device. By default its kernels run on torch's current stream for that device, so they
    order correctly with the torch ops that prepare inputs."""

    def __init__(self, device: int = 0, use_torch_stream: bool = True):
        h = C.c_void_p()
        check(_abi.lib.nbl_ctx_create(device, C.byref(h)))
        self.handle = h
        self.device = device
        self._unviewed = []  # memory of closed pools whose last view is gone
        if use_torch_stream:
            import torch
            self.set_stream(torch.cuda.current_stream(device).cuda_stream)

    # ---- context
    def set_stream(self, stream: int | None):
        """Runs later kernels on this cudaStream_t (0 / None = CUDA's default stream)."""
        check(_abi.lib.nbl_ctx_set_stream(self.handle, stream))

    def set_paged_kv(self, on: bool = True):
        """Backend-level K/V blocks as fp16 pages with the fused append and the paged kernels (nbl_ctx_set_paged_kv);
        call before reserve() and before allocating the blocks."""
        check(_abi.lib.nbl_ctx_set_paged_kv(self.handle, 1 if on else 0))

    def _free_unviewed(self):
        while self._unviewed:
            self._unviewed.pop().free()

    def sync(self):
        self._free_unviewed()
        check(_abi.lib.nbl_ctx_sync(self.handle))

    def check(self):
        """Raises NibbleError(NBL_E_DEVICE) if a kernel flagged an out-of-range device-side index."""
        self._free_unviewed()
        check(_abi.lib.nbl_ctx_check(self.handle))

    def close(self):
        if self.handle:
            check(_abi.lib.nbl_ctx_destroy(self.handle))
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    # ---- Backend memory (backend.h:45-53)
    def reserve(self, n_ctx: int, n_heads: int, max_rows: int = 1, max_width: int = 0):
        check(_abi.lib.nbl_reserve(self.handle, n_ctx, n_heads, max_rows, max_width))

    def alloc(self, n_floats: int) -> int:
        p = C.c_void_p()
        check(_abi.lib.nbl_alloc(self.handle, n_floats, C.byref(p)))
        return p.value

    def free(self, p: int | None):
        check(_abi.lib.nbl_free(self.handle, p))

    def read(self, host_dst, src: int, n: int):
        """Backend::read into a float32 numpy array (or anything exposing a ctypes data pointer)."""
        check(_abi.lib.nbl_read(self.handle, host_dst.ctypes.data, src, n))

    def write(self, dst: int, host_src, n: int):
        check(_abi.lib.nbl_write(self.handle, dst, host_src.ctypes.data, n))

    # ---- Backend ops on fp32 device buffers (pointers or CUDA tensors)
    def add_bias(self, x, bias, width: int, n: int):
        check(_abi.lib.nbl_add_bias(self.handle, _ptr(x), _ptr(bias), width, n))

    def rope(self, x, n: int, n_heads: int, head_dim: int, pos0: int, rope: RopeSpec):
        p, keep = rope._c()
        check(_abi.lib.nbl_rope(self.handle, _ptr(x), n, n_heads, head_dim, pos0, C.byref(p)))

    def attention(self, q, k, v, out, n: int, pos0: int, n_heads: int, n_kv_heads: int, head_dim: int):
        check(_abi.lib.nbl_attention(self.handle, _ptr(q), _ptr(k), _ptr(v), _ptr(out), n, pos0, n_heads, n_kv_heads,
                                     head_dim))

    # ---- the model's other Backend ops (backend.h:54-70) on fp32 device buffers
    def weight(self, host, dtype: int | None = None, ne0: int | None = None) -> Weight:
        return Weight(self, host, dtype, ne0)

    def embed(self, table: Weight, ids, out):
        """ids: host int32 array (a std::span in the reference); out [n, ne0] fp32."""
        import numpy as np
        ids = np.ascontiguousarray(ids, dtype=np.int32)
        check(_abi.lib.nbl_embed(self.handle, table.handle, ids.ctypes.data, ids.shape[0], _ptr(out)))

    def matmul(self, w: Weight, x, y, n: int):
        """y[n, ne1] = x[n, ne0] . W^T"""
        check(_abi.lib.nbl_matmul(self.handle, w.handle, _ptr(x), _ptr(y), n))

    def matmul_multi(self, ws, x, ys, n: int):
        """ys[i][n, ws[i].ne1] = x[n, ne0] . ws[i]^T for weights sharing one input (one launch for n <= 8)."""
        count = len(ws)
        warr = (C.c_void_p * count)(*[w.handle.value for w in ws])
        yarr = (C.c_void_p * count)(*[_ptr(y) for y in ys])
        check(_abi.lib.nbl_matmul_multi(self.handle, warr, count, _ptr(x), yarr, n))

    def rmsnorm(self, x, weight: Weight, y, n: int, eps: float):
        check(_abi.lib.nbl_rmsnorm(self.handle, _ptr(x), weight.handle, _ptr(y), n, eps))

    def add(self, x, y, count: int):
        check(_abi.lib.nbl_add(self.handle, _ptr(x), _ptr(y), count))

    def copy(self, dst, src, count: int):
        check(_abi.lib.nbl_copy(self.handle, _ptr(dst), _ptr(src), count))

    def silu_mul(self, gate, up, count: int):
        check(_abi.lib.nbl_silu_mul(self.handle, _ptr(gate), _ptr(up), count))

    # ---- paged path
    def kv_pool(self, n_pages: int, n_kv_heads: int, head_dim: int = 64, page_size: int = 16,
                dtype: int = F16) -> KVPool:
        self._free_unviewed()
        return KVPool(self, n_pages, n_kv_heads, head_dim, page_size, dtype)

    def rope_kv_append(self, kv: KVPool, q_in, k_in, v_in, q_out, tok_row, tok_pos, page_table, n_heads: int,
                       rope: RopeSpec, bq=None, bk=None, bv=None):
        """Fused bias -> RoPE -> narrowing -> page write for q_in.shape[0] tokens (see nbl_rope_kv_append)."""
        p, keep = rope._c()
        in_dt = _dtype(q_in)
        if _dtype(k_in) != in_dt or _dtype(v_in) != in_dt:
            raise ValueError("q_in, k_in, v_in must share a dtype")
        check(_abi.lib.nbl_rope_kv_append(
            self.handle, kv.handle, _ptr(q_in), _ptr(k_in), _ptr(v_in), in_dt, _ptr(bq), _ptr(bk), _ptr(bv),
            _ptr(q_out), _dtype(q_out), _ptr(tok_row), _ptr(tok_pos), _ptr(page_table), page_table.shape[-1],
            q_in.shape[0], n_heads, C.byref(p)))

    def attn_decode(self, kv: KVPool, q, page_table, seq_lens, max_seq_len: int, out, lse=None, n_splits: int = 0):
        """One query token per row: q/out [rows, n_heads, head_dim] fp32, page_table [rows, stride] int32."""
        if kv.dtype in _EIGHT_BITS:
            (rows, heads, dim), stride, f32 = q.shape, page_table.shape[-1], q.dtype
            if dim != kv.head_dim or _dtype(q) != F32 or out.dtype != f32 or out.numel() < rows * heads * dim:
                raise ValueError(f"expected float32 q and out [rows, n_heads, {kv.head_dim}]")
            if page_table.numel() < rows * stride or seq_lens.numel() < rows:
                raise ValueError("expected a length and a page-table row for each row of q")
            if lse is not None and (lse.dtype != f32 or lse.numel() < rows * heads):
                raise ValueError("expected a float32 lse [rows, n_heads]")
            check(_abi.lib.nbl_attn_decode(self.handle, kv.handle, _ptr(q), _ints(page_table), stride, _ints(seq_lens),
                                           max_seq_len, rows, heads, _ptr(out), _ptr(lse), n_splits))
            return
        check(_abi.lib.nbl_attn_decode(self.handle, kv.handle, _ptr(q), _ptr(page_table), page_table.shape[-1],
                                       _ptr(seq_lens), max_seq_len, q.shape[0], q.shape[1], _ptr(out), _ptr(lse),
                                       n_splits))

    def decode_step_host(self, kv: KVPool, q_in_h, k_in_h, v_in_h, page_table, seq_lens, max_seq_len: int,
                         rope: RopeSpec, out_h, bq=None, bk=None, bv=None, n_chunks: int = 0):
        """One decode step from host memory (see nbl_decode_step_host): q_in_h [rows, H, D], k_in_h/v_in_h
        [rows, KVH, D] and out_h [rows, H, D] are fp32 host tensors (pinned for overlapped copies); page_table
        and seq_lens (counting the new token) are device tensors."""
        for t in (q_in_h, k_in_h, v_in_h, out_h):
            if t.is_cuda or not t.is_contiguous() or t.dtype != torch_float32():
                raise ValueError("host tensors must be contiguous float32 CPU tensors")
        p, keep = rope._c()
        check(_abi.lib.nbl_decode_step_host(
            self.handle, kv.handle, q_in_h.data_ptr(), k_in_h.data_ptr(), v_in_h.data_ptr(), _ptr(bq), _ptr(bk),
            _ptr(bv), _ptr(page_table), page_table.shape[-1], _ptr(seq_lens), max_seq_len, q_in_h.shape[0],
            q_in_h.shape[1], C.byref(p), out_h.data_ptr(), n_chunks))

    def attn_prefill(self, kv: KVPool, q, q_start, q_len, kv_pos0, page_table, max_q_len: int, out):
        """Causal prefill: q [rows, n_heads, head_dim] (pool dtype), out [rows, n_heads, head_dim] fp32/pool dtype.
        (8-bit pools: q fp32, fp16 or bf16, out fp32 or q's dtype.)"""
        if kv.dtype in _EIGHT_BITS:
            rows, heads, dim = q.shape
            if dim != kv.head_dim or out.numel() < rows * heads * dim:
                raise ValueError(f"expected q and out [rows, n_heads, {kv.head_dim}]")
            start, length, pos0, table, stride, n = _items(q_start, q_len, kv_pos0, page_table)
            check(_abi.lib.nbl_attn_prefill(self.handle, kv.handle, _ptr(q), _dtype(q), rows, start, length, pos0, table,
                                            stride, n, heads, max_q_len, _ptr(out), _dtype(out)))
            return
        check(_abi.lib.nbl_attn_prefill(self.handle, kv.handle, _ptr(q), _dtype(q), q.shape[0], _ptr(q_start),
                                        _ptr(q_len), _ptr(kv_pos0), _ptr(page_table), page_table.shape[-1],
                                        q_start.shape[0], q.shape[1], max_q_len, _ptr(out), _dtype(out)))

    # ---- the 8-bit cache (kv_pool with dtype I8 or E4M3)
    def rotary_kv_append(self, kv: KVPool, q_in, k_in, v_in, q_out, q_start, q_len, kv_pos0, page_table, max_q_len: int,
                         rotary: RotarySpec, bq=None, bk=None, bv=None):
        """Fused bias -> rotary -> quantization -> page write of item i's q_len[i] tokens (rows q_start[i].. of q_in
        [rows, n_heads, D], k_in and v_in [rows, n_kv_heads, D]) at positions kv_pos0[i].. of page-table row i, and the
        rotated queries into q_out (see nbl_rotary_kv_append)."""
        p, keep = rotary._c()
        dtype = q_in.dtype
        if k_in.dtype is not dtype or v_in.dtype is not dtype:
            raise ValueError("q_in, k_in, v_in must share a dtype")
        n_rows, heads = _new_rows(kv, q_in, k_in, v_in, q_out)
        start, length, pos0, table, stride, n_items = _items(q_start, q_len, kv_pos0, page_table)
        if bq is not None:
            _check_bias(bq, heads, kv.head_dim)
        if bk is not None:
            _check_bias(bk, kv.n_kv_heads, kv.head_dim)
        if bv is not None:
            _check_bias(bv, kv.n_kv_heads, kv.head_dim)
        if rotary.freq_factors is not None and len(rotary.freq_factors) != (rotary.rotary_dim or kv.head_dim) // 2:
            raise ValueError("freq_factors must hold rotary_dim / 2 factors")
        check(_abi.lib.nbl_rotary_kv_append(
            self.handle, kv.handle, _ptr(q_in), _ptr(k_in), _ptr(v_in), _dtype(q_in), _ptr(bq), _ptr(bk), _ptr(bv),
            _ptr(q_out), _dtype(q_out), n_rows, start, length, pos0, table, stride, n_items, heads, max_q_len, C.byref(p)))

    def kv_read(self, kv: KVPool, start, length, kv_pos0, page_table, max_len: int, k_out=None, v_out=None):
        """Item i's positions kv_pos0[i].. as rows start[i].. of k_out / v_out [rows, n_kv_heads, D] (see nbl_kv_read)."""
        like = k_out if k_out is not None else v_out
        if like is None:
            raise ValueError("kv_read needs k_out or v_out")
        n_rows, size = like.shape[0], like.numel()
        if size != n_rows * kv.n_kv_heads * kv.head_dim or (
                like is not v_out and v_out is not None and (v_out.numel() != size or v_out.dtype is not like.dtype)):
            raise ValueError(f"expected k_out and v_out [rows, {kv.n_kv_heads}, {kv.head_dim}] of one size and dtype")
        first, n, pos0, table, stride, n_items = _items(start, length, kv_pos0, page_table)
        check(_abi.lib.nbl_kv_read(self.handle, kv.handle, n_rows, first, n, pos0, table, stride, n_items, max_len,
                                   _ptr(k_out), _ptr(v_out), _dtype(like)))

    def kv_import(self, kv: KVPool, page_ids, codes, scales):
        """codes [n, 2, n_kv_heads, 16, D] (int8 / float8_e4m3fn) and scales [n, 2, n_kv_heads] fp32 into pages page_ids."""
        _check_pages(kv, page_ids, codes, scales)
        check(_abi.lib.nbl_kv_import(self.handle, kv.handle, _ints(page_ids), page_ids.shape[0], _ptr(codes),
                                     _ptr(scales)))

    def kv_export(self, kv: KVPool, page_ids, codes, scales):
        """Pages page_ids into codes and scales, as kv_import takes them."""
        _check_pages(kv, page_ids, codes, scales)
        check(_abi.lib.nbl_kv_export(self.handle, kv.handle, _ints(page_ids), page_ids.shape[0], _ptr(codes),
                                     _ptr(scales)))

    # ---- page bookkeeping on the device (int32 CUDA tensors: page_table [rows, stride], seq_lens [rows],
    # ref_counts [n_pages])
    def kv_copy_pages(self, kv: KVPool, src_pages, dst_pages):
        n = src_pages.numel()
        if dst_pages.numel() != n:
            raise ValueError("src_pages and dst_pages must have one length")
        check(_abi.lib.nbl_kv_copy_pages(self.handle, kv.handle, _ints(src_pages), _ints(dst_pages), n))

    def kv_fork(self, kv: KVPool, page_table, seq_lens, ref_counts, src_rows, dst_rows):
        """Row dst_rows[i] becomes a branch of src_rows[i]: full pages shared, the part-filled one copied."""
        n_rows, stride, n = _book(kv, page_table, seq_lens, ref_counts, src_rows, dst_rows)
        check(_abi.lib.nbl_kv_fork(self.handle, kv.handle, _ints(page_table), stride, n_rows, _ints(seq_lens),
                                   _ints(ref_counts), _ints(src_rows), _ints(dst_rows), n))

    def kv_release(self, kv: KVPool, page_table, seq_lens, ref_counts, rows):
        n_rows, stride, n = _book(kv, page_table, seq_lens, ref_counts, rows, rows)
        check(_abi.lib.nbl_kv_release(self.handle, kv.handle, _ints(page_table), stride, n_rows, _ints(seq_lens),
                                      _ints(ref_counts), _ints(rows), n))

    def kv_extend(self, kv: KVPool, page_table, seq_lens, ref_counts, rows, new_lens):
        """Row rows[i] gets the pages that new_lens[i] tokens need, lowest free ids first, and that length."""
        n_rows, stride, n = _book(kv, page_table, seq_lens, ref_counts, rows, new_lens)
        check(_abi.lib.nbl_kv_extend(self.handle, kv.handle, _ints(page_table), stride, n_rows, _ints(seq_lens),
                                     _ints(ref_counts), _ints(rows), _ints(new_lens), n))

    def kv_compact(self, src: KVPool, dst: KVPool, page_table, seq_lens, table_out, ref_counts_out, n_used):
        """The rows' pages move from pool src into pool dst, numbered by first appearance; src stays as it is."""
        n_rows, stride = page_table.shape
        if table_out.shape != page_table.shape or ref_counts_out.numel() < dst.n_pages:
            raise ValueError("table_out must have page_table's shape and ref_counts_out one count per page of dst")
        if seq_lens.numel() < n_rows or n_used.numel() < 1:
            raise ValueError("expected seq_lens for every table row, and one element in n_used")
        check(_abi.lib.nbl_kv_compact(self.handle, src.handle, dst.handle, _ints(page_table), stride, n_rows,
                                      _ints(seq_lens), _ints(table_out), _ints(ref_counts_out), _ints(n_used)))

    def lse_merge_packed(self, packed, n_parts: int, rows: int, head_dim: int, out, lse=None):
        """packed [n_parts, rows * (head_dim + 1)] fp32 (per part: outputs then lse) -> out [rows, head_dim]."""
        check(_abi.lib.nbl_lse_merge_packed(self.handle, _ptr(packed), n_parts, rows, head_dim, _ptr(out), _ptr(lse)))

    def lse_merge(self, part_o, part_lse, out, lse=None):
        """part_o [P, rows, D], part_lse [P, rows] fp32 -> out [rows, D] (+ lse [rows])."""
        n_parts, rows, d = part_o.shape
        check(_abi.lib.nbl_lse_merge(self.handle, _ptr(part_o), _ptr(part_lse), n_parts, rows, d, _ptr(out),
                                     _ptr(lse)))
