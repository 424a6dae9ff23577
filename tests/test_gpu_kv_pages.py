"""Page bookkeeping on the GPU (copy, fork, release, extend, compact) against a plain Python book: tables, lengths, counts
and page contents are whole numbers or copies, so everything has to be equal."""
import numpy as np
import pytest

from nibble_b200.workloads import make_page_tables

pytestmark = pytest.mark.gpu
PAGE = 16


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def ints(v):
    return dev(np.asarray(v, np.int32))


class Book:
    """A pool's page tables kept the plain way, on the host."""

    def __init__(self, table, lens, n_pages, pool):
        self.table, self.lens, self.pool = table.copy(), np.array(lens, np.int32), pool.copy()
        self.refs = np.zeros(n_pages, np.int32)
        for e in table[table >= 0]:
            self.refs[e] += 1

    def free(self):
        return [int(p) for p in np.nonzero(self.refs == 0)[0]]

    def release(self, row):
        for e in self.table[row][self.table[row] >= 0]:
            self.refs[e] -= 1
        self.table[row] = -1
        self.lens[row] = 0

    def fork(self, src, dst):
        for d in dst:
            self.release(d)
        for s, d in zip(src, dst):
            full = self.lens[s] // PAGE
            self.table[d, :full] = self.table[s, :full]
            for e in self.table[s, :full]:
                self.refs[e] += 1
            self.lens[d] = self.lens[s]
        free = self.free()
        for s, d in zip(src, dst):
            full = self.lens[s] // PAGE
            if self.lens[s] % PAGE:
                if not free:
                    self.lens[d] = full * PAGE
                    continue
                page = free.pop(0)
                self.table[d, full] = page
                self.refs[page] = 1
                self.pool[page] = self.pool[self.table[s, full]]

    def extend(self, rows, lens):
        free = self.free()
        need = [-(-n // PAGE) - -(-int(self.lens[r]) // PAGE) for r, n in zip(rows, lens)]
        if sum(need) > len(free):
            return
        for r, n, k in zip(rows, lens, need):
            at = -(-int(self.lens[r]) // PAGE)
            for j in range(k):
                page = free.pop(0)
                self.table[r, at + j] = page
                self.refs[page] = 1
            self.lens[r] = n


class Device:
    def __init__(self, ctx, kv, book):
        self.ctx, self.kv = ctx, kv
        self.table, self.lens, self.refs = dev(book.table), dev(book.lens), dev(book.refs)

    def args(self):
        return self.kv, self.table, self.lens, self.refs

    def same(self, book):
        assert np.array_equal(self.table.cpu().numpy(), book.table)
        assert np.array_equal(self.lens.cpu().numpy(), book.lens)
        assert np.array_equal(self.refs.cpu().numpy(), book.refs)
        assert np.array_equal(self.kv.tensor().cpu().numpy(), book.pool)


def setup(ctx, lens, KV=2, spare=20, stride=40, seed=1):
    import torch
    table, n_pages = make_page_tables(lens, shuffle_seed=seed, stride=stride)
    kv = ctx.kv_pool(n_pages + spare, KV)
    t = kv.tensor()
    t.copy_(torch.randint(-30000, 30000, t.shape, device="cuda", dtype=torch.int16))
    book = Book(table, lens, n_pages + spare, t.cpu().numpy())
    return Device(ctx, kv, book), book


@pytest.mark.parametrize("KV", [1, 2, 8])
def test_fork_release_extend_over_many_steps(nbl_ctx, KV):
    lens = [1, 15, 16, 17, 100, 320, 0, 33] + [0] * 12 + [40, 7]
    d, book = setup(nbl_ctx, lens, KV, spare=150)
    rng = np.random.default_rng(KV)
    for step in range(12):
        kind = step % 4
        if kind in (0, 2):
            rows = rng.permutation(len(lens))
            n = int(rng.integers(1, 9))
            dst, src = rows[:n], rng.choice(rows[n:], n)
            nbl_ctx.kv_fork(*d.args(), ints(src), ints(dst))
            book.fork(src, dst)
        elif kind == 1:
            rows = rng.permutation(len(lens))[:7]
            to = np.minimum(book.lens[rows] + rng.integers(0, 40, 7), 40 * PAGE)
            nbl_ctx.kv_extend(*d.args(), ints(rows), ints(to))
            book.extend(rows, to)
        else:
            rows = rng.permutation(len(lens))[:3]
            nbl_ctx.kv_release(*d.args(), ints(rows))
            for r in rows:
                book.release(r)
        nbl_ctx.check()
        d.same(book)
    d.kv.close()


def test_fork_many_from_one_and_again(nbl_ctx):
    """300 branches of one row, twice: the second time they replace themselves and get the same pages."""
    lens = [100] + [0] * 300
    d, book = setup(nbl_ctx, lens, 1, spare=310)
    for _ in range(2):
        nbl_ctx.kv_fork(*d.args(), ints([0] * 300), ints(np.arange(1, 301)))
        nbl_ctx.check()
        book.fork([0] * 300, np.arange(1, 301))
        d.same(book)
    d.kv.close()


def test_large_pool_finds_the_last_free_pages(nbl_ctx):
    """The only free pages are the last ones of a pool that takes many steps to search."""
    lens = [9000 * PAGE - 3, 0, 0]
    d, book = setup(nbl_ctx, lens, 1, spare=2, stride=9001, seed=None)
    nbl_ctx.kv_fork(*d.args(), ints([0, 0]), ints([2, 1]))
    nbl_ctx.check()
    book.fork([0, 0], [2, 1])
    d.same(book)
    d.kv.close()


def test_no_free_page(nbl_ctx):
    import nibble_b200 as nb
    d, book = setup(nbl_ctx, [20, 20, 0, 0, 0], 1, spare=2)
    nbl_ctx.kv_extend(*d.args(), ints([0, 1]), ints([50, 50]))  # 4 pages wanted, 2 free: none is given
    with pytest.raises(nb.NibbleError, match="no free page"):
        nbl_ctx.check()
    d.same(book)
    nbl_ctx.kv_fork(*d.args(), ints([0, 1, 0]), ints([4, 2, 3]))  # the third finds none: its full page only
    with pytest.raises(nb.NibbleError, match="no free page"):
        nbl_ctx.check()
    book.fork([0, 1, 0], [4, 2, 3])
    d.same(book)
    assert book.lens[3] == 16
    d.kv.close()


def test_bad_rows_are_skipped_and_flagged(nbl_ctx):
    import nibble_b200 as nb

    def flagged():
        with pytest.raises(nb.NibbleError) as e:
            nbl_ctx.check()
        assert e.value.status == 5

    d, book = setup(nbl_ctx, [20, 33, 0, 5], 1)
    nbl_ctx.kv_fork(*d.args(), ints([9, 0, 0, 1]), ints([2, -1, 3, 3]))  # bad source, bad destination, row 3 twice
    flagged()
    book.fork([0], [3])
    d.same(book)
    nbl_ctx.kv_fork(*d.args(), ints([0, 1]), ints([1, 2]))  # row 1 would be source and destination
    flagged()
    book.fork([1], [2])
    d.same(book)
    nbl_ctx.kv_release(*d.args(), ints([4]))
    flagged()
    nbl_ctx.kv_release(*d.args(), ints([2, 2]))  # twice the same: released once
    nbl_ctx.check()
    book.release(2)
    d.same(book)
    nbl_ctx.kv_extend(*d.args(), ints([0, 0, 1]), ints([40, 50, 30]))  # row 0 twice (the first counts), row 1 cannot shrink
    flagged()
    book.extend([0], [40])
    d.same(book)
    with pytest.raises(nb.NibbleError):
        nbl_ctx.kv_fork(*d.args(), ints([0] * 5), ints([0] * 5))  # more forks than rows
    d.kv.close()


@pytest.mark.parametrize("name", ["F16", "BF16", "I8", "E4M3"])
def test_copy_and_fork_every_pool_type(nbl_ctx, name):
    """Pages of the 8-bit pools move whole, scales included."""
    import torch
    import nibble_b200 as nb
    dtype = getattr(nb, name)
    eight = name in ("I8", "E4M3")
    kv = nbl_ctx.kv_pool(9, 3, 128 if eight else 64, dtype=dtype)
    if eight:
        codes = torch.randint(-100, 100, (9, 2, 3, PAGE, 128), device="cuda", dtype=torch.int8)
        scales = torch.rand((9, 2, 3), device="cuda")
        nbl_ctx.kv_import(kv, ints(np.arange(9)), codes, scales)
        if name == "E4M3":  # the byte -1 is a NaN there: stored as 0 and flagged
            with pytest.raises(nb.NibbleError, match="infinity or NaN"):
                nbl_ctx.check()
    else:
        kv.tensor().copy_(torch.randint(-30000, 30000, kv.tensor().shape, device="cuda", dtype=torch.int16))

    def content():
        if not eight:
            return [kv.tensor().clone()]
        c, s = torch.empty_like(codes), torch.empty_like(scales)
        nbl_ctx.kv_export(kv, ints(np.arange(9)), c, s)
        return [c, s]

    before = content()
    nbl_ctx.kv_copy_pages(kv, ints([0, 1, 0]), ints([5, 6, 8]))
    nbl_ctx.check()
    for x, y in zip(content(), before):
        y[[5, 6, 8]] = y[[0, 1, 0]].clone()
        assert torch.equal(x, y)
    table, lens, refs = ints([[2, 3, -1], [-1, -1, -1]]), ints([20, 0]), ints([1, 1, 1, 1, 0, 1, 1, 1, 1])
    nbl_ctx.kv_fork(kv, table, lens, refs, ints([0]), ints([1]))
    nbl_ctx.check()
    assert table.tolist() == [[2, 3, -1], [2, 4, -1]] and refs.tolist() == [1, 1, 2, 1, 1, 1, 1, 1, 1]
    for x, y in zip(content(), before):
        y[4] = y[3].clone()
        assert torch.equal(x, y)
    kv.close()


@pytest.mark.parametrize("name", ["F16", "I8"])
def test_compact(nbl_ctx, name):
    import torch
    import nibble_b200 as nb
    lens = [40, 0, 100, 33, 16, 1]
    table, n_pages = make_page_tables(lens, shuffle_seed=3, stride=9)
    table[3, :2] = table[0, :2]  # shared pages
    table[4, 0] = table[2, 4]
    table[1, 0] = 5  # past row 1's length: not held
    dtype = getattr(nb, name)
    kv, to = nbl_ctx.kv_pool(n_pages, 2, dtype=dtype), nbl_ctx.kv_pool(n_pages + 3, 2, dtype=dtype)
    if name == "I8":
        codes = torch.randint(-100, 100, (n_pages, 2, 2, PAGE, 64), device="cuda", dtype=torch.int8)
        scales = torch.rand((n_pages, 2, 2), device="cuda")
        nbl_ctx.kv_import(kv, ints(np.arange(n_pages)), codes, scales)
    else:
        kv.tensor().copy_(torch.randint(-30000, 30000, kv.tensor().shape, device="cuda", dtype=torch.int16))
    out, refs, used = ints(np.full(table.shape, 77)), ints(np.full(n_pages + 3, 9)), ints([0])
    nbl_ctx.kv_compact(kv, to, dev(table), ints(lens), out, refs, used)
    nbl_ctx.check()
    order, want = [], np.full(table.shape, -1)
    for r, n in enumerate(lens):
        for j in range(-(-n // PAGE)):
            e = int(table[r, j])
            if e not in order:
                order.append(e)
            want[r, j] = order.index(e)
    assert used.item() == len(order)
    assert np.array_equal(out.cpu().numpy(), want)
    assert np.array_equal(refs.cpu().numpy(), np.bincount(want[want >= 0], minlength=n_pages + 3))
    if name == "I8":
        c, s = torch.empty_like(codes[:len(order)]), torch.empty_like(scales[:len(order)])
        nbl_ctx.kv_export(to, ints(np.arange(len(order))), c, s)
        assert torch.equal(c, codes[order]) and torch.equal(s, scales[order])
    else:
        assert torch.equal(to.tensor()[:len(order)], kv.tensor()[order])
    # a pool that is too small: what fits, and a flag
    small = nbl_ctx.kv_pool(4, 2, dtype=dtype)
    nbl_ctx.kv_compact(kv, small, dev(table), ints(lens), out, refs, used)
    with pytest.raises(nb.NibbleError, match="no free page"):
        nbl_ctx.check()
    assert np.array_equal(out.cpu().numpy(), np.where(want >= 4, -1, want)) and used.item() == len(order)
    with pytest.raises(nb.NibbleError):
        nbl_ctx.kv_compact(kv, kv, dev(table), ints(lens), out, refs, used)
    for p in (kv, to, small):
        p.close()


def test_a_view_outlives_its_closed_pool(nbl_ctx):
    import torch
    kv = nbl_ctx.kv_pool(4, 2)
    view = kv.tensor()
    view.fill_(7)
    kv.close()
    assert torch.equal(view, torch.full_like(view, 7))
    del view
    nbl_ctx.check()
