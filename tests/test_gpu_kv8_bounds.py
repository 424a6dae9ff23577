"""Calls on the 8-bit K/V cache that are at or past their bounds: what is out of them is flagged and left out, what is empty is
no work, what is large is not refused. Values are compared with the 64-bit forms and tolerances of test_gpu_kv8.py."""
import numpy as np
import pytest

from nibble_b200.workloads import make_page_tables
from test_gpu_kv8 import attend, dev, ints, np_of, random_pool, rows_of

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
