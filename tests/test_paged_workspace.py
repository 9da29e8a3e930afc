"""The workspace of sparse paged attention: one buffer, sized for the largest step, serves every smaller one."""
import numpy as np
import pytest

GEOMETRIES = [(1, 1, 3, 8192), (4, 2, 16, 8192), (16, 2, 32, 32768), (8, 4, 64, 524288), (8, 8, 250, 128 * 260), (2, 3, 2000, 128 * 2100)]


@pytest.fixture(scope="module")
def ops():
    from nomos_nvfp4_b200 import build, ops
    build.build()
    return ops


def query(ops, rows, nkv, kvg, top, max_len):
    return ops.attn_paged_sparse_workspace_bytes(rows=rows, nh=nkv * kvg, nkv=nkv, kvg=kvg, l_hd=128, top_pages=top, max_len=max_len)


@pytest.mark.parametrize("nkv,kvg,top,max_len", GEOMETRIES)
def test_query_grows_with_the_rows(ops, nkv, kvg, top, max_len):
    last = 0
    for rows in [*range(1, 300), 511, 512, 513, 1000, 2048, 8191, 8192, 8193, 9000, 16384, 50000]:
        n = query(ops, rows, nkv, kvg, top, max_len)
        assert n >= last, (rows, n, last)
        last = n


@pytest.mark.gpu
@pytest.mark.parametrize("nkv,kvg,top,max_len", GEOMETRIES)
def test_smaller_steps_fit(ops, nkv, kvg, top, max_len):
    """A buffer for 512 rows and every kind of smaller step on it.  (All rows are padding: nothing is read or written but the lists.)"""
    import torch
    from tests._gpu import DEV, dev
    most, wsb = 512, query(ops, 512, nkv, kvg, top, max_len)
    ws = torch.empty(wsb, dtype=torch.uint8, device=DEV)
    pools = [torch.zeros((4, nkv, 128, 128), dtype=torch.int8, device=DEV) for _ in range(2)] + [torch.ones((4, nkv, 128), device=DEV) for _ in range(2)]
    pools += [torch.zeros((4, nkv, 2, 128), dtype=torch.int8, device=DEV), torch.ones((4, nkv), device=DEV)]
    q = torch.zeros((most, nkv * kvg, 128), device=DEV)
    out = torch.full_like(q, -31)
    pad = dev(np.full(most, -1, np.int32))
    table = torch.zeros((most, (max_len + 127) // 128), dtype=torch.int32, device=DEV)
    for rows in [*range(1, 66), 100, 147, 148, 149, 200, 255, 256, 257, 300, 400, 511, 512]:
        for batch in sorted({1, max(1, rows // 2), rows}):
            ops.attn_paged_sparse_i8(None, q, *pools, table, pad, pad, out, None, ws, wsb, rows=rows, batch=batch, nh=nkv * kvg, nkv=nkv, kvg=kvg, l_hd=128, n_pages=4,
                                     max_pages=table.shape[1], max_len=max_len, top_pages=top)
    torch.cuda.synchronize()
    assert bool((out == -31).all()) and ops.device_faults() == 0
