"""Sizes near 2^31 whose loops would step past the largest 32-bit index: refused before anything is launched."""
import pytest

P = 0x1000                               # never dereferenced: validation fails first


@pytest.fixture(scope="module")
def ops():
    from nomos_nvfp4_b200 import build, ops
    build.build()
    return ops


def refused(ops, call, *args, **kw):
    with pytest.raises(ops.NomosError) as e:
        call(*args, **kw)
    assert e.value.status == -1, str(e.value)


@pytest.mark.parametrize("bad", [dict(vocab=(1 << 30) + 1), dict(vocab=(1 << 31) - 1), dict(max_draft=(1 << 30) + 1), dict(max_draft=(1 << 31) - 2)])
def test_verify_sizes(ops, bad):
    kw = dict(batch=1, max_draft=3, vocab=100, p_stride=1 << 31, q_stride=1 << 31)
    refused(ops, ops.spec_verify, 0, *[P] * 10, **{**kw, **bad})


def test_sparse_rows(ops):
    kw = dict(batch=2, nh=8, nkv=4, kvg=2, l_hd=128, n_pages=64, max_pages=16, max_len=2000, top_pages=4)
    for rows in ((1 << 30) + 1, (1 << 31) - 1):
        refused(ops, ops.attn_paged_sparse_i8, 0, *[P] * 13, 1 << 60, rows=rows, **kw)
