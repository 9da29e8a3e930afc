"""Refusals of the paged serving operators (no launch), and their plain restatements on cases worked out by hand."""
import numpy as np
import pytest

from tests import _paged_ref as ref

P = 0x1000                               # never dereferenced: validation fails first


@pytest.fixture(scope="module")
def ops():
    from nomos_nvfp4_b200 import build, ops
    build.build()
    return ops


@pytest.mark.parametrize("name,mirror", [("nomos_kv_plan", "KvPlan"), ("nomos_kv_rows", "KvRows"), ("nomos_attn_sparse", "AttnSparse"),
                                         ("nomos_attn_verify", "AttnVerify")])
def test_argument_blocks_match_the_header(ops, name, mirror):
    import ctypes
    import re
    from pathlib import Path
    from nomos_nvfp4_b200 import _lib
    text = (Path(__file__).resolve().parent.parent / "include" / "nomos_attn.h").read_text()
    body = re.search(r"typedef struct %s \{(.*?)\} %s_t;" % (name, name), text, flags=re.S).group(1)
    declared = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        kind, names = decl.split(None, 1)
        declared += [(n.strip(), kind) for n in names.split(",")]
    block = getattr(_lib, mirror)
    kinds = {ctypes.c_uint64: "uint64_t", ctypes.c_int64: "int64_t", ctypes.c_double: "double"}
    assert declared == [(n, kinds[t]) for n, t in block._fields_]
    assert _lib.packer(block).size == ctypes.sizeof(block) == 8 * len(declared)
    fn = {"KvPlan": "nomos_kv_paged_plan", "KvRows": "nomos_kv_paged_append_rows_i8", "AttnSparse": "nomos_attn_paged_sparse_i8",
          "AttnVerify": "nomos_attn_spec_verify"}[mirror]
    assert getattr(_lib.lib(), fn)(None, bytes(8 * len(declared))) == -1      # struct_bytes of another version
    assert getattr(_lib.lib(), fn)(None, None) == -1


def refused(ops, status, call, *args, **kw):
    with pytest.raises(ops.NomosError) as e:
        call(*args, **kw)
    assert e.value.status == status, str(e.value)


def test_plan_refusals(ops):
    kw = dict(batch=2, max_pages=4, n_pages=8, max_rows=16)
    for i in range(13):
        refused(ops, -1, ops.kv_paged_plan, 0, *[None if j == i else P for j in range(13)], **kw)
        refused(ops, -1, ops.kv_paged_plan, 0, *[P + 2 if j == i else P for j in range(13)], **kw)
    for bad in (dict(max_pages=0), dict(n_pages=0), dict(max_rows=-1), dict(max_pages=1 << 24), dict(n_pages=1 << 24), dict(batch=1 << 32),
                dict(max_rows=1 << 31), dict(max_rows=(1 << 30) + 1)):
        refused(ops, -1, ops.kv_paged_plan, 0, *[P] * 13, **{**kw, **bad})
    refused(ops, -2, ops.kv_paged_plan, 0, *[P] * 13, **{**kw, "batch": 8193})
    ops.kv_paged_plan(0, *[None] * 13, **{**kw, "batch": 0})


def test_append_rows_refusals(ops):
    kw = dict(n_rows=4, nkv=2, l_hd=128, l_kvd=256, n_pages=8)
    for i in range(9):
        args = [None if j == i else P for j in range(9)]
        refused(ops, -1, ops.kv_paged_append_rows_i8, 0, *args, **kw)      # (one bounds pool alone included)
        refused(ops, -1, ops.kv_paged_append_rows_i8, 0, *[P + 1 if j == i else P for j in range(9)], **kw)
    for bad in (dict(nkv=0), dict(n_pages=0), dict(l_kvd=255), dict(src_type=2), dict(n_pages=1 << 24)):
        refused(ops, -1, ops.kv_paged_append_rows_i8, 0, *[P] * 9, **{**kw, **bad})
    for bad in (dict(l_hd=256, l_kvd=512), dict(l_hd=64)):
        refused(ops, -2, ops.kv_paged_append_rows_i8, 0, *[P] * 9, **{**kw, **bad})
    ops.kv_paged_append_rows_i8(0, *[None] * 9, **{**kw, "n_rows": 0})


def test_page_bounds_refusals(ops):
    kw = dict(n=4, nkv=2, l_hd=128, n_pages=8)
    for i in range(5):
        refused(ops, -1, ops.kv_paged_page_bounds_i8, 0, *[None if j == i else P for j in range(5)], **kw)
    refused(ops, -2, ops.kv_paged_page_bounds_i8, 0, *[P] * 5, **{**kw, "l_hd": 256})
    ops.kv_paged_page_bounds_i8(0, *[None] * 5, **{**kw, "n": 0})


def test_sparse_refusals(ops):
    kw = dict(rows=3, batch=2, nh=8, nkv=4, kvg=2, l_hd=128, n_pages=64, max_pages=16, max_len=2000, top_pages=4, sink_pages=1,
              local_pages=2, softmax_scale=0.1)
    n = ops.attn_paged_sparse_workspace_bytes(rows=3, nh=8, nkv=4, kvg=2, l_hd=128, top_pages=4, max_len=2000)
    assert n > 0
    good = [P] * 13 + [n]
    for i in range(13):
        if i != 11:                                                    # sel_pages is optional
            refused(ops, -1, ops.attn_paged_sparse_i8, 0, *[None if j == i else x for j, x in enumerate(good)], **kw)
        refused(ops, -1, ops.attn_paged_sparse_i8, 0, *[P + 2 if j == i else x for j, x in enumerate(good)], **kw)
    for bad in (dict(kvg=3), dict(max_len=16 * 128 + 1), dict(local_pages=0), dict(sink_pages=-1), dict(sink_pages=3), dict(top_pages=2),
                dict(softmax_scale=0.0), dict(softmax_scale=-1.0), dict(softmax_scale=float("nan")), dict(softmax_scale=float("inf")),
                dict(q_type=2), dict(out_type=-1), dict(n_pages=0), dict(top_pages=0, sink_pages=0), dict(rows=1 << 40), dict(max_pages=1 << 33)):
        refused(ops, -1, ops.attn_paged_sparse_i8, 0, *good, **{**kw, **bad})
    for bad in (dict(l_hd=256), dict(nh=36, kvg=9)):
        refused(ops, -2, ops.attn_paged_sparse_i8, 0, *good, **{**kw, **bad})
    refused(ops, -2, ops.attn_paged_sparse_i8, 0, *good, **{**kw, "max_pages": 50000, "max_len": 50000 * 128})
    refused(ops, -3, ops.attn_paged_sparse_i8, 0, *good[:13], n - 1, **kw)
    for none in (dict(rows=0), dict(batch=0), dict(nh=0), dict(max_len=0)):
        ops.attn_paged_sparse_i8(0, *[None] * 13, 0, **{**kw, **none})
    assert ops.attn_paged_sparse_workspace_bytes(rows=0, nh=8, nkv=4, kvg=2, l_hd=128, top_pages=4, max_len=2000) == 0
    refused(ops, -1, ops.attn_paged_sparse_workspace_bytes, rows=3, nh=8, nkv=4, kvg=2, l_hd=128, top_pages=0, max_len=2000)


def test_verify_refusals(ops):
    kw = dict(batch=2, max_draft=3, vocab=100, p_stride=100, q_stride=100)
    optional = {1, 3}                                                  # draft_probs, n_draft
    for i in range(10):
        if i not in optional:                                          # (lengths: one of the two alone is refused)
            refused(ops, -1, ops.spec_verify, 0, *[None if j == i else P for j in range(10)], **kw)
        refused(ops, -1, ops.spec_verify, 0, *[P + 2 if j == i else P for j in range(10)], **kw)
    for bad in (dict(vocab=0), dict(max_draft=-1), dict(p_stride=99), dict(q_stride=99), dict(batch=1 << 31), dict(vocab=1 << 32, p_stride=1 << 33, q_stride=1 << 33)):
        refused(ops, -1, ops.spec_verify, 0, *[P] * 10, **{**kw, **bad})
    ops.spec_verify(0, *[None] * 10, **{**kw, "batch": 0})


def test_plan_by_hand():
    """Three requests over a stack [5, 6, 7]: one more row in a held page, 130 rows from nothing, one finished."""
    table = np.array([[3, -1, -1], [-1, -1, -1], [8, 9, -1]], np.int32)
    free = np.array([5, 6, 7, -1, -1, -1], np.int32)
    got = ref.plan(np.array([10, 0, 200]), np.array([1, 130, -1]), np.array([1, 0, 2]), free, 3, table, 140)
    assert got["table"][1].tolist() == [9, 8, -1] and got["free"].tolist() == [5, 6, 7, 8, 9, -1]     # the released pages lie on top
    assert got["held_out"].tolist() == [1, 2, 0] and got["free_count_out"] == 3 and got["granted"].tolist() == [1, 130, 0]
    assert got["row_start"].tolist() == [0, 1, 131, 131]
    assert got["slot_map"][0] == 3 * 128 + 10 and got["slot_map"][1] == 9 * 128 and got["slot_map"][129] == 8 * 128
    assert got["row_pos"][130] == 129 and got["row_seq"][131:].tolist() == [-1] * 9


def test_bounds_bound_every_key():
    rng = np.random.default_rng(0)
    codes, scales = ref.codec(rng.standard_normal((3, 2, 128, 128)).astype(np.float32) * np.exp(rng.standard_normal((3, 2, 128, 1))))
    kb, t = ref.bounds(codes, scales)
    v = codes.astype(np.float64) * scales[..., None]
    tt = t[..., None, None].astype(np.float64) * (1 + 2.0 ** -23)                # the rounding of t's division and of hi / t
    assert (v <= (kb[..., 0, :][..., None, :] * tt + 1e-6 * tt)).all() and (v >= (kb[..., 1, :][..., None, :] * tt - 1e-6 * tt)).all()


def test_verify_by_hand():
    p = np.zeros((1, 3, 4), np.float32)
    q = np.zeros((1, 2, 4), np.float32)
    p[0] = [[0.5, 0.5, 0, 0], [0.25, 0.25, 0.5, 0], [0, 0, 0, 1]]
    q[0] = [[1, 0, 0, 0], [1, 0, 0, 0]]
    t = np.array([[0, 0]])
    # u q < p: 0.49 * 1 < 0.5 accepted; 0.25 * 1 < 0.25 not: residual [0, .25, .5, 0] of 0.75; 0.4 * 0.75 = 0.3 lies in token 2
    assert ref.verify(p, q, t, None, np.array([[0.49, 0.25]]), np.array([0.4])) == [(1, [0, 2, -1])]
    assert ref.verify(p, q, t, None, np.array([[0.49, 0.24]]), np.array([0.0])) == [(2, [0, 0, 3])]
    assert ref.verify(p, q, t, np.array([0]), np.array([[0.49, 0.24]]), np.array([0.75])) == [(0, [1, -1, -1])]
    assert ref.verify(p, q, t, np.array([-1]), np.array([[0.49, 0.24]]), np.array([0.75])) == [None]
