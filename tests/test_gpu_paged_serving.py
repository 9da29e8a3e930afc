"""Paged serving operators on the GPU, through the C ABI, against the plain restatements of tests/_paged_ref.py: the step plan
(block tables, slot maps), the slot-mapped append with page bounds, sparse attention over selected pages, speculative
verification, and a serving loop of all four.

Everything that is a whole number (tables, slots, codes, selections, tokens) has to be equal.  Attention outputs are held to
the library's bar, 2e-3 x RMS of exact 64-bit attention over the same selection: the kernel rounds the query to 16-bit fixed
point (half a step of amax / 32639 per element: at head_dim 128 and unit keys a logit is off by some 1e-4 at most) and the
softmax weights to 2^-17 of their tile's largest, each an order of magnitude below the bar; a bf16 output adds 2^-8 of the
value."""
import numpy as np
import pytest
import torch

from nomos_nvfp4_b200 import ops
from tests import _paged_ref as ref
from tests._cases import bf16_normal
from tests._gpu import DEV, dev, host

pytestmark = pytest.mark.gpu
PAGE, HD = 128, 128


def i32(x):
    return dev(np.ascontiguousarray(x, np.int32))


# ------------------------------------------------------------------------------------------------ plan

def plan_case(rng, batch, max_pages, rows_each, finished, tight):
    n_new = rng.integers(0, 2 * rows_each + 1, batch).astype(np.int32)
    lens = rng.integers(0, max_pages * PAGE + 1, batch).astype(np.int32)
    lens = np.where(rng.random(batch) < 0.9, np.maximum(0, np.minimum(lens, max_pages * PAGE - n_new)), lens).astype(np.int32)
    held = np.minimum(max_pages, -(-lens // PAGE) + (rng.random(batch) < 0.2)).astype(np.int32)
    n_new[rng.permutation(batch)[:finished]] = -rng.integers(1, 5)
    n_pages = batch * max_pages + 3
    ids = rng.permutation(n_pages).astype(np.int32)
    table = np.full((batch, max_pages), -1, np.int32)
    used = 0
    for b in range(batch):
        table[b, :held[b]] = ids[used:used + held[b]]
        used += held[b]
    free = np.full(n_pages, -1, np.int32)
    count = n_pages - used
    if tight:
        count = min(count, max(0, batch * rows_each // (3 * PAGE)))
    free[:count] = ids[used:used + count]
    return lens, n_new, held, free, count, table


def run_plan(lens, n_new, held, free, count, table, max_rows, *, alias=False, offset=0, stream=None):
    batch, max_pages = table.shape
    d = {"lens": i32(lens), "n_new": i32(n_new), "held": i32(held), "free": i32(free), "count": i32([count]), "table": i32(table)}
    d["held_out"] = d["held"] if alias else torch.full((batch,), -7, dtype=torch.int32, device=DEV)
    d["free_count_out"] = d["count"] if alias else torch.full((1,), -7, dtype=torch.int32, device=DEV)
    d["granted"] = torch.full((batch,), -7, dtype=torch.int32, device=DEV)
    d["row_start"] = torch.full((batch + 1,), -7, dtype=torch.int32, device=DEV)
    for n in ("slot_map", "row_seq", "row_pos"):                       # with a border that has to stay as it is
        d[n + "_all"] = torch.full((max_rows + offset + 5,), -9, dtype=torch.int32, device=DEV)
        d[n] = d[n + "_all"][offset:offset + max_rows]
    ops.kv_paged_plan(stream, d["lens"], d["n_new"], d["held"], d["free"], d["count"], d["table"], d["held_out"], d["free_count_out"], d["granted"],
                      d["row_start"], d["slot_map"], d["row_seq"], d["row_pos"], batch=batch, max_pages=max_pages, n_pages=len(free), max_rows=max_rows)
    torch.cuda.synchronize()
    for n in ("slot_map", "row_seq", "row_pos"):
        a = host(d[n + "_all"])
        assert (a[:offset] == -9).all() and (a[offset + max_rows:] == -9).all(), "written outside the rows"
    assert np.array_equal(host(d["lens"]), lens) and np.array_equal(host(d["n_new"]), n_new)
    return d


def same_plan(d, want):
    for n in ("table", "free", "held_out", "granted", "row_start", "slot_map", "row_seq", "row_pos"):
        assert np.array_equal(host(d[n]), want[n]), n
    assert int(host(d["free_count_out"])[0]) == want["free_count_out"]


# (2440 before the larger ones: the first call whose shared memory needs the kernel's attribute is one of those just above 48 KB)
@pytest.mark.parametrize("batch,max_pages,rows_each,finished,tight,extra", [
    (1, 1, 1, 0, False, 0), (1, 3, 200, 0, False, 9), (1, 3, 200, 1, False, 2), (7, 4, 1, 2, False, 0), (33, 9, 60, 5, True, 31),
    (64, 32, 1, 0, False, 3), (100, 5, 130, 30, True, 1), (1000, 6, 9, 100, False, 0), (1025, 3, 40, 1, True, 7), (2050, 2, 1, 9, False, 0), (2440, 2, 1, 0, False, 5), (2457, 1, 2, 0, True, 0), (2500, 2, 3, 2500, False, 50),
    (5000, 4, 20, 77, True, 1), (8192, 2, 1, 0, False, 0), (40, 70, 1200, 3, False, 13), (40, 70, 1200, 3, True, -9000)])
@pytest.mark.parametrize("alias,offset", [(False, 0), (True, 1)])
def test_plan(batch, max_pages, rows_each, finished, tight, extra, alias, offset):
    rng = np.random.default_rng(batch * 31 + max_pages + offset)
    case = plan_case(rng, batch, max_pages, rows_each, finished, tight)
    max_rows = max(0, int(np.maximum(case[1], 0).sum()) + extra)       # a negative `extra`: the last requests' rows do not fit
    d = run_plan(*case, max_rows, alias=alias, offset=offset)
    same_plan(d, ref.plan(*case, max_rows))


def test_plan_without_rows_and_with_an_empty_pool():
    table = np.full((3, 4), -1, np.int32)
    args = (np.array([0, 5, 9]), np.array([0, 0, -1]), np.array([0, 1, 1]), np.full(8, 3, np.int32), 0, table)
    same_plan(run_plan(*args, 0), ref.plan(*args, 0))
    args = (np.array([0, 0, 100]), np.array([4, 1, 2]), np.array([0, 1, 1]), np.full(8, 3, np.int32), 0, table)
    want = ref.plan(*args, 9)
    assert want["granted"].tolist() == [0, 1, 2]                       # who lacks no page is served all the same
    same_plan(run_plan(*args, 9), want)


def test_plan_steps_in_place_hand_every_page_out_once():
    """Many steps in place, some plans dropped: no page is ever in two hands, none is lost."""
    rng = np.random.default_rng(11)
    batch, max_pages, n_pages = 24, 6, 80
    lens = np.zeros(batch, np.int32)
    held = i32(np.zeros(batch)); count = i32([n_pages]); free = i32(rng.permutation(n_pages)); table = i32(np.full((batch, max_pages), -1))
    other_held, other_count = torch.empty_like(held), torch.empty_like(count)
    granted = torch.empty_like(held); start = i32(np.zeros(batch + 1))
    max_rows = 1000
    rows = [torch.empty(max_rows, dtype=torch.int32, device=DEV) for _ in range(3)]
    for step in range(60):
        n_new = np.where(rng.random(batch) < 0.15, -1, rng.integers(0, 60, batch)).astype(np.int32)
        dropped = step % 5 == 4
        ops.kv_paged_plan(None, i32(lens), i32(n_new), held, free, count, table, other_held if dropped else held, other_count if dropped else count, granted, start,
                          *rows, batch=batch, max_pages=max_pages, n_pages=n_pages, max_rows=max_rows)
        torch.cuda.synchronize()
        if not dropped:
            g = host(granted)
            lens = np.where(n_new < 0, 0, lens + np.maximum(0, g - rng.integers(0, 3, batch))).astype(np.int32)   # some rows rejected
        h, t = host(held), host(table)
        mine = [int(x) for b in range(batch) for x in t[b, :h[b]]] + host(free)[: int(host(count)[0])].tolist()
        assert sorted(mine) == list(range(n_pages)), step
        assert (h * PAGE >= lens).all()


# ------------------------------------------------------------------------------------------------ append, page bounds

def empty_pools(n_pages, nkv, fill=0):
    k, v = (torch.full((n_pages, nkv, PAGE, HD), fill, dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.full((n_pages, nkv, PAGE), 2.0, device=DEV) for _ in range(2))
    return k, v, ks, vs, torch.full((n_pages, nkv, 2, HD), 99, dtype=torch.int8, device=DEV), torch.full((n_pages, nkv), 77.0, device=DEV)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("nkv,gap,shift", [(1, 0, 0), (4, 0, 0), (3, 5, 0), (2, 4, 1), (16, 8, 4)])
def test_append_rows(dtype, nkv, gap, shift):
    """Rows behind strides and offsets of their own, padding, slots outside the pool, two pages completed, one nearly."""
    rng = np.random.default_rng(nkv + gap + shift)
    n_pages = 7
    slots = np.concatenate([3 * PAGE + np.arange(100, 128), [-1, n_pages * PAGE, 2 ** 31 - 1, -(2 ** 31)], 5 * PAGE + np.arange(0, 127),
                            PAGE * 1 + np.arange(128)[::-1], [0]]).astype(np.int64)
    n = len(slots)
    width = nkv * HD + gap
    flat = {s: torch.from_numpy(rng.standard_normal(n * width + shift, dtype=np.float32) * 3).to(DEV) for s in "kv"}
    flat = {s: x.to(torch.bfloat16) if dtype == "bf16" else x for s, x in flat.items()}
    src = {s: x[shift:] for s, x in flat.items()}
    rows = {s: x[shift:].float().cpu().numpy().reshape(n, width)[:, :nkv * HD].reshape(n, nkv, HD) for s, x in flat.items()}
    k, v, ks, vs, kb, kbs = empty_pools(n_pages, nkv, 5)
    ops.kv_paged_append_rows_i8(None, src["k"], src["v"], k, v, ks, vs, kb, kbs, i32(slots.astype(np.int32)), n_rows=n, nkv=nkv, l_hd=HD, l_kvd=width,
                                n_pages=n_pages, src_type=ops.BF16 if dtype == "bf16" else ops.F32)
    torch.cuda.synchronize()
    for s, pool, scales in (("k", k, ks), ("v", v, vs)):
        want, want_s = np.full((n_pages, nkv, PAGE, HD), 5, np.int8), np.full((n_pages, nkv, PAGE), 2, np.float32)
        code, sc = ref.codec(rows[s])
        for r, at in enumerate(slots):
            if 0 <= at < n_pages * PAGE:
                want[at // PAGE, :, at % PAGE], want_s[at // PAGE, :, at % PAGE] = code[r], sc[r]
        assert np.array_equal(host(pool), want) and np.array_equal(host(scales), want_s)
    wkb, wkbs = ref.bounds(host(k), host(ks))
    done = [1, 3]
    assert np.array_equal(host(kb)[done], wkb[done]) and np.array_equal(host(kbs)[done], wkbs[done])
    rest = [0, 2, 4, 5, 6]
    assert (host(kb)[rest] == 99).all() and (host(kbs)[rest] == 77).all(), "bounds of pages that are not complete"


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("nkv,rows,gap,shift", [(1, 1, 0, 0), (2, 256, 8, 0), (17, 128, 0, 0), (16, 129, 0, 0), (40, 64, 3, 1), (5, 257, 0, 0), (33, 700, 0, 2), (8, 3000, 16, 0), (16, 2500, 0, 0)])
def test_append_rows_up_to_page_ends(dtype, nkv, rows, gap, shift):
    """Few rows (one launch, a block per head) and many (two launches), head counts on both sides of a block's sixteen, pages completed over
    two calls, and untouched elsewhere."""
    rng = np.random.default_rng(nkv * 7 + rows)
    n_pages = rows // PAGE + 5
    pages = rng.permutation(n_pages)
    base = 100                                                         # the first call leaves pages at 100, 228, ... of the sequence
    pos = np.concatenate([np.arange(base), base + np.arange(rows)])
    slots = pages[pos // PAGE] * PAGE + pos % PAGE
    width = nkv * HD + gap
    pools = empty_pools(n_pages, nkv, 3)
    codes, scales = np.full((n_pages, nkv, PAGE, HD), 3, np.int8), np.full((n_pages, nkv, PAGE), 2, np.float32)
    done = set()
    for part in (slice(0, base), slice(base, base + rows)):
        n = len(pos[part])
        flat = torch.from_numpy(rng.standard_normal(n * width + shift, dtype=np.float32)).to(DEV)
        flat = flat.to(torch.bfloat16) if dtype == "bf16" else flat
        x = flat[shift:].float().cpu().numpy().reshape(n, width)[:, :nkv * HD].reshape(n, nkv, HD)
        ops.kv_paged_append_rows_i8(None, flat[shift:], flat[shift:], *pools, i32(slots[part]), n_rows=n, nkv=nkv, l_hd=HD, l_kvd=width, n_pages=n_pages,
                                    src_type=ops.BF16 if dtype == "bf16" else ops.F32)
        torch.cuda.synchronize()
        c, s = ref.codec(x)
        codes[slots[part] // PAGE, :, slots[part] % PAGE], scales[slots[part] // PAGE, :, slots[part] % PAGE] = c, s
        done |= {int(p) // PAGE for p in slots[part] if p % PAGE == PAGE - 1}
        for i in (0, 1):
            assert np.array_equal(host(pools[i]), codes) and np.array_equal(host(pools[2 + i]), scales)
        kb, kbs = ref.bounds(codes, scales)
        for p in range(n_pages):
            if p in done:
                assert np.array_equal(host(pools[4])[p], kb[p]) and np.array_equal(host(pools[5])[p], kbs[p]), p
            else:
                assert (host(pools[4])[p] == 99).all() and (host(pools[5])[p] == 77).all(), p


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("rows", [100, 1500])
def test_append_rows_back_to_back(rows, captured):
    """Sources rewritten right before every append and pools read right after it, nothing waited for: no call sees another one's rows."""
    rng = np.random.default_rng(rows)
    nkv, n_pages, rounds = 8, rows // PAGE + 3, 12
    slots = i32(100 + np.arange(rows))
    data = torch.from_numpy(rng.standard_normal((rounds, 2, rows, nkv, HD), dtype=np.float32)).to(DEV).to(torch.bfloat16)
    src = torch.zeros_like(data[0])
    pools = empty_pools(n_pages, nkv)
    got = [[torch.empty_like(x) for x in pools] for _ in range(rounds)]

    def step(i):
        src.copy_(data[i])
        ops.kv_paged_append_rows_i8(None, src[0], src[1], *pools, slots, n_rows=rows, nkv=nkv, l_hd=HD, l_kvd=nkv * HD, n_pages=n_pages, src_type=ops.BF16)
        for x, y in zip(got[i], pools):
            x.copy_(y)

    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for i in range(rounds):
                step(i)
        for _ in range(2):
            graph.replay()
    else:
        for i in range(rounds):
            step(i)
    torch.cuda.synchronize()
    at = 100 + np.arange(rows)
    for i in range(rounds):
        for j in range(2):
            code, scale = ref.codec(data[i, j].float().cpu().numpy())
            assert np.array_equal(host(got[i][j])[at // PAGE, :, at % PAGE], code) and np.array_equal(host(got[i][2 + j])[at // PAGE, :, at % PAGE], scale), (i, j)
        done = range(0, (100 + rows) // PAGE)
        kb, kbs = ref.bounds(host(got[i][0]), host(got[i][2]))
        for p in done:
            assert np.array_equal(host(got[i][4])[p], kb[p]) and np.array_equal(host(got[i][5])[p], kbs[p]), (i, p)


def test_append_rows_is_the_one_row_append():
    """The same codes and scales as the decode append, rows with infinities, NaN, zeros and denormals among them; no bounds asked for."""
    rng = np.random.default_rng(3)
    nkv, batch, n_pages = 2, 8, 4
    x = rng.standard_normal((batch, nkv, HD), dtype=np.float32)
    x[0] = 0; x[1, 0, 5] = np.inf; x[2, 1, 7] = np.nan; x[3] *= 1e-42; x[4] *= 1e37; x[5, 0] = np.nan; x[6, :, ::2] = -np.inf
    pos = np.array([0, 127, 128, 200, 255, 256, 400, 511], np.int32)
    table = np.tile(np.array([2, 0, 3, 1], np.int32), (batch, 1))
    a, b = empty_pools(n_pages, nkv), empty_pools(n_pages, nkv)
    ops.kv_paged_append_quant_i8(None, dev(x), dev(x), *a[:4], i32(table), i32(pos), batch=batch, nkv=nkv, l_hd=HD, l_kvd=nkv * HD, max_pages=4)
    slots = table[0, pos // PAGE] * PAGE + pos % PAGE
    ops.kv_paged_append_rows_i8(None, dev(x), dev(x), *b[:4], None, None, i32(slots), n_rows=batch, nkv=nkv, l_hd=HD, l_kvd=nkv * HD, n_pages=n_pages)
    torch.cuda.synchronize()
    for p, q in zip(a[:4], b[:4]):
        assert np.array_equal(host(p).view(np.uint8), host(q).view(np.uint8))


def test_page_bounds_of_listed_pages():
    rng = np.random.default_rng(4)
    nkv, n_pages = 3, 9
    code, sc = ref.codec(rng.standard_normal((n_pages, nkv, PAGE, HD)) * np.exp(2 * rng.standard_normal((n_pages, nkv, 1, HD))))
    sc[1] *= 1e-44; sc[2, 0, 5] = np.inf; sc[2, 1, 9] = np.nan; sc[3] = 3e38; code[4] = 0; sc[5] *= -1
    pages = np.array([8, 1, -1, 2, n_pages, 3, 4, 5, 2 ** 31 - 1], np.int32)
    k, _, ks, _, kb, kbs = empty_pools(n_pages, nkv)
    k.copy_(dev(code)); ks.copy_(dev(sc))
    ops.kv_paged_page_bounds_i8(None, k, ks, kb, kbs, i32(pages), n=len(pages), nkv=nkv, l_hd=HD, n_pages=n_pages)
    torch.cuda.synchronize()
    want, want_s = ref.bounds(code, sc)
    for p in range(n_pages):
        if p in (8, 1, 2, 3, 4, 5):
            assert np.array_equal(host(kb)[p], want[p]) and np.array_equal(host(kbs)[p], want_s[p]), p
        else:
            assert (host(kb)[p] == 99).all() and (host(kbs)[p] == 77).all()


# ------------------------------------------------------------------------------------------------ sparse attention

class Pools:
    """Quantised pages in any order, their bounds, and the block tables of sequences of given lengths."""

    def __init__(self, rng, lens, nkv, n_pages=None, extra=2, outliers=False):
        self.lens, self.nkv = lens, nkv
        need = [-(-t // PAGE) for t in lens]
        self.max_pages = max(need) + extra
        self.n_pages = n_pages or sum(need) + 3
        x = rng.standard_normal((self.n_pages, nkv, PAGE, HD), dtype=np.float32) + 0.7 * rng.standard_normal((self.n_pages, nkv, 1, HD), dtype=np.float32)
        if outliers:
            x[..., ::37] *= 8
        self.k, self.ks = ref.codec(x)
        self.v, self.vs = ref.codec(rng.standard_normal((self.n_pages, nkv, PAGE, HD), dtype=np.float32))
        ids = rng.permutation(self.n_pages)
        self.table = np.full((len(lens), self.max_pages), -1, np.int32)
        at = 0
        for b, m in enumerate(need):
            self.table[b, :m] = ids[at:at + m]
            at += m
            if lens[b] % PAGE:                                         # behind the last key: whatever the page held before
                tail = self.table[b, m - 1]
                self.ks[tail, :, lens[b] % PAGE:] = np.nan
                self.vs[tail, :, lens[b] % PAGE:] = np.nan
                self.v[tail, :, lens[b] % PAGE:] = 127
        self.rebound()

    def rebound(self):
        self.kb, self.kbs = ref.bounds(self.k, self.ks)
        # a page that is not complete has no bounds: a sequence's last one, and those nobody holds
        full = {int(p) for b, t in enumerate(self.lens) for p in self.table[b, :t // PAGE]}
        for p in range(self.n_pages):
            if p not in full:
                self.kb[p], self.kbs[p] = -1, np.nan

    def device(self):
        return [dev(x) for x in (self.k, self.v, self.ks, self.vs, self.kb, self.kbs)]


def run_sparse(pools, q, row_seq, row_pos, *, top, sink=1, local=1, scale=0.09, q_type="fp32", out_type="fp32", stream=None, calls=1, max_len=None):
    rows, nh, _ = q.shape
    nkv = pools.nkv
    dq = torch.from_numpy(np.ascontiguousarray(q, np.float32)).to(DEV)
    dq = dq.to(torch.bfloat16) if q_type == "bf16" else dq
    out = torch.full((rows, nh, HD), -31.0, dtype=torch.bfloat16 if out_type == "bf16" else torch.float32, device=DEV)
    sel = torch.full((rows, nkv, top), -55, dtype=torch.int32, device=DEV)
    max_len = max_len or max(pools.lens)
    kw = dict(rows=rows, nh=nh, nkv=nkv, kvg=nh // nkv, l_hd=HD, top_pages=top, max_len=max_len)
    wsb = ops.attn_paged_sparse_workspace_bytes(**kw)
    ws = torch.randint(0, 255, (wsb,), dtype=torch.uint8, device=DEV)  # never needs zeroing
    for _ in range(calls):
        ops.attn_paged_sparse_i8(stream, dq, *pools.device(), i32(pools.table), i32(row_seq), i32(row_pos), out, sel, ws, wsb, **kw, batch=len(pools.lens),
                                 n_pages=pools.n_pages, max_pages=pools.max_pages, sink_pages=sink, local_pages=local, softmax_scale=scale,
                                 q_type=ops.BF16 if q_type == "bf16" else ops.F32, out_type=ops.BF16 if out_type == "bf16" else ops.F32)
    torch.cuda.synchronize()
    assert ops.device_faults() == 0
    return out.float().cpu().numpy(), host(sel)


def check_sparse(pools, q, row_seq, row_pos, got, sel, *, top, sink=1, local=1, scale=0.09, out_bf16=False, max_len=None):
    max_len = max_len or max(pools.lens)
    nkv = pools.nkv
    for r, (b, pos) in enumerate(zip(row_seq, row_pos)):
        if not (0 <= b < len(pools.lens) and 0 <= pos < max_len):
            assert (got[r] == -31).all() and (sel[r] == -55).all(), f"row {r} is padding"
            continue
        pages = pools.table[b, :pos // PAGE + 1]
        qr = q[r].reshape(nkv, -1, HD).astype(np.float32)
        want = ref.select(qr, pools.kb, pools.kbs, pages, top, sink, local)
        for h in range(nkv):
            n = len(want[h])
            assert sel[r, h, :n].tolist() == want[h] and (sel[r, h, n:] == -1).all(), (r, h)
        exact = ref.attend(qr, pools.k, pools.ks, pools.v, pools.vs, pages, want, pos, scale).reshape(-1, HD)
        err = np.abs(got[r] - exact)
        bar = 2e-3 * np.sqrt(np.mean(exact ** 2)) + (2.0 ** -8 * np.abs(exact) if out_bf16 else 0)
        assert (err <= bar).all(), (r, float((err - bar).max()))


@pytest.mark.parametrize("kvg,nkv", [(1, 2), (2, 4), (3, 2), (8, 2)])
@pytest.mark.parametrize("top,sink,local", [(1, 0, 1), (4, 1, 1), (7, 1, 3), (16, 0, 2)])
def test_sparse_decode(kvg, nkv, top, sink, local):
    """One row per sequence at every kind of length, padding rows between and behind them."""
    rng = np.random.default_rng(kvg * 100 + top)
    lens = [1, 127, 128, 129, 513, 2048, 2049, 4000]
    pools = Pools(rng, lens, nkv, outliers=True)
    row_seq = np.array([0, 1, 2, -1, 3, 4, 5, 6, 7, 8, 5, -1])
    row_pos = np.array([0, 126, 127, 5, 128, 512, 2047, 2048, 3999, 3, -1, -1])
    q = bf16_normal(rng, (len(row_seq), nkv * kvg, HD))
    for q_type, out_type in (("fp32", "fp32"), ("bf16", "bf16")):
        got, sel = run_sparse(pools, q, row_seq, row_pos, top=top, sink=sink, local=local, q_type=q_type, out_type=out_type, calls=2)
        check_sparse(pools, q, row_seq, row_pos, got, sel, top=top, sink=sink, local=local, out_bf16=out_type == "bf16")


@pytest.mark.parametrize("keys,top", [(1000, 5), (20000, 32), (140000, 64)])
def test_sparse_rows_of_a_sequence(keys, top):
    """Verify rows (each with a selection of its own), and a row far back in the same sequence; long sequences in several clusters."""
    rng = np.random.default_rng(keys)
    nkv, kvg = 2, 2
    pools = Pools(rng, [keys, 300], nkv)
    row_seq = np.array([0] * 9 + [1, 1, 0])
    row_pos = np.concatenate([np.arange(keys - 9, keys), [298, 299, keys // 2]])
    q = bf16_normal(rng, (len(row_seq), nkv * kvg, HD))
    got, sel = run_sparse(pools, q, row_seq, row_pos, top=top, local=2)
    check_sparse(pools, q, row_seq, row_pos, got, sel, top=top, local=2)


@pytest.mark.parametrize("alike", [False, True])
@pytest.mark.parametrize("pages,tops", [(2300, (3, 100, 143, 144, 700)), (1040, (5, 65, 300)), (4097, (256, 257))])
def test_sparse_many_pages(pages, tops, alike):
    """Contexts of thousands of pages (a few physical ones, listed over and over): selection in clusters of every size, more keys than a lane
    keeps in registers, and pages with equal bounds in every CTA of a cluster, where the lowest numbers win."""
    rng = np.random.default_rng(pages)
    nkv, kvg, few = 2, 2, 40
    pools = Pools(rng, [few * PAGE], nkv)
    phys = pools.table[0, :few].copy()
    keys = pages * PAGE - 45
    pools.lens, pools.max_pages = [keys, 500 * PAGE], pages
    pools.table = np.stack([phys[:1].repeat(pages) if alike else rng.choice(phys, pages) for _ in range(2)]).astype(np.int32)
    row_seq, row_pos = np.array([0, 0, 1]), np.array([keys - 1, keys // 2, 500 * PAGE - 1])
    q = bf16_normal(rng, (3, nkv * kvg, HD))
    for top in tops:
        local = 2 if top > 3 else 1
        got, sel = run_sparse(pools, q, row_seq, row_pos, top=top, local=local)
        check_sparse(pools, q, row_seq, row_pos, got, sel, top=top, local=local)


def test_sparse_most_pages():
    """The longest context there is: 49152 pages, one physical page listed over and over between a few others."""
    rng = np.random.default_rng(21)
    pages, few = 49152, 12
    pools = Pools(rng, [few * PAGE], 1)
    phys = pools.table[0, :few].copy()
    pools.lens, pools.max_pages = [pages * PAGE], pages
    pools.table = np.full((1, pages), phys[0], np.int32)
    pools.table[0, rng.choice(pages, 60, replace=False)] = rng.choice(phys[1:], 60)
    row_seq, row_pos = np.array([0, 0]), np.array([pages * PAGE - 1, pages * PAGE - PAGE])
    q = bf16_normal(rng, (2, 1, HD))
    for top in (9, 300):
        got, sel = run_sparse(pools, q, row_seq, row_pos, top=top)
        check_sparse(pools, q, row_seq, row_pos, got, sel, top=top)


def test_sparse_over_all_pages_is_paged_decode():
    """top_pages covering every sequence: dense attention, and the dense entry point's output (each within the bar of the exact one)."""
    rng = np.random.default_rng(8)
    lens, nkv, kvg = [700, 5, 1024], 3, 2
    pools = Pools(rng, lens, nkv)
    q = bf16_normal(rng, (3, nkv * kvg, HD))
    row_pos = np.array(lens) - 1
    got, sel = run_sparse(pools, q, np.arange(3), row_pos, top=pools.max_pages)
    check_sparse(pools, q, np.arange(3), row_pos, got, sel, top=pools.max_pages)
    out = torch.empty((3, nkv * kvg, HD), device=DEV)
    wsb = ops.attn_paged_workspace_bytes(3, nkv * kvg, nkv, kvg, HD, max(lens))
    ws = torch.empty(wsb, dtype=torch.uint8, device=DEV)
    ops.attn_paged_decode_i8(None, dev(np.ascontiguousarray(q, np.float32)), *pools.device()[:4], i32(pools.table), i32(lens), out, ws, wsb, batch=3, nh=nkv * kvg, nkv=nkv,
                             kvg=kvg, l_hd=HD, n_pages=pools.n_pages, max_pages=pools.max_pages, max_len=max(lens), softmax_scale=0.09)
    torch.cuda.synchronize()
    assert np.abs(got - host(out)).max() <= 2 * 2e-3 * np.sqrt(np.mean(got ** 2))


def test_sparse_ties_zeros_and_pages_that_are_not_finite():
    rng = np.random.default_rng(9)
    nkv, kvg, top = 2, 2, 6
    lens = [30 * PAGE + 17] * 4
    pools = Pools(rng, lens, nkv)
    t = pools.table
    for j in range(1, 30):                                             # sequence 0: all pages alike -> the lowest ones
        pools.k[t[0, j]], pools.ks[t[0, j]] = pools.k[t[0, 0]], pools.ks[t[0, 0]]
    pools.ks[t[1, 11], 0, 3] = np.nan                                  # sequence 1: pages that score as the largest finite value
    pools.ks[t[1, 13], 0, 100] = np.inf
    pools.k[t[3, :20]] = 0                                             # sequence 3: zero pages against negative bounds and zero
    pools.rebound()
    q = bf16_normal(rng, (6, nkv * kvg, HD))
    q[2] = 0                                                           # a query of zeros: every score 0
    q[4, 0, 5], q[4, 1, 6] = np.inf, np.nan                            # count 0 in the score
    q[5] *= 1e-40
    row_seq = np.array([0, 1, 2, 3, 2, 3])
    row_pos = np.full(6, 30 * PAGE + 16)
    got, sel = run_sparse(pools, q, row_seq, row_pos, top=top)
    for r in range(6):
        pages = t[row_seq[r], :31]
        want = ref.select(q[r].reshape(nkv, kvg, HD), pools.kb, pools.kbs, pages, top, 1, 1)
        for h in range(nkv):
            assert sel[r, h].tolist() == want[h], (r, h)
    assert sel[0, 0].tolist() == [0, 1, 2, 3, 4, 30] and sel[2, 1].tolist() == [0, 1, 2, 3, 4, 30]
    assert {11, 13} <= set(sel[1, 0].tolist())
    check_sparse(pools, q[:1], row_seq[:1], row_pos[:1], got[:1], sel[:1], top=top)
    check_sparse(pools, q[2:4], row_seq[2:4], row_pos[2:4], got[2:4], sel[2:4], top=top)


@pytest.mark.parametrize("rows,pad,nkv,kvg,top,idle", [(20, 0, 16, 2, 8, 0), (24, 8, 16, 1, 9, 0), (21, 5, 15, 2, 13, 3), (40, 0, 8, 4, 256, 0), (39, 1, 8, 8, 11, 0)])
def test_sparse_rounds_of_units_and_a_split_rest(rows, pad, nkv, kvg, top, idle):
    """More (row, KV head) units than run at once: those left over by whole rounds are split, those before them are not; padding behind
    and between the rows."""
    rng = np.random.default_rng(rows + nkv)
    lens = [int(x) for x in rng.integers(1100, 1700, rows)]
    pools = Pools(rng, lens, nkv)
    row_seq, row_pos = np.concatenate([np.arange(rows), np.full(pad, -1)]), np.concatenate([np.array(lens) - 1, np.full(pad, -1)])
    row_seq[rng.permutation(rows)[:idle]] = -1
    q = bf16_normal(rng, (rows + pad, nkv * kvg, HD))
    got, sel = run_sparse(pools, q, row_seq, row_pos, top=top, calls=2)
    check_sparse(pools, q, row_seq, row_pos, got, sel, top=top)


def test_sparse_workspace_fits_whatever_is_padding():
    """The workspace query knows the rows but not the batch, from which a call guesses how many of them are padding and splits accordingly:
    no call of a sweep over both is refused.  (All rows are padding: the launches write nothing.)"""
    rng = np.random.default_rng(14)
    pools = Pools(rng, [300], 1)
    bufs = pools.device()
    for nkv, kvg in ((1, 1), (3, 2), (16, 2), (8, 8)):
        k, v, ks, vs = (torch.zeros((4, nkv, *x.shape[2:]), dtype=x.dtype, device=DEV) for x in bufs[:4])
        kb, kbs = torch.zeros((4, nkv, 2, HD), dtype=torch.int8, device=DEV), torch.zeros((4, nkv), device=DEV)
        for rows in (1, 5, 19, 20, 24, 37, 64, 100, 149, 255, 256, 257):
            q = torch.zeros((rows, nkv * kvg, HD), device=DEV)
            out = torch.full_like(q, -31)
            pad = i32(np.full(rows, -1))
            for top, keys in ((3, 128 * 64), (8, 128 * 64), (9, 128 * 9), (21, 128 * 200), (64, 128 * 64), (250, 128 * 260)):
                kw = dict(rows=rows, nh=nkv * kvg, nkv=nkv, kvg=kvg, l_hd=HD, top_pages=top, max_len=keys)
                wsb = ops.attn_paged_sparse_workspace_bytes(**kw)
                ws = torch.empty(wsb, dtype=torch.uint8, device=DEV)
                for batch in sorted({1, 2, 3, rows // 5 + 1, rows // 3 + 1, rows // 2 + 1, max(1, rows - 7), rows, 300}):
                    table = torch.zeros((batch, keys // PAGE), dtype=torch.int32, device=DEV)
                    ops.attn_paged_sparse_i8(None, q, k, v, ks, vs, kb, kbs, table, pad, pad, out, None, ws, wsb, **kw, batch=batch, n_pages=4,
                                             max_pages=keys // PAGE)
            torch.cuda.synchronize()
            assert bool((out == -31).all())
    assert ops.device_faults() == 0


def test_sparse_more_rows_than_one_launch():
    """8192 rows make a launch: the rest takes a second one, with a split and a part of the workspace of its own."""
    rng = np.random.default_rng(10)
    nkv, kvg, rows, top = 1, 2, 8192 + 37, 3
    pools = Pools(rng, [900], nkv)
    row_pos = rng.integers(0, 900, rows)
    row_seq = np.zeros(rows, int)
    row_seq[::7] = -1
    q = bf16_normal(rng, (rows, nkv * kvg, HD))
    got, sel = run_sparse(pools, q, row_seq, row_pos, top=top)
    assert (got[::7] == -31).all() and (sel[::7] == -55).all()
    some = np.concatenate([rng.choice(8192, 60, replace=False), np.arange(8180, rows)])
    check_sparse(pools, q[some], row_seq[some], row_pos[some], got[some], sel[some], top=top)


def test_sparse_far_into_a_large_pool():
    """Byte offsets beyond 2^32: pages at the end of a pool of 5 GB per plane."""
    rng = np.random.default_rng(12)
    nkv, kvg, n_pages, top = 16, 2, 20000, 4
    small = Pools(rng, [1500], nkv)
    used = small.table[0, :12].copy()
    far = np.concatenate([n_pages - 1 - np.arange(6), 17000 + 3 * np.arange(6)])
    big = [torch.empty((n_pages, *x.shape[1:]), dtype=torch.from_numpy(x[:0]).dtype, device=DEV) for x in (small.k, small.v, small.ks, small.vs, small.kb, small.kbs)]
    for d, x in zip(big, (small.k, small.v, small.ks, small.vs, small.kb, small.kbs)):
        d[torch.from_numpy(far).to(DEV)] = dev(x[used])
    table = np.full((1, 14), -1, np.int32)
    table[0, :12] = far
    q = bf16_normal(rng, (1, nkv * kvg, HD))
    out = torch.zeros((1, nkv * kvg, HD), device=DEV)
    kw = dict(rows=1, nh=nkv * kvg, nkv=nkv, kvg=kvg, l_hd=HD, top_pages=top, max_len=1500)
    wsb = ops.attn_paged_sparse_workspace_bytes(**kw)
    ws = torch.empty(wsb, dtype=torch.uint8, device=DEV)
    ops.attn_paged_sparse_i8(None, dev(np.ascontiguousarray(q, np.float32)), *big, i32(table), i32([0]), i32([1499]), out, None, ws, wsb, **kw, batch=1, n_pages=n_pages,
                             max_pages=14, softmax_scale=0.09)
    k_new = bf16_normal(rng, (1, nkv, HD))
    ops.kv_paged_append_rows_i8(None, dev(k_new), dev(k_new), *big, i32([far[0] * PAGE + 127]), n_rows=1, nkv=nkv, l_hd=HD, l_kvd=nkv * HD, n_pages=n_pages)
    torch.cuda.synchronize()
    pages = small.table[0, :12]
    qr = q[0].reshape(nkv, kvg, HD).astype(np.float32)
    want = ref.select(qr, small.kb, small.kbs, pages, top, 1, 1)
    exact = ref.attend(qr, small.k, small.ks, small.v, small.vs, pages, want, 1499, 0.09).reshape(-1, HD)
    assert np.abs(host(out)[0] - exact).max() <= 2e-3 * np.sqrt(np.mean(exact ** 2))
    code, sc = ref.codec(k_new[0])
    assert np.array_equal(host(big[0][far[0], :, 127]), code) and np.array_equal(host(big[2][far[0], :, 127]), sc)
    wkb, wkbs = ref.bounds(host(big[0][far[0]]), host(big[2][far[0]]))
    assert np.array_equal(host(big[4][far[0]]), wkb) and np.array_equal(host(big[5][far[0]]), wkbs)


# ------------------------------------------------------------------------------------------------ verification

def verify_case(rng, batch, k, vocab, close=0.5):
    z = 3 * rng.standard_normal((batch, k + 1, vocab))
    soft = lambda x: (np.exp(x - x.max(-1, keepdims=True)) / np.exp(x - x.max(-1, keepdims=True)).sum(-1, keepdims=True)).astype(np.float32)  # noqa: E731
    p, q = soft(z), soft(z[:, :k] + close * rng.standard_normal((batch, k, vocab)))
    tokens = np.array([[rng.choice(vocab, p=q[b, i].astype(np.float64) / q[b, i].astype(np.float64).sum()) for i in range(k)] for b in range(batch)]).reshape(batch, k)
    return p, q, tokens.astype(np.int32), rng.random((batch, k), dtype=np.float32), rng.random(batch, dtype=np.float32)


def run_verify(p, q, tokens, n_draft, ua, us, *, p_pad=0, q_pad=0, shift=0, lens=None, stream=None):
    batch, k1, vocab = p.shape

    def rows(x, pad):                                                  # rows `pad` apart, the first one `shift` elements into its buffer
        flat = np.full(shift + x.shape[0] * x.shape[1] * (vocab + pad), np.nan, np.float32)
        flat[shift:].reshape(*x.shape[:2], vocab + pad)[..., :vocab] = x
        return dev(flat)[shift:]

    acc = torch.full((batch,), -5, dtype=torch.int32, device=DEV)
    out = torch.full((batch, k1), -5, dtype=torch.int32, device=DEV)
    dl = None if lens is None else i32(lens)
    ops.spec_verify(stream, rows(p, p_pad), None if q is None else rows(q, q_pad), i32(tokens) if k1 > 1 else None, None if n_draft is None else i32(n_draft),
                    dev(ua) if k1 > 1 else None, dev(us), dl, dl, acc, out, batch=batch, max_draft=k1 - 1, vocab=vocab, p_stride=vocab + p_pad, q_stride=vocab + q_pad)
    torch.cuda.synchronize()
    want = ref.verify(p, q, tokens, n_draft, ua, us)
    acc, out = host(acc), host(out)
    for b, w in enumerate(want):
        if w is None:
            assert acc[b] == -5 and (out[b] == -5).all()
            assert dl is None or host(dl)[b] == lens[b]
        else:
            assert (acc[b], out[b].tolist()) == w, b
            assert dl is None or host(dl)[b] == lens[b] + w[0] + 1
    return acc, out


@pytest.mark.parametrize("batch,k,vocab", [(1, 1, 1), (1, 3, 5), (3, 8, 31), (2, 4, 1000), (5, 40, 129), (1, 8, 32000), (300, 2, 2049), (2, 3, 50001), (2, 1, 262144)])
@pytest.mark.parametrize("pads", [(0, 0, 0), (3, 8, 1)])
def test_verify(batch, k, vocab, pads):
    rng = np.random.default_rng(batch + k + vocab)
    p, q, tokens, ua, us = verify_case(rng, batch, k, vocab)
    n_draft = rng.integers(-1, k + 3, batch)
    kw = dict(p_pad=pads[0], q_pad=pads[1], shift=pads[2])
    run_verify(p, q, tokens, n_draft, ua, us, lens=rng.integers(0, 1000, batch), **kw)
    run_verify(p, q, tokens, None, ua, us, **kw)
    run_verify(p, None, tokens, None, ua * 0.05, us, **kw)
    run_verify(p, q, tokens, np.zeros(batch), ua, us, **kw)            # nothing drafted: a plain draw


def test_verify_without_drafts():
    rng = np.random.default_rng(1)
    p, _, _, _, us = verify_case(rng, 4, 0, 777)
    run_verify(p, None, np.zeros((4, 0), np.int32), None, np.zeros((4, 0), np.float32), us, lens=[0, 1, 2, 3])


def test_verify_more_sequences_than_a_grid():
    """65535 sequences make a launch."""
    rng = np.random.default_rng(6)
    batch, k, vocab = 65535 + 9, 1, 3
    p = rng.dirichlet(np.ones(vocab), (batch, k + 1)).astype(np.float32)
    q = rng.dirichlet(np.ones(vocab), (batch, k)).astype(np.float32)
    run_verify(p, q, rng.integers(0, vocab, (batch, k)), rng.integers(-1, k + 1, batch), rng.random((batch, k), dtype=np.float32), rng.random(batch, dtype=np.float32),
               lens=rng.integers(0, 9, batch))


def test_operators_on_two_streams_at_once():
    """The whole-number operators hold no state between calls: two of each in flight on two streams."""
    rng = np.random.default_rng(13)
    streams = [torch.cuda.Stream() for _ in range(2)]
    cases = [plan_case(rng, 700 + i, 6, 90, 20, False) for i in range(2)]
    probs = [verify_case(rng, 3, 4, 3000 + i) for i in range(2)]
    work = []
    for i, c in enumerate(cases):
        lens, n_new, held, free, count, table = c
        max_rows = int(np.maximum(n_new, 0).sum())
        d = {"lens": i32(lens), "n_new": i32(n_new), "held": i32(held), "free": i32(free), "count": i32([count]), "table": i32(table),
             "held_out": i32(held * 0), "free_count_out": i32([0]), "granted": i32(held * 0), "row_start": i32(np.zeros(len(lens) + 1))}
        d |= {n: i32(np.zeros(max_rows)) for n in ("slot_map", "row_seq", "row_pos")}
        p, q, tokens, ua, us = probs[i]
        v = [dev(p), dev(q), i32(tokens), None, dev(ua), dev(us), None, None, i32(np.zeros(3)), i32(np.zeros((3, 5)))]
        work.append((d, v, max_rows))
    torch.cuda.synchronize()
    for _ in range(20):
        for i, (d, v, max_rows) in enumerate(work):
            ops.kv_paged_plan(streams[i], d["lens"], d["n_new"], d["held"], d["free"], d["count"], d["table"], d["held_out"], d["free_count_out"], d["granted"],
                              d["row_start"], d["slot_map"], d["row_seq"], d["row_pos"], batch=700 + i, max_pages=6, n_pages=len(cases[i][3]), max_rows=max_rows)
            ops.spec_verify(streams[i], *v, batch=3, max_draft=4, vocab=3000 + i, p_stride=3000 + i, q_stride=3000 + i)
    torch.cuda.synchronize()
    for i, (d, v, max_rows) in enumerate(work):
        same_plan(d, ref.plan(*cases[i], max_rows))
        p, q, tokens, ua, us = probs[i]
        for b, w in enumerate(ref.verify(p, q, tokens, None, ua, us)):
            assert (int(v[8][b]), v[9][b].tolist()) == w


def test_verify_corners():
    """Probabilities and random numbers on borders: u = 0, the largest u below 1, equal rows, zero rows, one-hot rows, tokens that are none."""
    vocab, k = 700, 3
    rng = np.random.default_rng(2)
    top = np.float32(1 - 2.0 ** -24)
    p, q, tokens, ua, us = verify_case(rng, 12, k, vocab)
    ua[:4], us[:6] = 0, [0, top, 0, top, 0.5, 0.25]
    p[1, :, :] = 0; p[1, :, 699] = 1                                   # one-hot on the last token
    q[2] = p[2, :k]; ua[2] = top                                       # equal rows: accepted whatever u is below 1
    p[3, 0] = 0                                                        # nothing to draw from
    ua[4] = 1.0; q[4] = p[4, :k]                                       # out of range: rejected with an empty residual -> p itself
    tokens[5, 0], tokens[6, 0], tokens[7, 1] = -1, vocab, 2 ** 31 - 1
    p[8, 0] = 0; p[8, 0, :2] = 2.0 ** -60                              # weights that count as nothing
    q[9, 0] = 0; ua[9, 0] = top                                        # drafted a token of probability 0: accepted where p > 0
    p[10] = np.float32(2.0 ** -9); p[10, :, 512:] = 0; us[10] = 0.5; q[10] = 0   # exact sums: u * total on a border
    p[10, :, :1] = 0; p[10, :, 512] = np.float32(2.0 ** -9)
    us[11] = 1.0                                                       # out of range: the last token that weighs anything
    acc, out = run_verify(p, q, tokens, None, ua, us)
    assert out[1, acc[1]] == 699 and out[3, 0] == -1 and acc[3] == 0 and acc[2] == k
    run_verify(p, None, tokens, None, ua, us)


def test_verify_draws_the_distribution():
    """Over many uniforms the emitted tokens of one drafted position follow the target: exact per-token counts of the reference, and the
    law of speculative sampling within five standard deviations of a multinomial count."""
    rng = np.random.default_rng(3)
    vocab, n = 40, 4096
    p1, q1, *_ = verify_case(rng, 1, 1, vocab, close=1.0)
    tokens = rng.choice(vocab, (n, 1), p=q1[0, 0].astype(np.float64) / q1[0, 0].astype(np.float64).sum()).astype(np.int32)
    ua, us = rng.random((n, 1), dtype=np.float32), rng.random(n, dtype=np.float32)
    acc, out = run_verify(np.repeat(p1, n, 0), np.repeat(q1, n, 0), tokens, None, ua, us)
    count = np.bincount(out[:, 0], minlength=vocab)
    want = p1[0, 0].astype(np.float64)
    assert (np.abs(count - n * want) <= 5 * np.sqrt(n * want * (1 - want)) + 1).all()


# ------------------------------------------------------------------------------------------------ the loop

class Loop:
    """A batch scheduler's step on the device, every launch of fixed size: plan, append, sparse attention, verify."""

    def __init__(self, rng, batch, nkv, kvg, max_pages, n_pages, k, vocab, top):
        self.batch, self.nkv, self.kvg, self.max_pages, self.n_pages, self.k, self.vocab, self.top = batch, nkv, kvg, max_pages, n_pages, k, vocab, top
        self.max_rows = batch * (k + 1) + 3
        zeros = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)   # noqa: E731
        self.lens, self.n_new, self.held, self.granted, self.start = zeros(batch), zeros(batch), zeros(batch), zeros(batch), zeros(batch + 1)
        self.free, self.count, self.table = i32(rng.permutation(n_pages)), i32([n_pages]), torch.full((batch, max_pages), -1, dtype=torch.int32, device=DEV)
        self.rows = [zeros(self.max_rows) for _ in range(3)]           # slot_map, row_seq, row_pos
        self.pools = empty_pools(n_pages, nkv)
        self.src = [torch.zeros((self.max_rows, nkv, HD), device=DEV) for _ in range(2)]
        self.q = torch.zeros((self.max_rows, nkv * kvg, HD), device=DEV)
        self.out = torch.zeros_like(self.q)
        self.sel = zeros(self.max_rows, nkv, top)
        self.p, self.dq = torch.zeros((batch, k + 1, vocab), device=DEV), torch.zeros((batch, k, vocab), device=DEV)
        self.tokens, self.n_draft, self.ua, self.us = zeros(batch, k), zeros(batch), torch.zeros((batch, k), device=DEV), torch.zeros(batch, device=DEV)
        self.acc, self.emitted = zeros(batch), zeros(batch, k + 1)
        self.kw = dict(rows=self.max_rows, nh=nkv * kvg, nkv=nkv, kvg=kvg, l_hd=HD, top_pages=top, max_len=max_pages * PAGE)
        self.wsb = ops.attn_paged_sparse_workspace_bytes(**self.kw)
        self.ws = torch.empty(self.wsb, dtype=torch.uint8, device=DEV)

    def step(self, stream=None):
        ops.kv_paged_plan(stream, self.lens, self.n_new, self.held, self.free, self.count, self.table, self.held, self.count, self.granted, self.start, *self.rows,
                          batch=self.batch, max_pages=self.max_pages, n_pages=self.n_pages, max_rows=self.max_rows)
        ops.kv_paged_append_rows_i8(stream, *self.src, *self.pools, self.rows[0], n_rows=self.max_rows, nkv=self.nkv, l_hd=HD, l_kvd=self.nkv * HD, n_pages=self.n_pages)
        ops.attn_paged_sparse_i8(stream, self.q, *self.pools, self.table, self.rows[1], self.rows[2], self.out, self.sel, self.ws, self.wsb, **self.kw, batch=self.batch,
                                 n_pages=self.n_pages, max_pages=self.max_pages, softmax_scale=0.09)
        ops.spec_verify(stream, self.p, self.dq, self.tokens, self.n_draft, self.ua, self.us, self.lens, self.lens, self.acc, self.emitted, batch=self.batch, max_draft=self.k,
                        vocab=self.vocab, p_stride=self.vocab, q_stride=self.vocab)


@pytest.mark.parametrize("captured", [False, True])
def test_serving_loop(captured):
    """Thirty steps of a batch that drafts, is rejected, ends and starts again, issued one by one or replayed from one graph on a stream of
    its own; every step against the plain restatements run beside it on host copies of the state."""
    rng = np.random.default_rng(77)
    lp = Loop(rng, batch=5, nkv=2, kvg=2, max_pages=9, n_pages=30, k=7, vocab=50, top=4)
    stream = torch.cuda.Stream()
    graph = None
    if captured:
        lp.n_new.fill_(0); lp.n_draft.fill_(-1)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            lp.step()                                                  # one eager step: everything idle
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            lp.step()
    lens = np.zeros(lp.batch, np.int64)
    lens_start = np.array([0, 900, 500, 128, 1])
    keys = [np.zeros((0, 2, lp.nkv, HD), np.float32) for _ in range(lp.batch)]     # every K/V row a sequence has cached
    prompt = True
    for step in range(30):
        # ---- what the scheduler and the model would bring
        idle = rng.random(lp.batch) < 0.1
        done = (rng.random(lp.batch) < 0.05) & ~idle
        n_draft = np.where(idle | done, -1, rng.integers(0, lp.k + 1, lp.batch))
        n_new = np.where(idle, 0, np.where(done, -1, n_draft + 1))
        if prompt:                                                     # the prompts, cached up front
            for b in range(lp.batch):
                n = int(lens_start[b])
                need = -(-n // PAGE)
                pages = host(lp.free)[int(host(lp.count)[0]) - need:int(host(lp.count)[0])][::-1].copy()
                lp.table[b, :need] = i32(pages)
                lp.count -= need
                lp.held[b] = need
                rows = bf16_normal(rng, (n, 2, lp.nkv, HD))
                keys[b] = rows
                if n:
                    slots = pages[np.arange(n) // PAGE] * PAGE + np.arange(n) % PAGE
                    ops.kv_paged_append_rows_i8(None, dev(rows[:, 0].copy()), dev(rows[:, 1].copy()), *lp.pools, i32(slots), n_rows=n, nkv=lp.nkv, l_hd=HD, l_kvd=lp.nkv * HD,
                                                n_pages=lp.n_pages)
                lens[b] = n
            lp.lens.copy_(i32(lens))
            prompt = False
        src = bf16_normal(rng, (lp.max_rows, 2, lp.nkv, HD))
        q = bf16_normal(rng, (lp.max_rows, lp.nkv * lp.kvg, HD))
        p, dq, tokens, ua, us = verify_case(rng, lp.batch, lp.k, lp.vocab)
        before = ref.plan(lens, n_new, host(lp.held), host(lp.free), int(host(lp.count)[0]), host(lp.table), lp.max_rows)
        n_draft = np.where(before["granted"] > 0, n_draft, -1)         # a request without pages waits
        for t, x in ((lp.n_new, i32(n_new)), (lp.src[0], dev(src[:, 0].copy())), (lp.src[1], dev(src[:, 1].copy())), (lp.q, dev(q)), (lp.p, dev(p)), (lp.dq, dev(dq)),
                     (lp.tokens, i32(tokens)), (lp.ua, dev(ua)), (lp.us, dev(us)), (lp.n_draft, i32(n_draft))):
            t.copy_(x)
        lp.out.fill_(-31); lp.sel.fill_(-55)
        torch.cuda.synchronize()
        if captured:
            graph.replay()
        else:
            lp.step()
        torch.cuda.synchronize()
        # ---- the same beside it
        for name, t in (("table", lp.table), ("held_out", lp.held), ("granted", lp.granted), ("row_start", lp.start), ("slot_map", lp.rows[0]), ("row_seq", lp.rows[1]),
                        ("row_pos", lp.rows[2])):
            assert np.array_equal(host(t), before[name]), (step, name)
        for b in range(lp.batch):
            if n_new[b] < 0:
                lens[b], keys[b] = 0, keys[b][:0]
        n_pages_used = lp.n_pages
        k = np.zeros((n_pages_used, lp.nkv, PAGE, HD), np.int8); v = np.zeros_like(k)
        ks = np.ones((n_pages_used, lp.nkv, PAGE), np.float32); vs = np.ones_like(ks)
        for b in range(lp.batch):
            g = int(before["granted"][b])
            first = before["row_start"][b]
            all_rows = np.concatenate([keys[b][:lens[b]], src[first:first + g]])
            keys[b] = all_rows
            for j in range(-(-len(all_rows) // PAGE)):
                part = all_rows[j * PAGE:(j + 1) * PAGE]
                at = before["table"][b, j]
                for s, pool, sc in ((0, k, ks), (1, v, vs)):
                    code, scale = ref.codec(part[:, s])
                    pool[at, :, :len(part)], sc[at, :, :len(part)] = code.transpose(1, 0, 2), scale.T
        kb, kbs = ref.bounds(k, ks)
        got, sel = host(lp.out), host(lp.sel)
        for r in range(lp.max_rows):
            b, pos = before["row_seq"][r], before["row_pos"][r]
            if b < 0:
                assert (got[r] == -31).all() and (sel[r] == -55).all()
                continue
            pages = before["table"][b, :pos // PAGE + 1]
            qr = q[r].reshape(lp.nkv, lp.kvg, HD).astype(np.float32)
            want = ref.select(qr, kb, kbs, pages, lp.top, 1, 1)
            assert [x[x >= 0].tolist() for x in sel[r]] == want, (step, r)
            exact = ref.attend(qr, k, ks, v, vs, pages, want, pos, 0.09).reshape(-1, HD)
            assert np.abs(got[r] - exact).max() <= 2e-3 * np.sqrt(np.mean(exact ** 2)), (step, r)
        for b, w in enumerate(ref.verify(p, dq, tokens, n_draft, ua, us)):
            if w is not None:
                assert (int(lp.acc[b]), lp.emitted[b].tolist()) == w, (step, b)
                lens[b] += w[0] + 1
        # a finished request's length is the scheduler's to clear
        lp.lens.copy_(torch.where(lp.n_new < 0, 0, lp.lens))
        assert np.array_equal(host(lp.lens), lens)
    assert ops.device_faults() == 0


def test_two_captured_steps_share_buffers():
    """Two graphs of different batch geometry over one workspace, replayed in turn: the workspace carries nothing from one to the next."""
    rng = np.random.default_rng(5)
    nkv, kvg, top = 2, 2, 4
    cases = []
    for lens in ([2500, 300, 900], [4000]):
        pools = Pools(rng, lens, nkv)
        rows = len(lens) * 2
        seq = np.repeat(np.arange(len(lens)), 2)
        pos = np.stack([np.array(lens) - 2, np.array(lens) - 1], 1).reshape(-1)
        q = bf16_normal(rng, (rows, nkv * kvg, HD))
        kw = dict(rows=rows, nh=nkv * kvg, nkv=nkv, kvg=kvg, l_hd=HD, top_pages=top, max_len=max(lens))
        cases.append((pools, q, seq, pos, kw, pools.device() + [i32(pools.table), i32(seq), i32(pos)], dev(np.ascontiguousarray(q, np.float32)),
                      torch.full((rows, nkv * kvg, HD), -31.0, device=DEV), torch.full((rows, nkv, top), -55, dtype=torch.int32, device=DEV)))
    wsb = max(ops.attn_paged_sparse_workspace_bytes(**c[4]) for c in cases)
    ws = torch.randint(0, 255, (wsb,), dtype=torch.uint8, device=DEV)
    graphs = []
    for pools, q, seq, pos, kw, bufs, dq, out, sel in cases:
        def call():
            ops.attn_paged_sparse_i8(None, dq, *bufs, out, sel, ws, wsb, **kw, batch=len(pools.lens), n_pages=pools.n_pages, max_pages=pools.max_pages, softmax_scale=0.09)
        call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        graphs.append(g)
    for _ in range(3):
        for c in cases:
            c[7].fill_(-31.0)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for pools, q, seq, pos, kw, bufs, dq, out, sel in cases:
            check_sparse(pools, q, seq, pos, host(out), host(sel), top=top)
