"""Accuracy of sparse paged attention as the scores grow, and that it repeats itself to the bit.

What the kernel rounds (every tolerance below follows from this list):
  query    16-bit fixed point of the row's largest element, a = max|q|: each element is off by half a step, a / 32639 / 2, plus
           the binary32 rounding of its quotient (below 0.01 of a step): a logit by  scale * 0.51 a / 32639 * sum|k_d|
  logits   binary32 products and sums of numbers no larger than the base-2 logit plus |log2 of the value scale|: six roundings or
           approximate functions of 2^-22 each, 2^-19 of that magnitude covers them; exponentials another 2^-21 of a weight
  weights  on the value codes: half a unit of 1 / 65535 of their page's largest (weight * value scale)
  sums     binary32: 2^-18 of the sum of magnitudes covers some sixty roundings
With d the largest error of a logit and c = cosh d, out' - out = sum w (e^eps - c) (v - out) / sum w e^eps, so that
|out' - out| <= sinh(d) e^d * sum w |v - out| / sum w; the other two add to that."""
import numpy as np
import pytest
import torch

from nomos_nvfp4_b200 import ops
from tests import _paged_ref as ref
from tests._cases import bf16_normal
from tests._gpu import DEV, dev

pytestmark = pytest.mark.gpu
PAGE, HD = 128, 128


def i32(x):
    return dev(np.ascontiguousarray(x, np.int32))


def pages(rng, n, nkv):
    k, ks = ref.codec(rng.standard_normal((n, nkv, PAGE, HD), dtype=np.float32) + 0.7 * rng.standard_normal((n, nkv, 1, HD), dtype=np.float32))
    v, vs = ref.codec(rng.standard_normal((n, nkv, PAGE, HD), dtype=np.float32))
    return [k, v, ks, vs, *ref.bounds(k, ks)]


def exact_and_bound(q, pools, table, sel, pos, scale):
    """64-bit attention of one row over its selection, and how far the kernel may be from it."""
    k, v, ks, vs = pools[:4]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for h in range(q.shape[0]):
        at = [table[j] for j in sel[h]]
        see = np.concatenate([np.arange(j * PAGE, (j + 1) * PAGE) for j in sel[h]]) <= pos
        kk = (k[at, h].astype(np.float64) * ks[at, h].astype(np.float64)[..., None]).reshape(-1, HD)
        code, s = v[at, h].astype(np.float64).reshape(-1, HD), vs[at, h].astype(np.float64).reshape(-1)
        vv = code * s[:, None]
        for j in range(q.shape[1]):
            x = q[h, j].astype(np.float64)
            z = np.where(see, kk @ x * scale, -np.inf)
            w = np.exp(z - z.max())
            o = w @ vv / w.sum()
            d = scale * 0.51 * np.abs(x).max() / 32639 * np.abs(kk[see]).sum(-1).max()
            d += 2.0 ** -19 * np.log(2) * (np.abs(z[see]).max() / np.log(2) + np.abs(np.log2(s[see])).max()) + 2.0 ** -21
            heaviest = (w * s).reshape(-1, PAGE).max(-1, keepdims=True).repeat(PAGE, 1).reshape(-1)       # of the key's page
            fixed = (heaviest[see, None] * np.abs(code[see])).sum(0) * 0.5 / 65535 / w.sum()
            sums = 2.0 ** -18 * (w[see, None] * np.abs(vv[see])).sum(0) / w.sum()
            out[h, j] = o
            bound[h, j] = np.sinh(d) * np.exp(d) * (w[see, None] * np.abs(vv[see] - o)).sum(0) / w.sum() + fixed + sums
    return out.reshape(-1, HD), bound.reshape(-1, HD)


@pytest.mark.parametrize("gain", [1, 8, 30, 100, 1000])
@pytest.mark.parametrize("kvg,top", [(2, 5), (4, 40)])
def test_error_grows_with_the_scores_as_stated(gain, kvg, top):
    rng = np.random.default_rng(gain + kvg)
    nkv, n, rows, scale = 2, 17, 24, HD ** -0.5
    pools = pages(rng, n, nkv)
    table = rng.permutation(n)
    row_pos = rng.integers(0, n * PAGE, rows)
    row_pos[0] = n * PAGE - 1
    q = bf16_normal(rng, (rows, nkv * kvg, HD)) * np.float32(gain)
    out = torch.zeros((rows, nkv * kvg, HD), device=DEV)
    sel = torch.zeros((rows, nkv, top), dtype=torch.int32, device=DEV)
    kw = dict(rows=rows, nh=nkv * kvg, nkv=nkv, kvg=kvg, l_hd=HD, top_pages=top, max_len=n * PAGE)
    wsb = ops.attn_paged_sparse_workspace_bytes(**kw)
    ws = torch.empty(wsb, dtype=torch.uint8, device=DEV)
    ops.attn_paged_sparse_i8(None, dev(np.ascontiguousarray(q, np.float32)), *[dev(x) for x in pools], i32(table[None]), i32(np.zeros(rows)), i32(row_pos), out, sel, ws, wsb, **kw,
                             batch=1, n_pages=n, max_pages=n, softmax_scale=scale)
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    for r in range(rows):
        qr = q[r].reshape(nkv, kvg, HD).astype(np.float32)
        chosen = ref.select(qr, pools[4], pools[5], table[:row_pos[r] // PAGE + 1], top, 1, 1)
        exact, bound = exact_and_bound(qr, pools, table, chosen, row_pos[r], scale)
        assert (np.abs(got[r] - exact) <= bound).all(), (r, float((np.abs(got[r] - exact) / bound).max()))
        if gain == 1:
            assert np.abs(got[r] - exact).max() <= 2e-3 * np.sqrt(np.mean(exact ** 2)), r


@pytest.mark.parametrize("batch,s,nkv,kvg,keys,top,pad", [(1, 1, 4, 2, 8192, 16, 0), (1, 1, 8, 4, 60000, 64, 0), (24, 1, 16, 2, 3000, 9, 8), (4, 9, 16, 2, 4000, 20, 0)])
def test_repeats_itself(batch, s, nkv, kvg, keys, top, pad):
    """The same call again, on a workspace of other noise each time and with other work in between: the same bits, whichever CTA of a split
    row comes last."""
    g = torch.Generator(device=DEV).manual_seed(keys + top)
    per = (keys + PAGE - 1) // PAGE
    n = batch * per
    k, v = (torch.randint(-127, 128, (n, nkv, PAGE, HD), generator=g, device=DEV, dtype=torch.int32).to(torch.int8) for _ in range(2))
    ks, vs = (0.02 * torch.rand((n, nkv, PAGE), generator=g, device=DEV) for _ in range(2))
    kb, kbs = torch.zeros((n, nkv, 2, HD), dtype=torch.int8, device=DEV), torch.zeros((n, nkv), device=DEV)
    ops.kv_paged_page_bounds_i8(None, k, ks, kb, kbs, torch.arange(n, dtype=torch.int32, device=DEV), n=n, nkv=nkv, l_hd=HD, n_pages=n)
    table = torch.randperm(n, generator=g, device=DEV).to(torch.int32).view(batch, per)
    rows = batch * s + pad
    seq = i32(np.concatenate([np.repeat(np.arange(batch), s), np.full(pad, -1)]))
    pos = i32(np.concatenate([np.tile(keys - s + np.arange(s), batch), np.full(pad, -1)]))
    q = torch.randn((rows, nkv * kvg, HD), generator=g, device=DEV)
    kw = dict(rows=rows, nh=nkv * kvg, nkv=nkv, kvg=kvg, l_hd=HD, top_pages=top, max_len=keys)
    wsb = ops.attn_paged_sparse_workspace_bytes(**kw)
    ws = torch.empty(wsb, dtype=torch.uint8, device=DEV)
    first = None
    for i in range(20):
        ws.random_(0, 256, generator=g)
        out = torch.full_like(q, -31)
        sel = torch.full((rows, nkv, top), -55, dtype=torch.int32, device=DEV)
        ops.attn_paged_sparse_i8(None, q, k, v, ks, vs, kb, kbs, table, seq, pos, out, sel, ws, wsb, **kw, batch=batch, n_pages=n, max_pages=per, softmax_scale=0.02)
        torch.cuda.synchronize()
        if first is None:
            first = out, sel
            assert bool(torch.isfinite(out).all()) and bool((out[batch * s:] == -31).all())
        assert torch.equal(out.view(torch.int32), first[0].view(torch.int32)) and torch.equal(sel, first[1]), i
