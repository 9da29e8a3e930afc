"""Plain restatements of the paged serving operators, for their tests: whole numbers as Python / NumPy integers, the
definition's binary32 steps as NumPy float32, everything else in 64 bits."""
from __future__ import annotations

import numpy as np

PAGE, HD = 128, 128
F = np.float32
FLT_MAX = np.finfo(np.float32).max


def plan(lens, n_new, held, free, free_count, table, max_rows):
    """The operator request by request; returns its outputs (table and free list as copies)."""
    table, free = table.copy(), free.copy()
    batch, max_pages = table.shape
    stack = [int(x) for x in free[:free_count]]
    for b in range(batch):
        if n_new[b] < 0:
            stack += [int(x) for x in table[b, :held[b]]]
    pushed = stack[free_count:]
    free[free_count:free_count + len(pushed)] = pushed
    held_out = np.where(n_new < 0, 0, held).astype(np.int32)
    granted = np.zeros(batch, np.int32)
    start = np.zeros(batch + 1, np.int64)
    rows = {n: np.full(max_rows, -1, np.int32) for n in ("slot_map", "row_seq", "row_pos")}
    short = False
    wanted, avail = 0, len(stack)
    for b in range(batch):
        n = max(int(n_new[b]), 0)
        start[b + 1] = start[b] + n
        keys = int(lens[b]) + n
        if n == 0 or start[b + 1] > max_rows or keys > max_pages * PAGE:
            continue
        need = max(0, -(-keys // PAGE) - int(held[b]))
        wanted += need
        short = short or wanted > avail
        if need and short:
            continue
        for i in range(need):
            table[b, held[b] + i] = stack.pop()
        held_out[b] = held[b] + need
        granted[b] = n
        for i in range(n):
            r, pos = start[b] + i, int(lens[b]) + i
            rows["slot_map"][r] = table[b, pos // PAGE] * PAGE + pos % PAGE
            rows["row_seq"][r], rows["row_pos"][r] = b, pos
    return {"table": table, "free": free, "held_out": held_out, "free_count_out": len(stack), "granted": granted,
            "row_start": np.minimum(start, max_rows).astype(np.int32), **rows}


def codec(x):
    """int8 row codec over the last axis: codes, fp32 scales."""
    x = np.asarray(x, F)
    s = (np.abs(x).max(-1) / F(127)).astype(F)
    s[s == 0] = 1
    y = x * (F(1) / s)[..., None]
    y = np.where(y >= 0, y + F(0.5), y - F(0.5))
    return np.clip(np.trunc(y), -127, 127).astype(np.int8), s


def bounds(codes, scales):
    """Page bounds of [..., 128 rows, 128] codes with [..., 128] row scales: int8 [..., 2, 128], fp32 [...]."""
    with np.errstate(all="ignore"):
        v = codes.astype(F) * scales[..., None].astype(F)
        hi, lo = v.max(-2), v.min(-2)
        a = np.maximum(np.abs(hi), np.abs(lo)).max(-1)
        t = (a / F(127)).astype(F)
        t = np.where(t == 0, F(1), t)
        up = np.minimum(np.ceil(hi / t[..., None]), 127)
        down = np.maximum(np.floor(lo / t[..., None]), -127)
    fine = np.isfinite(scales).all(-1) & np.isfinite(a)
    kb = np.where(fine[..., None, None], np.stack([up, down], -2), 0)
    return np.nan_to_num(kb).astype(np.int8), np.where(fine, t, np.inf).astype(F)


def select(q, kb, kbs, pages, top, sink, local):
    """Page numbers a row reads, per KV head.  q [nkv, g, 128] fp32; kb, kbs: the pools; pages: the row's page list."""
    nkv = q.shape[0]
    n = len(pages)
    if n <= top:
        return [list(range(n))] * nkv
    code, s = codec(np.where(np.isfinite(q), q, F(0)))
    code = code.astype(np.int64)
    out = []
    for h in range(nkv):
        b = kb[pages, h].astype(np.int64)                                        # [n, 2, 128]
        whole = np.maximum(code[h][None, :, :] * b[:, None, 0], code[h][None, :, :] * b[:, None, 1]).sum(-1)   # [n, g]
        with np.errstate(all="ignore"):
            score = (whole.astype(F) * kbs[pages, h][:, None]).astype(F) * s[h][None]
        score = np.where(np.isnan(score), FLT_MAX, np.clip(score, -FLT_MAX, FLT_MAX)).astype(np.float64).max(-1)
        score[:sink] = np.inf
        score[n - local:] = np.inf
        out.append(sorted(np.argsort(-score, kind="stable")[:top].tolist()))
    return out


def attend(q, k, ks, v, vs, pages, sel, pos, scale):
    """Exact attention of one row: q [nkv, g, 128]; pools; the row's page list and its selection per KV head."""
    out = np.zeros(q.shape, np.float64)
    for h in range(q.shape[0]):
        at = [pages[j] for j in sel[h]]
        key = np.concatenate([np.arange(j * PAGE, (j + 1) * PAGE) for j in sel[h]])
        see = key <= pos
        kk = (k[at, h].astype(np.float64) * ks[at, h].astype(np.float64)[..., None]).reshape(-1, HD)[see]
        vv = (v[at, h].astype(np.float64) * vs[at, h].astype(np.float64)[..., None]).reshape(-1, HD)[see]
        z = q[h].astype(np.float64) @ kk.T * scale
        w = np.exp(z - z.max(-1, keepdims=True))
        out[h] = w @ vv / w.sum(-1, keepdims=True)
    return out


def verify(p, q, tokens, n_draft, u_accept, u_sample):
    """Accepted counts and emitted tokens, sequence by sequence; None for idle sequences."""
    batch, k1, vocab = p.shape
    out = []
    for b in range(batch):
        n = k1 - 1 if n_draft is None else min(int(n_draft[b]), k1 - 1)
        if n < 0:
            out.append(None)
            continue
        a = 0
        while a < n:
            x = int(tokens[b, a])
            if not 0 <= x < vocab:
                break
            qx = 1.0 if q is None else float(q[b, a, x])
            if not float(u_accept[b, a]) * qx < float(p[b, a, x]):
                break
            a += 1
        pr = p[b, a].astype(np.float64)
        w = pr
        if a < n:
            qr = np.zeros(vocab) if q is None else q[b, a].astype(np.float64)
            if q is None and 0 <= tokens[b, a] < vocab:
                qr[tokens[b, a]] = 1.0
            w = np.maximum(pr - qr, 0)
        whole = np.rint(np.clip(w, 0, 1) * 2.0 ** 50).astype(np.int64)
        if whole.sum() == 0:
            whole = np.rint(np.clip(pr, 0, 1) * 2.0 ** 50).astype(np.int64)
        upto = np.cumsum(whole)
        total = int(upto[-1])
        t = min(max(int(np.floor(float(u_sample[b]) * float(total))), 0), total - 1)
        token = int(np.searchsorted(upto, t, side="right")) if total > 0 else -1
        out.append((a, [int(x) for x in tokens[b, :a]] + [token] + [-1] * (k1 - 1 - a)))
    return out
