"""Serving operators over paged int8 caches: the work a batch scheduler has them do, their plain forms and inputs.

Kinds of case (`kind`):
  plan     block tables and slot maps from request lengths: pages handed out and taken back, a slot, sequence and position for
           every new row of the step
  append   the new rows of a step quantised into the slots the plan gave them, and the bounds of the pages they complete
  sparse   attention of every query row over the pages of its sequence that a bound on the logits selects
  verify   drafted tokens accepted or rejected against the target's probabilities, and the next token drawn
A page is 128 keys of every KV head, head_dim 128; caches hold int8 rows with one fp32 scale each.
"""
import math

import torch

own = False
DEV = "cuda"
PAGE = 128
HD = 128
FLT_MAX = torch.finfo(torch.float32).max
TT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # a decode step of a small batch: one row per request, few requests at a page's end; latency is everything
        {"name": "plan_decode_64", "kind": "plan", "batch": 64, "max_pages": 256, "rows_each": 1, "finished": 0, "pad": 0, "tight": False},
        # a mixed step of continuous batching, padded to a captured graph's rows: some requests just finished, and not all of the
        # others get their pages
        {"name": "plan_mixed_500", "kind": "plan", "batch": 500, "max_pages": 128, "rows_each": 37, "finished": 20, "pad": 100, "tight": True},
        # long prompts of a large batch admitted at once
        {"name": "plan_prompts_1024", "kind": "plan", "batch": 1024, "max_pages": 64, "rows_each": 255, "finished": 3, "pad": 0, "tight": False},
        # the rows of a decode step on their way into the cache
        {"name": "append_decode_64", "kind": "append", "batch": 64, "nkv": 16, "rows_each": 1, "io": "fp32"},
        # prompt chunks of a batch: most pages they touch are completed, so their bounds are worked out too
        {"name": "append_chunks_8x1021", "kind": "append", "batch": 8, "nkv": 16, "rows_each": 1021, "io": "bf16"},
        # one short chat's token: 64 pages, of which 16 are read
        {"name": "sparse_decode_1x8k", "kind": "sparse", "batch": 1, "nh": 8, "nkv": 4, "keys": 8192, "S": 1, "top": 16, "pad": 0, "io": "bf16"},
        # one very long context: the bounds of 4096 pages against the keys of 64
        {"name": "sparse_decode_1x512k", "kind": "sparse", "batch": 1, "nh": 32, "nkv": 8, "keys": 524288, "S": 1, "top": 64, "pad": 0, "io": "bf16"},
        # batched decode at the benchmark's geometry, ragged lengths, padded to a captured graph's batch
        {"name": "sparse_decode_24x32k", "kind": "sparse", "batch": 24, "nh": 32, "nkv": 16, "keys": 32768, "S": 1, "top": 32, "pad": 8, "io": "bf16"},
        # speculative verify: nine rows per sequence, each with a selection of its own
        {"name": "sparse_verify9_4x16k", "kind": "sparse", "batch": 4, "nh": 32, "nkv": 16, "keys": 16393, "S": 9, "top": 32, "pad": 0, "io": "fp32"},
        # one sequence's eight drafts over a small vocabulary
        {"name": "verify_1x8_32000", "kind": "verify", "batch": 1, "drafts": 8, "vocab": 32000, "probs": True},
        # a drafter that gives tokens only, odd vocabulary
        {"name": "verify_48x3_50001_tokens", "kind": "verify", "batch": 48, "drafts": 3, "vocab": 50001, "probs": False},
        # a large batch over a large vocabulary: two rows of a megabyte each per sequence
        {"name": "verify_96x8_262144", "kind": "verify", "batch": 96, "drafts": 8, "vocab": 262144, "probs": True},
    ]


def _size(rng, lo, hi):
    """A size spread over the logarithm of its range, odd or even."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "append", "sparse", "sparse", "verify"])
    if kind == "plan":
        b, rows = _size(rng, 1, 1024), _size(rng, 1, 255)
        return {"kind": "plan", "batch": b, "max_pages": _size(rng, 8, 256), "rows_each": rows, "finished": rng.randint(0, b // 4), "pad": rng.choice([0, rng.randint(1, 500)]),
                "tight": rng.random() < 0.3}
    if kind == "append":
        b = _size(rng, 1, 64)
        return {"kind": "append", "batch": b, "nkv": rng.choice([1, 4, 8, 16]), "rows_each": _size(rng, 1, 8168 // b), "io": rng.choice(["bf16", "fp32"])}
    if kind == "sparse":
        nh, nkv = rng.choice([(8, 4), (32, 16), (32, 8), (16, 16), (32, 4), (6, 2)])
        b, s = _size(rng, 1, 24), rng.choice([1, 1, 1, 2, 5, 9])
        return {"kind": "sparse", "batch": b, "nh": nh, "nkv": nkv, "keys": _size(rng, 300, 524288 // b), "S": s,
                "top": _size(rng, 4, 32 if b * s > 4 else 64), "pad": rng.choice([0, rng.randint(1, 8)]), "io": rng.choice(["bf16", "fp32"])}
    return {"kind": "verify", "batch": _size(rng, 1, 96), "drafts": rng.randint(1, 8), "vocab": _size(rng, 1000, 262144), "probs": rng.choice([True, True, False])}


# ------------------------------------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(g, lo, hi, n):
    return torch.randint(lo, hi + 1, (n,), generator=g, device=DEV, dtype=torch.int32)


def prepare(case, seed):
    st = {"plan": _prepare_plan, "append": _prepare_append, "sparse": _prepare_sparse, "verify": _prepare_verify}[case["kind"]](case, _gen(seed))
    return {"c": case, **st}


def _prepare_plan(c, g):
    """A pool in use: every request holds the pages of its keys and, now and then, one left over from a rejected draft."""
    b, mp = c["batch"], c["max_pages"]
    # new rows spread evenly over 1 .. 2 * rows_each - 1, so that their sum is the same for every seed; -1 = finished
    n_new = 1 + torch.arange(b, device=DEV) * (2 * c["rows_each"] - 2) // max(1, b - 1)
    n_new[: c["finished"]] = -1
    n_new = n_new[torch.randperm(b, generator=g, device=DEV)].to(torch.int32)
    lens = (torch.rand(b, generator=g, device=DEV) * (mp * PAGE - n_new).clamp(min=1)).to(torch.int32)
    held = ((lens + PAGE - 1) // PAGE + (torch.rand(b, generator=g, device=DEV) < 0.1).to(torch.int32)).clamp(max=mp).to(torch.int32)
    n_pages = b * mp
    ids = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((b, mp), -1, dtype=torch.int32, device=DEV)
    used = torch.arange(mp, device=DEV)[None] < held[:, None]
    n_used = int(used.sum())
    table[used] = ids[:n_used]
    free = torch.full((n_pages,), -1, dtype=torch.int32, device=DEV)
    free[: n_pages - n_used] = ids[n_used:]
    max_rows = int(n_new.clamp(min=0).sum()) + c["pad"]
    spare = n_pages - n_used
    if c["tight"]:                                             # about half of the pages that the step would like
        spare = min(spare, b * c["rows_each"] // (2 * PAGE))
    st = {"lens": lens, "n_new": n_new, "held": held, "table": table, "free": free, "n_pages": n_pages, "max_rows": max_rows}
    st["free_count"] = torch.tensor([spare], dtype=torch.int32, device=DEV)
    for name, n in (("held_out", b), ("free_count_out", 1), ("granted", b), ("row_start", b + 1), ("slot_map", max_rows), ("row_seq", max_rows), ("row_pos", max_rows)):
        st[name] = torch.zeros(n, dtype=torch.int32, device=DEV)
    return st


def _key_rows(g, pages, nkv, outliers):
    """K rows as a model leaves them: a centre that drifts from page to page, noise around it, four outlier channels per head (x8)."""
    centre = 0.7 * torch.randn((pages, nkv, 1, HD), generator=g, device=DEV)
    return (centre + torch.randn((pages, nkv, PAGE, HD), generator=g, device=DEV)) * outliers


def _outliers(g, nkv):
    o = torch.ones((nkv, 1, HD), device=DEV)
    return o.scatter_(2, torch.rand((nkv, 1, HD), generator=g, device=DEV).topk(4, dim=2).indices, 8.0)


def _pools(g, n_pages, nkv):
    """Pools of quantised pages with their bounds, filled in pieces that leave the card room."""
    st = {n + "_pool": torch.empty((n_pages, nkv, PAGE, HD), dtype=torch.int8, device=DEV) for n in "kv"}
    st |= {n + "s_pool": torch.empty((n_pages, nkv, PAGE), device=DEV) for n in "kv"}
    st["kb_pool"] = torch.empty((n_pages, nkv, 2, HD), dtype=torch.int8, device=DEV)
    st["kbs_pool"] = torch.empty((n_pages, nkv), device=DEV)
    o, step = _outliers(g, nkv), max(1, 8192 // nkv)
    for i in range(0, n_pages, step):
        n = min(step, n_pages - i)
        st["k_pool"][i:i + n], st["ks_pool"][i:i + n] = _codec(_key_rows(g, n, nkv, o))
        st["v_pool"][i:i + n], st["vs_pool"][i:i + n] = _codec(torch.randn((n, nkv, PAGE, HD), generator=g, device=DEV))
        st["kb_pool"][i:i + n], st["kbs_pool"][i:i + n] = _bounds(st["k_pool"][i:i + n], st["ks_pool"][i:i + n])
    return st


def _prepare_append(c, g):
    """Rows at ragged positions of sequences whose pages lie anywhere in the pool."""
    b, nkv = c["batch"], c["nkv"]
    n = _ints(g, max(1, c["rows_each"] - 3), c["rows_each"], b)
    base = _ints(g, 0, 2 * PAGE, b)
    per = (2 * PAGE + c["rows_each"]) // PAGE + 1
    st = _pools(g, b * per, nkv)
    table = torch.randperm(b * per, generator=g, device=DEV).view(b, per)
    seq = torch.repeat_interleave(torch.arange(b, device=DEV), n.long())
    pos = base.long()[seq] + torch.arange(seq.numel(), device=DEV) - (n.cumsum(0) - n).long()[seq]
    st["slot_map"] = (table[seq, pos // PAGE] * PAGE + pos % PAGE).to(torch.int32)
    rows = seq.numel()
    st["src_k"] = (torch.randn((rows, nkv, HD), generator=g, device=DEV) * _outliers(g, nkv).view(nkv, HD)).to(TT[c["io"]])
    st["src_v"] = torch.randn((rows, nkv, HD), generator=g, device=DEV).to(TT[c["io"]])
    st["n_pages"], st["rows"] = b * per, rows
    return st


def _prepare_sparse(c, g):
    b, s, nkv = c["batch"], c["S"], c["nkv"]
    per = (c["keys"] + PAGE - 1) // PAGE
    st = _pools(g, b * per, nkv)
    st["table"] = torch.randperm(b * per, generator=g, device=DEV).to(torch.int32).view(b, per)
    lens = (c["keys"] * (0.5 + 0.5 * torch.rand(b, generator=g, device=DEV))).to(torch.int32).clamp(min=s)
    lens[0] = c["keys"]                                        # the longest is as long as the case says
    pad = torch.full((c["pad"],), -1, dtype=torch.int32, device=DEV)
    st["row_seq"] = torch.cat([torch.arange(b, device=DEV, dtype=torch.int32).repeat_interleave(s), pad])
    st["row_pos"] = torch.cat([(lens[:, None] - s + torch.arange(s, device=DEV, dtype=torch.int32)).view(-1), pad]).to(torch.int32)
    rows = b * s + c["pad"]
    st["q"] = torch.randn((rows, c["nh"], HD), generator=g, device=DEV).to(TT[c["io"]])
    st["out"] = torch.zeros((rows, c["nh"], HD), dtype=torch.bfloat16, device=DEV)
    st["sel"] = torch.full((rows, nkv, c["top"]), -1, dtype=torch.int32, device=DEV)
    st["rows"], st["per"], st["n_pages"] = rows, per, b * per
    st["ws"] = None                                            # made by the first call that needs one
    return st


def _prepare_verify(c, g):
    """Rows of a softmax with a heavy head, drafts drawn from a drafter that is close to the target."""
    b, k, v = c["batch"], c["drafts"], c["vocab"]
    head = 4.0 - 0.5 * torch.arange(1, v + 1, device=DEV).float().log()
    p = torch.empty((b, k + 1, v), device=DEV)
    q = torch.empty((b, k, v), device=DEV)
    tokens = torch.empty((b, k), dtype=torch.int32, device=DEV)
    for i in range(b):
        z = head[torch.randperm(v, generator=g, device=DEV)] + 1.5 * torch.randn((k + 1, v), generator=g, device=DEV)
        p[i] = torch.softmax(z, -1)
        q[i] = torch.softmax(z[:k] + 0.4 * torch.randn((k, v), generator=g, device=DEV), -1)
        # the drafter's own draw: the largest of q / Exp(1)
        tokens[i] = (q[i] / -torch.log(torch.rand((k, v), generator=g, device=DEV).clamp(min=1e-30))).argmax(-1).to(torch.int32)
    n_draft = torch.full((b,), k, dtype=torch.int32, device=DEV)
    n_draft[1::5] = k // 2                                     # some sequences drafted less
    st = {"p": p, "q": q if c["probs"] else None, "tokens": tokens, "n_draft": n_draft, "lens": _ints(g, 1, 100000, b)}
    st["u_accept"] = torch.rand((b, k), generator=g, device=DEV) * (1.0 if c["probs"] else 0.3)
    st["u_sample"] = torch.rand((b,), generator=g, device=DEV)
    st["accepted"] = torch.zeros(b, dtype=torch.int32, device=DEV)
    st["emitted"] = torch.zeros((b, k + 1), dtype=torch.int32, device=DEV)
    st["lens_out"] = torch.zeros(b, dtype=torch.int32, device=DEV)
    return st


# ------------------------------------------------------------------------------------------------ one pass

def run(st):
    kind = st["c"]["kind"]
    if own:
        return {"plan": _own_plan, "append": _own_append, "sparse": _own_sparse, "verify": _own_verify}[kind](st)
    return {"plan": _plain_plan, "append": _plain_append, "sparse": _plain_sparse, "verify": _plain_verify}[kind](st)


def _own_plan(st):
    from nomos_nvfp4_b200 import ops
    ops.kv_paged_plan(None, st["lens"], st["n_new"], st["held"], st["free"], st["free_count"], st["table"], st["held_out"], st["free_count_out"], st["granted"],
                      st["row_start"], st["slot_map"], st["row_seq"], st["row_pos"], batch=st["c"]["batch"], max_pages=st["c"]["max_pages"], n_pages=st["n_pages"],
                      max_rows=st["max_rows"])
    return {n: st[n] for n in ("table", "free", "held_out", "free_count_out", "granted", "row_start", "slot_map", "row_seq", "row_pos")}


def _plain_plan(st):
    c, lens, n_new, held, table, free = st["c"], st["lens"].long(), st["n_new"].long(), st["held"].long(), st["table"], st["free"]
    b, mp, max_rows = c["batch"], c["max_pages"], st["max_rows"]
    rows = n_new.clamp(min=0)
    end = rows.cumsum(0)
    released = torch.where(n_new < 0, held, 0)
    fits = (n_new > 0) & (end <= max_rows) & (lens + n_new <= mp * PAGE)
    need = torch.where(fits, ((lens + n_new + PAGE - 1) // PAGE - held).clamp(min=0), 0)
    upto = need.cumsum(0)
    avail = st["free_count"].long() + released.sum()
    ok = fits & ((need == 0) | (upto <= avail))
    need = torch.where(ok, need, 0)
    granted = torch.where(ok, n_new, 0)
    # the stack of free pages with the finished requests' pages on top (one place more takes what is not given)
    j = torch.arange(mp, device=DEV)
    place = st["free_count"].long() + (released.cumsum(0) - released)[:, None] + j
    give = (j < released[:, None]) & (place < st["n_pages"])
    stack = torch.nn.functional.pad(free, (0, 1)).scatter_(0, torch.where(give, place, st["n_pages"]).view(-1), table.view(-1))
    free.copy_(stack[:-1])
    new = (j >= held[:, None]) & (j < (held + need)[:, None])
    at = (avail - 1) - (upto - need)[:, None] - (j - held[:, None])
    table.copy_(torch.where(new, free[at.clamp(0, st["n_pages"] - 1)], table))
    r = torch.arange(max_rows, device=DEV)
    seq = torch.searchsorted(end, r, right=True).clamp(max=b - 1)
    live = ok[seq] & (r < end[-1])
    pos = lens[seq] + r - (end - rows)[seq]
    slot = table[seq, (pos // PAGE).clamp(max=mp - 1)].long() * PAGE + pos % PAGE
    full = [torch.where(live, y, -1).to(torch.int32) for y in (slot, seq, pos)]
    start = torch.nn.functional.pad(end, (1, 0)).clamp(max=max_rows)
    return {"table": table, "free": free, "held_out": torch.where(n_new < 0, 0, held + need).to(torch.int32), "free_count_out": (avail - need.sum()).to(torch.int32),
            "granted": granted.to(torch.int32), "row_start": start.to(torch.int32), "slot_map": full[0], "row_seq": full[1], "row_pos": full[2]}


def _own_append(st):
    from nomos_nvfp4_b200 import ops
    c = st["c"]
    ops.kv_paged_append_rows_i8(None, st["src_k"], st["src_v"], st["k_pool"], st["v_pool"], st["ks_pool"], st["vs_pool"], st["kb_pool"], st["kbs_pool"], st["slot_map"],
                                n_rows=st["rows"], nkv=c["nkv"], l_hd=HD, l_kvd=c["nkv"] * HD, n_pages=st["n_pages"], src_type=ops.BF16 if c["io"] == "bf16" else ops.F32)
    return {n: st[n] for n in ("k_pool", "v_pool", "ks_pool", "vs_pool", "kb_pool", "kbs_pool")}


def _codec(x):
    """Rows -> int8 codes and fp32 scales: scale amax / 127 (0 -> 1), code trunc(x * (1 / scale) +- 0.5).  The divisors are tensors:
    a division by a Python number is done as a product with its reciprocal."""
    x = x.float()
    s = x.abs().amax(-1) / torch.full((), 127.0, device=x.device)
    s = torch.where(s == 0, 1.0, s)
    y = x * (torch.ones_like(s) / s)[..., None]
    return torch.where(y >= 0, y + 0.5, y - 0.5).trunc().clamp(-127, 127).to(torch.int8), s


def _bounds(codes, scales):
    """[..., 128 rows, 128 channels] codes -> per channel the largest and smallest value of the page, rounded outwards to int8."""
    v = codes.float() * scales[..., None]
    hi, lo = v.amax(-2), v.amin(-2)
    t = torch.maximum(hi.abs(), lo.abs()).amax(-1) / torch.full((), 127.0, device=v.device)
    t = torch.where(t == 0, 1.0, t)
    up, down = (hi / t[..., None]).ceil().clamp(max=127), (lo / t[..., None]).floor().clamp(min=-127)
    return torch.stack([up, down], -2).to(torch.int8), t


def _plain_append(st):
    slot = st["slot_map"].long()
    page, row = slot // PAGE, slot % PAGE
    for n in "kv":
        codes, scales = _codec(st["src_" + n])
        st[n + "_pool"][page, :, row] = codes
        st[n + "s_pool"][page, :, row] = scales
    done = page[row == PAGE - 1]
    st["kb_pool"][done], st["kbs_pool"][done] = _bounds(st["k_pool"][done], st["ks_pool"][done])
    return {n: st[n] for n in ("k_pool", "v_pool", "ks_pool", "vs_pool", "kb_pool", "kbs_pool")}


def _own_sparse(st):
    from nomos_nvfp4_b200 import ops
    c = st["c"]
    nh, nkv = c["nh"], c["nkv"]
    if st["ws"] is None:
        n = ops.attn_paged_sparse_workspace_bytes(rows=st["rows"], nh=nh, nkv=nkv, kvg=nh // nkv, l_hd=HD, top_pages=c["top"], max_len=c["keys"])
        st["ws"] = torch.empty(n, dtype=torch.uint8, device=DEV)
    ops.attn_paged_sparse_i8(None, st["q"], st["k_pool"], st["v_pool"], st["ks_pool"], st["vs_pool"], st["kb_pool"], st["kbs_pool"], st["table"], st["row_seq"], st["row_pos"],
                             st["out"], st["sel"], st["ws"], st["ws"].numel(), rows=st["rows"], batch=c["batch"], nh=nh, nkv=nkv, kvg=nh // nkv, l_hd=HD,
                             n_pages=st["n_pages"], max_pages=st["per"], max_len=c["keys"], top_pages=c["top"], sink_pages=1, local_pages=2, softmax_scale=HD ** -0.5,
                             q_type=ops.BF16 if c["io"] == "bf16" else ops.F32, out_type=ops.BF16)
    return {"out": st["out"], "sel": st["sel"]}


def _plain_sparse(st):
    c = st["c"]
    nkv, g, top = c["nkv"], c["nh"] // c["nkv"], c["top"]
    n = st["rows"] - c["pad"]                                  # the padding comes last
    pos, table = st["row_pos"][:n].long(), st["table"][st["row_seq"][:n].long()].long()       # [n], [n, P]
    q = st["q"][:n].float().view(n, nkv, g, HD)
    # a bound on every page's logits: int8 query against the int8 bounds (whole numbers below 2^24: exact in fp32)
    codes, s = _codec(q)
    both = torch.cat([codes.clamp(min=0), codes.clamp(max=0)], -1).float()                    # [n, nkv, g, 256]
    bound = torch.einsum("nhgd,nphd->nhgp", both, st["kb_pool"][table].view(n, -1, nkv, 2 * HD).float())
    bound = (bound * st["kbs_pool"][table].transpose(1, 2)[:, :, None]) * s[..., None]
    score = bound.amax(2).nan_to_num(FLT_MAX, FLT_MAX, -FLT_MAX)                              # [n, nkv, P]
    page = torch.arange(table.shape[1], device=DEV)
    seen = (pos // PAGE + 1)[:, None, None]
    score = torch.where((page < 1) | (page >= seen - 2), math.inf, score)                     # first page and last two: always
    score = torch.where(page < seen, score, -math.inf)
    best, order = torch.sort(score, dim=-1, descending=True, stable=True)
    best, order = best[..., :top], order[..., :top]
    sel = torch.where(best > -math.inf, order, 1 << 30).sort(-1).values
    if sel.shape[-1] < top:
        sel = torch.nn.functional.pad(sel, (0, top - sel.shape[-1]), value=1 << 30)
    kept = sel < 1 << 30
    phys = table[torch.arange(n, device=DEV)[:, None, None], torch.where(kept, sel, 0)]       # [n, nkv, top]
    head = torch.arange(nkv, device=DEV)[None, :, None]
    k = st["k_pool"][phys, head].float() * st["ks_pool"][phys, head][..., None]               # [n, nkv, top, 128, 128]
    logits = torch.einsum("nhgd,nhkd->nhgk", q, k.view(n, nkv, -1, HD)) * HD ** -0.5
    del k
    key = sel[..., None] * PAGE + torch.arange(PAGE, device=DEV)
    mask = (kept[..., None] & (key <= pos[:, None, None, None])).view(n, nkv, 1, -1)
    logits = torch.where(mask, logits, -math.inf)
    w = torch.where(mask, (logits - logits.amax(-1, keepdim=True)).exp(), 0.0)
    v = st["v_pool"][phys, head].float() * st["vs_pool"][phys, head][..., None]
    o = torch.einsum("nhgk,nhkd->nhgd", w, v.view(n, nkv, -1, HD)) / w.sum(-1, keepdim=True)
    st["out"][:n] = o.reshape(n, nkv * g, HD).to(torch.bfloat16)
    st["sel"][:n] = torch.where(kept, sel, -1).to(torch.int32)
    return {"out": st["out"], "sel": st["sel"]}


def _own_verify(st):
    from nomos_nvfp4_b200 import ops
    c = st["c"]
    ops.spec_verify(None, st["p"], st["q"], st["tokens"], st["n_draft"], st["u_accept"], st["u_sample"], st["lens"], st["lens_out"], st["accepted"], st["emitted"],
                    batch=c["batch"], max_draft=c["drafts"], vocab=c["vocab"], p_stride=c["vocab"], q_stride=c["vocab"])
    return {"accepted": st["accepted"], "emitted": st["emitted"], "lens": st["lens_out"]}


def _plain_verify(st):
    p, q, tokens, n = st["p"], st["q"], st["tokens"].long(), st["n_draft"].long()
    b, k, v = p.shape[0], p.shape[1] - 1, p.shape[2]
    i = torch.arange(k, device=DEV)
    px = p[:, :k].gather(2, tokens[..., None])[..., 0].double()
    qx = torch.ones_like(px) if q is None else q.gather(2, tokens[..., None])[..., 0].double()
    good = (st["u_accept"].double() * qx < px) & (i < n[:, None])
    a = good.long().cumprod(1).sum(1)
    row = torch.arange(b, device=DEV)
    x = tokens[row, a.clamp(max=k - 1)]
    rejected = a < n
    pr = p[row, a].double()
    if q is None:
        qr = torch.zeros_like(pr).scatter_(1, x[:, None], 1.0)
    else:
        qr = q[row, a.clamp(max=k - 1)].double()
    # whole numbers of 2^-50: sums do not depend on their order
    w = torch.where(rejected[:, None], (pr - qr).clamp(min=0), pr)
    w = (w.clamp(max=1) * 2.0 ** 50).round().long()
    none = w.sum(1, keepdim=True) == 0
    w = torch.where(none, (pr.clamp(0, 1) * 2.0 ** 50).round().long(), w)
    upto = w.cumsum(1)
    total = upto[:, -1]
    t = (st["u_sample"].double() * total.double()).floor().long().clamp(min=0).minimum(total - 1)
    token = torch.searchsorted(upto, t[:, None], right=True)[:, 0]
    token = torch.where(total > 0, token, -1)
    j = torch.arange(k + 1, device=DEV)
    drafted = torch.nn.functional.pad(tokens, (0, 1))
    emitted = torch.where(j < a[:, None], drafted, torch.where(j == a[:, None], token[:, None], -1))
    return {"accepted": a.to(torch.int32), "emitted": emitted.to(torch.int32), "lens": st["lens"] + a.to(torch.int32) + 1}


# ------------------------------------------------------------------------------------------------ work and exact values

def work(case):
    c = case
    if c["kind"] == "plan":
        rows = c["batch"] * c["rows_each"]
        # lengths, counts and page counts in; tables' new pages and three numbers for every row out
        return {"bytes": 24 * c["batch"] + 12 * (rows + c["pad"]) + 8 * rows / PAGE, "flops": 0}
    if c["kind"] == "append":
        rows = c["batch"] * c["rows_each"]
        size = 2 if c["io"] == "bf16" else 4
        done = rows / PAGE * c["nkv"]                           # pages completed: their bounds are written
        return {"bytes": rows * c["nkv"] * 2 * (HD * size + HD + 4) + 4 * rows + done * (2 * HD + 4), "flops": 0}
    if c["kind"] == "sparse":
        rows, pages = c["batch"] * c["S"], 0.75 * c["keys"] / PAGE if c["batch"] > 1 else c["keys"] / PAGE
        read = min(c["top"], pages)
        size = 2 if c["io"] == "bf16" else 4
        # the bounds once per sequence, the selected pages once per sequence (its rows select much the same ones)
        by = c["batch"] * c["nkv"] * (pages * (2 * HD + 4) + read * PAGE * 2 * (HD + 4)) + rows * c["nh"] * HD * (size + 2) + 4 * rows * c["nkv"] * c["top"]
        return {"bytes": by, "flops": rows * c["nh"] * (4 * HD * read * PAGE + 4 * HD * pages)}
    # one target row per sequence, and the drafter's where a draft is rejected: nearly always at eight drafts
    share = min(1.0, 0.1 * c["drafts"] + 0.2) if c["probs"] else 0.0
    return {"bytes": c["batch"] * c["vocab"] * 4 * (1 + share), "flops": 0}


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(st)
    if case["kind"] == "sparse":
        return _exact_sparse(st)
    return None                                                # whole numbers throughout


def _exact_append(st):
    """Scales in 64 bits; codes are whole numbers and have no such value."""
    slot = st["slot_map"].long()
    ks, vs, kbs = st["ks_pool"].double(), st["vs_pool"].double(), st["kbs_pool"].double()
    for pool, src in ((ks, st["src_k"]), (vs, st["src_v"])):
        s = src.double().abs().amax(-1) / 127
        pool[slot // PAGE, :, slot % PAGE] = torch.where(s == 0, 1.0, s)
    # a page's bound scale is its largest |code| * scale / 127, and a row's largest code is always +-127
    done = (slot // PAGE)[slot % PAGE == PAGE - 1]
    kbs[done] = ks[done].amax(-1)
    return {"k_pool": None, "v_pool": None, "ks_pool": ks, "vs_pool": vs, "kb_pool": None, "kbs_pool": kbs}


def _exact_sparse(st):
    """Row by row in 64 bits.  The definition quantises the query and rounds the bound in binary32; numpy does that here."""
    import numpy as np
    c, f = st["c"], np.float32
    nkv, g, top = c["nkv"], c["nh"] // c["nkv"], c["top"]
    out = torch.zeros(st["out"].shape, dtype=torch.float64, device=DEV)
    for r, (b, pos) in enumerate(zip(st["row_seq"].tolist(), st["row_pos"].tolist())):
        if b < 0:
            continue
        n = pos // PAGE + 1
        pages = st["table"][b, :n].long()
        x = st["q"][r].float().cpu().numpy().reshape(nkv, g, HD)
        s = np.abs(x).max(-1) / f(127)
        s[s == 0] = 1
        code = x * (f(1) / s)[..., None]
        code = np.clip(np.trunc(code + np.copysign(f(0.5), code)), -127, 127)
        kb = st["kb_pool"][pages].double()                      # [n, nkv, 2, 128]
        cd = torch.from_numpy(code).to(DEV).double()
        whole = torch.einsum("hgd,phd->hgp", cd.clamp(min=0), kb[:, :, 0]) + torch.einsum("hgd,phd->hgp", cd.clamp(max=0), kb[:, :, 1])
        score = whole.cpu().numpy().astype(f) * st["kbs_pool"][pages].cpu().numpy().T[:, None]
        score = (score * s[..., None]).max(1)                   # [nkv, n]
        if n > top:
            score[:, 0] = score[:, n - 2:] = np.inf
        for h in range(nkv):
            keep = np.sort(np.argsort(-score[h], kind="stable")[:top])
            at = pages[torch.from_numpy(keep).to(DEV)]
            k = (st["k_pool"][at, h].double() * st["ks_pool"][at, h].double()[..., None]).reshape(-1, HD)
            v = (st["v_pool"][at, h].double() * st["vs_pool"][at, h].double()[..., None]).reshape(-1, HD)
            m = len(k) - (PAGE - 1 - pos % PAGE)                # the last page kept is the row's own
            w = torch.softmax(st["q"][r].double().view(nkv, g, HD)[h] @ k[:m].T * HD ** -0.5, -1)
            out[r].view(nkv, g, HD)[h] = w @ v[:m]
    return {"out": out, "sel": None}
