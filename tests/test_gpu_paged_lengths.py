"""Lengths of a serving step that nobody plans on the host: the verification takes the plan's `granted`, so that requests without pages wait
and prompt chunks advance by their rows, with nothing read back between the four calls."""
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


def softmax(z):
    e = np.exp(z - z.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def expected(p, q, tokens, n_draft, ua, us, granted, lens, acc, out):
    """Requests one by one: nothing granted -> as they were; no tokens asked of (n_draft < 0) -> longer by the rows granted; else the drafts
    whose rows were granted are verified, and the length grows by the other rows and the drafts that stand."""
    k = p.shape[1] - 1
    lens, acc, out = lens.copy(), acc.copy(), out.copy()
    for b in range(len(lens)):
        g, n = int(granted[b]), k if n_draft is None else int(n_draft[b])
        if g <= 0:
            continue
        if n < 0:
            lens[b] += g
            continue
        n = min(n, k, g - 1)
        (a, row), = ref.verify(p[b:b + 1], None if q is None else q[b:b + 1], tokens[b:b + 1], np.array([n]), ua[b:b + 1], us[b:b + 1])
        acc[b], out[b] = a, row
        lens[b] += g - n + a
    return lens, acc, out


@pytest.mark.parametrize("vocab", [37, 4001])
@pytest.mark.parametrize("probs,drafts", [(True, True), (False, True), (True, False)])
@pytest.mark.parametrize("in_place", [False, True])
def test_granted(vocab, probs, drafts, in_place):
    rng = np.random.default_rng(vocab)
    batch, k = 60, 5
    z = 2 * rng.standard_normal((batch, k + 1, vocab))
    p, q = softmax(z), softmax(z[:, :k] + 0.4 * rng.standard_normal((batch, k, vocab)))
    tokens = np.argmax(q + 0.5 * rng.random(q.shape) * q.max(), -1)
    n_draft = rng.integers(-2, k + 3, batch) if drafts else None
    granted = rng.choice([0, 0, -1, 1, 2, 3, 6, 7, 300], batch)
    lens = rng.integers(0, 5000, batch)
    ua, us = rng.random((batch, k), dtype=np.float32), rng.random(batch, dtype=np.float32)
    dl = i32(lens)
    do = dl if in_place else i32(np.full(batch, -3))
    acc, out = i32(np.full(batch, -5)), i32(np.full((batch, k + 1), -5))
    ops.spec_verify(None, dev(p), dev(q) if probs else None, i32(tokens), None if n_draft is None else i32(n_draft), dev(ua), dev(us), dl, do, acc, out, batch=batch,
                    max_draft=k, vocab=vocab, p_stride=vocab, q_stride=vocab, granted=i32(granted))
    torch.cuda.synchronize()
    want = expected(p, q if probs else None, tokens, n_draft, ua, us, granted, lens, np.full(batch, -5), np.full((batch, k + 1), -5))
    assert np.array_equal(host(acc), want[1]) and np.array_equal(host(out), want[2])
    assert np.array_equal(host(do), want[0] if in_place else np.where(granted > 0, want[0], -3))
    assert np.array_equal(host(dl), want[0] if in_place else lens)


def test_granted_without_lengths_and_without_drafts():
    rng = np.random.default_rng(1)
    p = softmax(rng.standard_normal((4, 1, 90)))
    us = rng.random(4, dtype=np.float32)
    acc, out = i32(np.full(4, -5)), i32(np.full((4, 1), -5))
    lens = i32([0, 7, 8, 9])
    for dl in (None, lens):
        ops.spec_verify(None, dev(p), None, None, None, None, dev(us), dl, dl, acc, out, batch=4, max_draft=0, vocab=90, p_stride=90, q_stride=90,
                        granted=i32([130, 0, 1, 4]))
    torch.cuda.synchronize()
    want = ref.verify(p, None, np.zeros((4, 0), np.int32), None, np.zeros((4, 0)), us)
    assert host(acc).tolist() == [0, -5, 0, 0] and host(out)[:, 0].tolist() == [want[0][1][0], -5, want[2][1][0], want[3][1][0]]
    assert host(lens).tolist() == [130, 7, 9, 13]


def test_accepted_counts_over_the_drafted_ones():
    """n_accepted written over n_draft: lengths still follow from what was drafted."""
    rng = np.random.default_rng(8)
    batch, k, vocab = 40, 6, 500
    z = 2 * rng.standard_normal((batch, k + 1, vocab))
    p, q = softmax(z), softmax(z[:, :k] + 0.6 * rng.standard_normal((batch, k, vocab)))
    tokens = np.argmax(q, -1)
    n_draft, granted, lens = rng.integers(-1, k + 1, batch), rng.integers(0, 40, batch), rng.integers(0, 5000, batch)
    ua, us = rng.random((batch, k), dtype=np.float32), rng.random(batch, dtype=np.float32)
    dl, both, out = i32(lens), i32(n_draft), i32(np.full((batch, k + 1), -5))
    ops.spec_verify(None, dev(p), dev(q), i32(tokens), both, dev(ua), dev(us), dl, dl, both, out, batch=batch, max_draft=k, vocab=vocab, p_stride=vocab, q_stride=vocab,
                    granted=i32(granted))
    torch.cuda.synchronize()
    want = expected(p, q, tokens, n_draft, ua, us, granted, lens, n_draft, np.full((batch, k + 1), -5))
    assert np.array_equal(host(dl), want[0]) and np.array_equal(host(both), want[1]) and np.array_equal(host(out), want[2])


class Step:
    """The four calls as the integration notes list them, a request's length cleared when it ends; every launch of fixed size."""

    def __init__(self, rng, batch, nkv, kvg, max_pages, n_pages, max_rows, k, vocab, top):
        self.batch, self.nkv, self.max_pages, self.n_pages, self.max_rows, self.k, self.vocab, self.top = batch, nkv, max_pages, n_pages, max_rows, k, vocab, top
        zeros = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)   # noqa: E731
        self.lens, self.n_new, self.held, self.granted, self.start, self.n_draft = zeros(batch), zeros(batch), zeros(batch), zeros(batch), zeros(batch + 1), zeros(batch)
        self.free, self.count, self.table = i32(rng.permutation(n_pages)), i32([n_pages]), torch.full((batch, max_pages), -1, dtype=torch.int32, device=DEV)
        self.rows = [zeros(max_rows) for _ in range(3)]
        self.pools = [torch.zeros((n_pages, nkv, PAGE, HD), dtype=torch.int8, device=DEV) for _ in range(2)] + [torch.ones((n_pages, nkv, PAGE), device=DEV) for _ in range(2)]
        self.pools += [torch.zeros((n_pages, nkv, 2, HD), dtype=torch.int8, device=DEV), torch.ones((n_pages, nkv), device=DEV)]
        self.src = [torch.zeros((max_rows, nkv, HD), device=DEV) for _ in range(2)]
        self.q = torch.zeros((max_rows, nkv * kvg, HD), device=DEV)
        self.out = torch.zeros_like(self.q)
        self.p, self.dq = torch.zeros((batch, k + 1, vocab), device=DEV), torch.zeros((batch, k, vocab), device=DEV)
        self.tokens, self.ua, self.us = zeros(batch, k), torch.zeros((batch, k), device=DEV), torch.zeros(batch, device=DEV)
        self.acc, self.emitted = zeros(batch), zeros(batch, k + 1)
        self.kw = dict(rows=max_rows, nh=nkv * kvg, nkv=nkv, kvg=kvg, l_hd=HD, top_pages=top, max_len=max_pages * PAGE)
        self.wsb = ops.attn_paged_sparse_workspace_bytes(**self.kw)
        self.ws = torch.empty(self.wsb, dtype=torch.uint8, device=DEV)

    def __call__(self):
        ops.kv_paged_plan(None, self.lens, self.n_new, self.held, self.free, self.count, self.table, self.held, self.count, self.granted, self.start, *self.rows,
                          batch=self.batch, max_pages=self.max_pages, n_pages=self.n_pages, max_rows=self.max_rows)
        ops.kv_paged_append_rows_i8(None, *self.src, *self.pools, self.rows[0], n_rows=self.max_rows, nkv=self.nkv, l_hd=HD, l_kvd=self.nkv * HD, n_pages=self.n_pages)
        ops.attn_paged_sparse_i8(None, self.q, *self.pools, self.table, self.rows[1], self.rows[2], self.out, None, self.ws, self.wsb, **self.kw, batch=self.batch,
                                 n_pages=self.n_pages, max_pages=self.max_pages, softmax_scale=0.09)
        ops.spec_verify(None, self.p, self.dq, self.tokens, self.n_draft, self.ua, self.us, self.lens, self.lens, self.acc, self.emitted, batch=self.batch, max_draft=self.k,
                        vocab=self.vocab, p_stride=self.vocab, q_stride=self.vocab, granted=self.granted)


@pytest.mark.parametrize("captured", [False, True])
def test_steps_with_prompt_chunks_and_a_pool_that_runs_out(captured):
    """Prompts in chunks (tokens asked of the last one only), drafts, requests that end, far more requests than the pool serves; the host
    hands in what each request would like and learns nothing before the step is over.  Requests that were refused bring the same again."""
    rng = np.random.default_rng(31)
    batch, nkv, kvg, k = 6, 1, 2, 3
    st = Step(rng, batch, nkv, kvg, max_pages=6, n_pages=10, max_rows=700, k=k, vocab=30, top=3)
    graph = None
    if captured:
        st.n_draft.fill_(-1)
        st()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            st()
    lens = np.zeros(batch, np.int64)
    prompt = np.array([300, 517, 128, 1, 640, 260])                    # keys still to come of each prompt
    keys = [np.zeros((0, 2, nkv, HD), np.float32) for _ in range(batch)]
    acc, emitted = np.zeros(batch, np.int64), np.zeros((batch, k + 1), np.int64)
    refused = chunks = 0
    for step in range(40):
        n_new, n_draft = np.zeros(batch, int), np.full(batch, -1)
        for b in range(batch):
            if prompt[b] > 0:
                n_new[b] = min(prompt[b], int(rng.integers(1, 200)))
                n_draft[b] = 0 if n_new[b] == prompt[b] else -1
            elif rng.random() < 0.1 or lens[b] > 5 * PAGE:
                n_new[b], prompt[b] = -1, int(rng.integers(1, 500))    # ends, and another one takes its place
                lens[b], keys[b] = 0, keys[b][:0]
            elif rng.random() < 0.9:
                n_draft[b] = rng.integers(0, k + 1)
                n_new[b] = n_draft[b] + 1
        src, q = bf16_normal(rng, (st.max_rows, 2, nkv, HD)), bf16_normal(rng, (st.max_rows, nkv * kvg, HD))
        z = rng.standard_normal((batch, k + 1, st.vocab))
        p, dq = softmax(z), softmax(z[:, :k] + 0.3 * rng.standard_normal((batch, k, st.vocab)))
        tokens = np.argmax(dq, -1)
        ua, us = rng.random((batch, k), dtype=np.float32), rng.random(batch, dtype=np.float32)
        for t, x in ((st.n_new, i32(n_new)), (st.n_draft, i32(n_draft)), (st.src[0], dev(src[:, 0].copy())), (st.src[1], dev(src[:, 1].copy())), (st.q, dev(q)), (st.p, dev(p)),
                     (st.dq, dev(dq)), (st.tokens, i32(tokens)), (st.ua, dev(ua)), (st.us, dev(us))):
            t.copy_(x)
        st.lens.masked_fill_(st.n_new < 0, 0)
        st.out.fill_(-31)
        want = ref.plan(lens, n_new, host(st.held), host(st.free), int(host(st.count)[0]), host(st.table), st.max_rows)
        torch.cuda.synchronize()
        graph.replay() if captured else st()
        torch.cuda.synchronize()
        granted = host(st.granted)
        assert np.array_equal(granted, want["granted"]) and np.array_equal(host(st.table), want["table"])
        refused += int(((n_new > 0) & (granted == 0)).sum())
        # the rows that were placed, and attention over what every sequence holds
        got = host(st.out)
        for b in range(batch):
            first, g = int(want["row_start"][b]), int(granted[b])
            rows = src[first:first + g]
            keys[b] = np.concatenate([keys[b][:lens[b]], rows])
            if g == 0:
                assert (got[first:int(want["row_start"][b + 1])] == -31).all()
                continue
            pages = want["table"][b, :-(-len(keys[b]) // PAGE)]
            pool = [host(x) for x in st.pools[:4]]
            for s in (0, 1):
                code, scale = ref.codec(keys[b][:, s])
                at = np.arange(len(keys[b]))
                assert np.array_equal(pool[s][pages[at // PAGE], :, at % PAGE], code) and np.array_equal(pool[2 + s][pages[at // PAGE], :, at % PAGE], scale), (step, b)
            kb, kbs = host(st.pools[4]), host(st.pools[5])
            for r in (first, first + g - 1):
                pos = int(lens[b]) + r - first
                qr = q[r].reshape(nkv, kvg, HD).astype(np.float32)
                sel = ref.select(qr, kb, kbs, pages[:pos // PAGE + 1], st.top, 1, 1)
                exact = ref.attend(qr, pool[0], pool[2], pool[1], pool[3], pages[:pos // PAGE + 1], sel, pos, 0.09).reshape(-1, HD)
                assert np.abs(got[r] - exact).max() <= 2e-3 * np.sqrt(np.mean(exact ** 2)), (step, b, r)
            if prompt[b] > 0:
                prompt[b] -= g
                chunks += n_draft[b] < 0
        lens, acc, emitted = expected(p, dq, tokens, n_draft, ua, us, granted, lens, acc, emitted)
        assert np.array_equal(host(st.lens), lens), step
        assert np.array_equal(host(st.acc), acc) and np.array_equal(host(st.emitted), emitted), step
    assert refused > 5 and chunks > 5 and ops.device_faults() == 0
