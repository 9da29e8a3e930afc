"""Verification at the borders of its range: probabilities that rounding left above 1, and residuals that are empty although the
random numbers are ordinary."""
import numpy as np
import pytest
import torch

from nomos_nvfp4_b200 import ops
from tests._gpu import DEV, dev, host

pytestmark = pytest.mark.gpu


def verify(p, q, tokens, ua, us):
    batch, k1, vocab = p.shape
    acc = torch.full((batch,), -5, dtype=torch.int32, device=DEV)
    out = torch.full((batch, k1), -5, dtype=torch.int32, device=DEV)
    ops.spec_verify(None, dev(p), None if q is None else dev(q), dev(tokens.astype(np.int32)), None, dev(ua.astype(np.float32)), dev(us.astype(np.float32)), None, None,
                    acc, out, batch=batch, max_draft=k1 - 1, vocab=vocab, p_stride=vocab, q_stride=vocab)
    torch.cuda.synchronize()
    return host(acc), host(out)


@pytest.mark.parametrize("vocab", [40, 5000, 70001])
def test_probabilities_above_one(vocab):
    """A place where p > q > 1 weighs nothing (p counts as 1): alone it leaves an empty residual, and the target's row decides;
    beside others it takes nothing from their sum."""
    one = np.float32(1)
    p, q = np.zeros((3, 2, vocab), np.float32), np.zeros((3, 1, vocab), np.float32)
    tokens = np.zeros((3, 1), int)                                     # token 0: p = 0, rejected
    at = vocab - 7
    p[:, 0, at], q[:, 0, at] = one + np.float32(2.0 ** -22), one + np.float32(2.0 ** -23)
    # sequence 0: nothing else has p > q.  The row's weights are 0.25 at 2 and 1 at `at`
    p[0, 0, 2], q[0, 0, 2] = 0.25, 0.5
    # sequence 1: 2^-40 at 3 is the residual (less than the place above 1 would take away)
    p[1, 0, 3] = 2.0 ** -40
    # sequence 2: two places share the residual, one on either side
    p[2, 0, 5], p[2, 0, vocab - 1] = 0.5, 0.5
    acc, out = verify(p, q, tokens, np.full((3, 1), 0.5), np.array([0.1, 0.5, 0.75]))
    assert acc.tolist() == [0, 0, 0]
    assert out.tolist() == [[2, -1], [3, -1], [vocab - 1, -1]]
    # all accepted: the last row draws with the place above 1 counted as 1.  0.5 * (0.25 + 1) lies behind 0.25
    p[:, 0, 0], p[:, 1, 2], p[:, 1, at] = 1, 0.25, one + np.float32(2.0 ** -20)
    acc, out = verify(p, q, tokens, np.full((3, 1), 0.5), np.array([0.1, 0.2, 0.5]))
    assert acc.tolist() == [1, 1, 1] and out.tolist() == [[0, 2], [0, at], [0, at]]


def test_empty_residual_with_ordinary_random_numbers():
    """The target's own row decides where nothing is left of p - q: equal rows and a drafted token of probability 0, a token outside
    the vocabulary, residual weights below 2^-51."""
    vocab = 300
    p, q = np.zeros((3, 2, vocab), np.float32), np.zeros((3, 1, vocab), np.float32)
    p[:, 0, 10], p[:, 0, 20] = 0.5, 0.5
    q[:, 0] = p[:, 0]
    tokens = np.array([[30], [vocab], [30]])                           # p(30) = q(30) = 0: u * 0 < 0 does not hold
    q[2, 0, 10] -= np.float32(0.25); q[2, 0, 20] += np.float32(0.25)
    p[2, 0, 10], q[2, 0, 10] = np.float32(2.0 ** -30 + 2.0 ** -53), np.float32(2.0 ** -30)
    acc, out = verify(p, q, tokens, np.full((3, 1), 0.5), np.array([0.25, 0.75, 0.75]))
    assert acc.tolist() == [0, 0, 0] and out.tolist() == [[10, -1], [20, -1], [20, -1]]
