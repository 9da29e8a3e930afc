"""Verification with the plan's `granted`: refusals, and argument blocks of callers built without the field (no launch)."""
import struct

import pytest

P = 0x1000                               # never dereferenced: validation fails first


@pytest.fixture(scope="module")
def ops():
    from nomos_nvfp4_b200 import build, ops
    build.build()
    return ops


def test_misaligned(ops):
    kw = dict(batch=2, max_draft=3, vocab=100, p_stride=100, q_stride=100)
    with pytest.raises(ops.NomosError) as e:
        ops.spec_verify(0, *[P] * 10, **kw, granted=P + 2)
    assert e.value.status == -1
    ops.spec_verify(0, *[None] * 10, **{**kw, "batch": 0}, granted=None)


def test_blocks_without_the_field(ops):
    from nomos_nvfp4_b200 import _lib
    fn, size = _lib.lib().nomos_attn_spec_verify, _lib.packer(_lib.AttnVerify).size

    def call(struct_bytes, length, batch=0):
        fields = [struct_bytes] + [0] * 10 + [batch, 3, 100, 100, 100]     # no pointers: a batch is refused, none is nothing to do
        return fn(None, struct.pack("=16Q", *fields).ljust(length, b"\xff"))

    assert size == 17 * 8
    assert call(size, size) == 0 and call(size - 8, size - 8) == 0 and call(size - 8, size) == 0
    assert call(size, size, batch=1) == -1 and call(size - 8, size - 8, batch=1) == -1
    for other in (0, 8, size - 16, size - 4, size + 8):
        assert call(other, size + 8) == -1
