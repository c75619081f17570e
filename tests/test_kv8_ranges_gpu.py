"""Attention over the paged 8-bit KV cache for V far from 1, against 64 bits."""
import numpy as np
import pytest

import kv8ref
from kv8ref import E4M3, INT8
from test_kv8_gpu import Dev, no_device_error   # noqa: F401 (the fixture)

pytestmark = pytest.mark.gpu
KINDS = [INT8, E4M3]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens,new,g,width", [
    (40, 1, 1, 0), (50, 6, 2, 0), (2000, 1, 4, 0), (2000, 9, 1, 0), (30000, 1, 1, 0),   # one split, a cluster's, records
    (100, 30, 1, 0), (100, 30, 1, 520), (100, 60, 1, 520), (300, 100, 1, 520), (2000, 40, 1, 520)])   # pieces, tiles, split tiles
def test_outputs_next_to_the_largest_float(cuda, kind, tokens, new, g, width):
    """V within a factor of two of the largest float: an average of V is finite, a sum of two tokens is not."""
    rng = np.random.default_rng(tokens + new)
    hd, bs = 64, 16
    nb = -(-tokens // bs)
    d = Dev(cuda, kind, nb, bs, 1, hd, 1)
    d.ref.code[1][:] = kv8ref.encode(kv8ref.QMAX[kind] * np.sign(rng.uniform(-0.2, 1, d.ref.code[1].shape)), kind)
    d.ref.code[1][..., 0] = kv8ref.encode(kv8ref.QMAX[kind], kind)
    d.ref.scale[1][:] = 2.0 ** (120 if kind == INT8 else 118)
    for c in range(2):
        d.code[c].copy_(cuda.from_numpy(d.ref.code[c]))
        d.scale[c].copy_(cuda.from_numpy(d.ref.scale[c]))
    table = np.full((1, max(nb, width)), -1, np.int32)
    table[0, :nb] = np.arange(nb)
    q = rng.standard_normal((new, g, hd)).astype(np.float32)
    row0, pos = np.array([0, new]), np.array([tokens - new])
    got = d.attn(q, 0.1, table, row0, pos)
    want, bound = kv8ref.attention(d.ref, q, np.float32(0.1), table, row0, pos)
    assert np.all(np.isfinite(got))
    assert np.all(np.abs(got - want) <= bound)
