"""Attention over the paged 8-bit KV cache where the scales of V are far apart,
far from 1 or zero, against a 64-bit evaluation with a purely relative bound."""
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


def reference(cache, q, scale, table, row0, pos):
    """(out, bound), float64.  kv8ref.attention's terms, relative to sum w |v|, without its absolute one, and
      - a weight below 2^-126 of the largest may be lost (fp32's normal range),
      - weights times V scales are held as two fp16 parts with 2^-25 as the error of the last one; the largest
        stands between 2^5 and 2^15, except that none is scaled up by more than 2^125,
      - 2^-148 per token where fp32 itself has no more digits."""
    rows, H, hd = q.shape
    G = H // cache.kh
    out, bound = np.zeros((rows, H, hd)), np.zeros((rows, H, hd))
    for r in range(len(pos)):
        total = int(pos[r]) + int(row0[r + 1] - row0[r])
        blocks = np.asarray(table[r, :-(-total // cache.bs)])
        k, v = cache.rows(blocks, total)
        vs = np.repeat(cache.scale[1][blocks].astype(np.float64), cache.bs, 0)[:total]
        for i in range(int(row0[r]), int(row0[r + 1])):
            n = int(pos[r]) + i - int(row0[r]) + 1
            for h in range(H):
                kk, vv, sv, qq = k[h // G][:n], v[h // G][:n], vs[:n, h // G], q[i, h].astype(np.float64)
                s = kk @ qq * scale
                size = np.abs(kk) @ np.abs(qq) * abs(scale)
                w = np.exp(s - s.max())
                top = np.maximum((w * sv).max() * 2.0 ** 5, 2.0 ** -115) / w.sum()
                lost = np.where(w < 2.0 ** -125, w, 0) / w.sum()
                w /= w.sum()
                out[i, h] = w @ vv
                d = (2.0 ** -22 + (hd / 16 + 20) * 2.0 ** -23) * size.max() + 4 * 2.0 ** -23 * np.abs(s).max()
                rel = np.expm1(2 * d) + 2.0 ** -20 + 2 * (n / 16 + 64) * 2.0 ** -23
                bound[i, h] = (rel * w + lost) @ np.abs(vv) + n * (448 * 2.0 ** -35 * top + 2.0 ** -148)
    return out, bound


def run(torch, kind, score, v_scale, new, hd=64, seed=0):
    """One request, blocks of 16 tokens: score[b] (integers) is the base 2 logarithm of the softmax weight
    of block b's tokens, v_scale[b] the scale of its V; the last `new` tokens are the rows."""
    rng = np.random.default_rng(seed)
    nb, bs = len(score), 16
    d = Dev(torch, kind, nb, bs, 1, hd, seed)
    d.ref.code[0][:] = 0
    d.ref.code[0][:, 0, :, 0] = kv8ref.encode(np.asarray(score, np.float64), kind)[:, None]
    d.ref.scale[0][:] = 1
    d.ref.scale[1][:, 0] = v_scale
    for c in range(2):
        d.code[c].copy_(torch.from_numpy(d.ref.code[c]))
        d.scale[c].copy_(torch.from_numpy(d.ref.scale[c]))
    q = np.zeros((new, 2, hd), np.float32)
    q[:, 0, 0], q[:, 1, 0] = 1.0, rng.uniform(0.5, 1, new)
    scale = np.float32(np.log(2))
    row0, pos = np.array([0, new]), np.array([nb * bs - new])
    want, bound = reference(d.ref, q, float(scale), np.arange(nb, dtype=np.int32)[None], row0, pos)
    # with over 8192 tokens in a row of the table all sizes above 16 queries go to k_kv8_attn_many
    for width in (nb, 520):
        table = np.full((1, width), -1, np.int32)
        table[0, :nb] = np.arange(nb)
        got = d.attn(q, float(scale), table, row0, pos)
        assert np.all(np.isfinite(got)), (width, np.argwhere(~np.isfinite(got))[:3])
        far = np.abs(got - want) - bound
        assert np.all(far <= 0), (width, float((far / bound).max()), np.unravel_index(np.argmax(far / bound), far.shape))
    return got


# two heads per kv head: up to 8 and 16 queries (k_kv8_attn_few), tiles of 32, 64 and 128 of them
ROWS = [1, 4, 8, 14, 30, 60]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", ROWS[1:])
@pytest.mark.parametrize("big", [2.0 ** 8, 2.0 ** 60, 2.0 ** 117])
def test_masked_tokens_with_large_v_behind_zero_v(cuda, kind, new, big):
    """The first rows see blocks whose V is all zero; blocks behind their position have any scale."""
    nb = (new + 15) // 16 + 1
    got = run(cuda, kind, [3] * nb, [0.0] + [big] * (nb - 1), new=16 * nb - 1 if new > 16 else new)
    assert got.size
    # every row of the first blocks sees zeros only
    zero = [0.0] * (nb - 1) + [big]
    got = run(cuda, kind, [3] * nb, zero, new=min(new + 16, 16 * nb))
    seen = min(new + 16, 16 * nb) - 16
    assert np.all(got[:seen] == 0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", ROWS)
@pytest.mark.parametrize("e", [-126, -120, -115, -111, -110, -100, 60, 110])
def test_v_scales_far_from_one(cuda, kind, new, e):
    run(cuda, kind, [3, 1, 0, 2, 4, 0, 1, 3], [2.0 ** e, 0.75 * 2.0 ** e] * 4, new=new)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", ROWS)
@pytest.mark.parametrize("gap", [30, 100, 108, 112, 116, 120, 124])
@pytest.mark.parametrize("order", [1, -1])
def test_v_is_zero_where_the_weights_are(cuda, kind, new, gap, order):
    """All but 2^-gap of the softmax falls on tokens whose V is zero: what is left is the output."""
    for low in (2.0 ** -20, 1.0, 2.0 ** 90):
        # (blocks 2 and 3, and 10 and 11, go to the same warp of k_kv8_attn_few)
        score = [0, 0, 120, 120 - gap, 0, 120 - gap, 0, 0, 0, 0, 120 - gap, 0][::order] + [0] * 4
        scale = [0.0, 0.0, 0.0, low, 0.0, 0.5 * low, 0.0, 0.0, 0.0, 0.0, low, 0.0][::order] + [0.0] * 4
        run(cuda, kind, score, scale, new=new)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", ROWS)
def test_v_scales_apart_by_any_power(cuda, kind, new):
    rng = np.random.default_rng(new)
    for seed in range(6):
        nb = int(rng.integers(5, 30))
        e = rng.integers(-126, 118, nb)
        score = rng.integers(-120, 120, nb) if seed % 2 else np.full(nb, 100) - rng.integers(0, 4, nb) * 36
        run(cuda, kind, score, np.where(rng.random(nb) < 0.2, 0, 2.0 ** e), new=new, hd=128 if seed % 3 else 32, seed=seed)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens,new,g,width", [(40, 1, 2, 0), (50, 6, 2, 0), (2000, 2, 4, 0), (30000, 1, 2, 0), (100, 30, 1, 0),
                                                (100, 30, 2, 520), (300, 100, 2, 520), (2000, 40, 1, 520)])
def test_nan_and_infinite_queries_stay_in_their_rows(cuda, kind, tokens, new, g, width):
    """A query with a NaN or an infinity gives a row of NaN, whatever path it takes; all others are as without it."""
    rng = np.random.default_rng(tokens)
    hd, bs = 64, 16
    nb = -(-tokens // bs)
    d = Dev(cuda, kind, nb, bs, 1, hd, 1)
    table = np.full((1, max(nb, width)), -1, np.int32)
    table[0, :nb] = np.arange(nb)
    q = rng.standard_normal((new, g, hd)).astype(np.float32)
    row0, pos = np.array([0, new]), np.array([tokens - new])
    want = d.attn(q, 0.1, table, row0, pos)
    for bad in (np.nan, np.inf):
        x = q.copy()
        x[new // 2, g - 1, 5] = bad
        got = d.attn(x, 0.1, table, row0, pos)
        hit = np.zeros((new, g), bool)
        hit[new // 2, g - 1] = True
        assert np.all(np.isnan(got[hit]))
        np.testing.assert_array_equal(got[~hit], want[~hit])
