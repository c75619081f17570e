"""The paged 8-bit KV cache's host side, no GPU needed: refused arguments, the
workspace size, and the 64-bit restatement that the GPU tests compare with
(tests/kv8ref.py)."""
import ctypes

import numpy as np
import pytest

import kv8ref
import vxb200

PARAM, UNSUPPORTED = -4, -7
BUF = ctypes.addressof(ctypes.create_string_buffer(64)) & ~63   # an aligned address; never read


def cache(ctype=1, nb=4, bs=16, kh=2, hd=64, k=BUF, v=BUF, ks=BUF, vs=BUF):
    return vxb200.KV8(ctype, nb, bs, kh, hd, k, v, ks, vs)


def append(c, k=BUF, ldk=128, v=BUF, ldv=128, slot=BUF, n=1):
    return vxb200.lib().vxc_kv8_append(c.ref if c else None, k, ldk, v, ldv, slot, n, None)


def attn(c, q=BUF, ldq=256, h=4, scale=0.1, table=BUF, mb=2, row0=BUF, pos=BUF, n_req=1, n_rows=1, most=1, out=BUF,
         ldo=256, ws=BUF, wsb=1 << 40):
    return vxb200.lib().vxc_kv8_attn(c.ref if c else None, q, ldq, h, scale, table, mb, row0, pos, n_req, n_rows, most,
                                     out, ldo, ws, wsb, None)


def tables(length=BUF, new=BUF, n_req=1, bs=16, nb=4, mb=2, table=BUF, held=BUF, ring=BUF, state=BUF, n_rows=1,
           row0=BUF, slot=BUF):
    return vxb200.lib().vxc_kv8_tables(length, new, n_req, bs, nb, mb, table, held, ring, state, n_rows, row0, slot, None)


BAD_CACHES = [dict(ctype=0), dict(ctype=3), dict(nb=0), dict(nb=-1), dict(bs=0), dict(bs=8), dict(bs=40), dict(bs=272),
              dict(kh=0), dict(kh=65536), dict(hd=0), dict(hd=80), dict(hd=256), dict(k=None), dict(v=None),
              dict(ks=None), dict(vs=None), dict(k=BUF + 8), dict(v=BUF + 4), dict(ks=BUF + 2), dict(nb=1 << 28)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_bad_cache_is_refused(bad):
    c = cache(**bad)
    assert append(c) == PARAM
    assert b"vxc_kv8_append" in vxb200.lib().vxc_error_string()
    assert attn(c) == PARAM
    assert b"vxc_kv8_attn" in vxb200.lib().vxc_error_string()
    assert c.attn_workspace_bytes(4, 1, 1, 1, 2) == 0


def test_missing_cache_is_refused():
    assert append(None) == PARAM and attn(None) == PARAM


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(slot=None), dict(k=BUF + 4), dict(v=BUF + 8),
                                 dict(ldk=124), dict(ldv=0), dict(ldk=130), dict(n=-1), dict(n=(1 << 22) + 1)], ids=str)
def test_append_refusals(bad):
    assert append(cache(), **bad) == PARAM


@pytest.mark.parametrize("bad", [dict(h=0), dict(h=3), dict(h=-2), dict(h=65538), dict(q=None), dict(out=None),
                                 dict(table=None), dict(row0=None), dict(pos=None), dict(q=BUF + 4), dict(out=BUF + 8),
                                 dict(ldq=252), dict(ldo=100), dict(ldq=258), dict(n_req=0), dict(n_req=8193),
                                 dict(n_rows=-1), dict(n_rows=(1 << 22) + 1), dict(most=0), dict(mb=0), dict(mb=1 << 28),
                                 dict(n_rows=1 << 20, h=2048, ldq=1 << 20, ldo=1 << 20),
                                 dict(scale=float("nan")), dict(scale=float("inf"))], ids=str)
def test_attn_refusals(bad):
    assert attn(cache(), **bad) == PARAM


@pytest.mark.parametrize("bad", [dict(length=None), dict(new=None), dict(table=None), dict(held=None), dict(ring=None),
                                 dict(state=None), dict(row0=None), dict(slot=None), dict(n_req=0), dict(n_req=8193),
                                 dict(bs=0), dict(bs=24), dict(bs=512), dict(nb=0), dict(mb=0), dict(n_rows=-1),
                                 dict(nb=1 << 28), dict(mb=1 << 28)], ids=str)
def test_tables_refusals(bad):
    assert tables(**bad) == PARAM


@pytest.mark.parametrize("off", [1, 2, 3])
def test_misaligned_integer_arrays_are_refused(off):
    for name in ("length", "new", "table", "held", "ring", "state", "row0", "slot"):
        assert tables(**{name: BUF + off}) == PARAM, name
        assert b"vxc_kv8_tables" in vxb200.lib().vxc_error_string()
    assert append(cache(), slot=BUF + off) == PARAM
    for name in ("table", "row0", "pos"):
        assert attn(cache(), **{name: BUF + off}) == PARAM, name
        assert b"vxc_kv8_attn" in vxb200.lib().vxc_error_string()


def test_without_a_device_every_call_is_unsupported():
    if vxb200.lib().vxc_device_count() > 0:
        pytest.skip("a CUDA device is present")
    assert append(cache()) == UNSUPPORTED
    assert attn(cache()) == UNSUPPORTED
    assert tables() == UNSUPPORTED


def test_sequence_set_and_model_refusals():
    L = vxb200.lib()
    h = ctypes.c_void_p()
    assert L.vxc_seqs_create_kv8(None, 1, 64, 64, 1, 64, 0, ctypes.byref(h)) == PARAM
    for kind, nb in ((0, 0), (3, 0), (1, -1)):
        assert L.vxc_seqs_create_kv8(BUF, 1, 64, 64, kind, 64, nb, ctypes.byref(h)) == PARAM
    assert L.vx_model_set_kv_cache(None, 1) == PARAM


# ---- the restatement itself ---------------------------------------------------

def test_e4m3_codes_against_torch():
    torch = pytest.importorskip("torch")
    b = torch.arange(256, dtype=torch.uint8)
    want = b.view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(kv8ref.e4m3_value(b.numpy()), want)
    x = np.concatenate([np.linspace(-448, 448, 20001), np.linspace(-0.05, 0.05, 20001)]).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(kv8ref.encode(x, kv8ref.E4M3), want)


@pytest.mark.parametrize("kind", [1, 2])
def test_scale_is_the_smallest_power_of_two(kind):
    for a in [1e-44, 1e-38, 0.3, 1.0, 126.9, 127.0, 127.1, 254.0, 447.9, 448.0, 449.0, 3e38]:
        s = kv8ref.pow2_scale(float(np.float32(a)), kind)
        assert np.float32(a) <= kv8ref.QMAX[kind] * s
        assert s == 2.0 ** -126 or np.float32(a) > kv8ref.QMAX[kind] * s / 2


@pytest.mark.parametrize("kind", [1, 2])
def test_growing_scale_keeps_one_step(kind):
    """Token after token into one block, each larger than the last: an element is
    off by at most half a step of each scale it was rounded to, below one step of
    the last (int8); e4m3 by half a step of its own size for the first rounding
    and subnormal steps for the others."""
    rng = np.random.default_rng(0)
    c = kv8ref.Cache(kind, 1, 16, 1, 32)
    x = (rng.standard_normal((16, 1, 32)) * 2.0 ** np.arange(16)[:, None, None] / 64).astype(np.float32)
    for t in range(16):
        c.append(x[t:t + 1], x[t:t + 1], [t])
    k, _ = c.rows(np.array([0]), 16)
    s = float(c.scale[0][0, 0])
    step = s if kind == 1 else np.maximum(np.abs(x[:, 0]) * 2.0 ** -4, s * 2.0 ** -9)
    assert np.all(np.abs(k[0] - x[:, 0]) <= step)


def test_tables_restatement_conserves_blocks():
    rng = np.random.default_rng(1)
    n, bs, nb, mb = 5, 16, 40, 12
    table, held = np.full((n, mb), -1, np.int32), np.zeros(n, np.int32)
    ring, state = rng.permutation(nb).astype(np.int32), np.array([7, nb, 0], np.int32)
    for _ in range(50):
        length, new = rng.integers(0, 100, n), rng.integers(0, 60, n)
        kv8ref.tables(length, new, bs, nb, table, held, ring, state, 400)
        live = [b for r in range(n) for b in table[r, :held[r]]]
        free = [ring[(state[0] + i) % nb] for i in range(state[1])]
        assert sorted(live + free) == list(range(nb))
