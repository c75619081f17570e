"""The paged 8-bit KV cache on the GPU (vxc_kv8_tables, vxc_kv8_append,
vxc_kv8_attn) against its 64-bit restatement tests/kv8ref.py: tables, slots
and codes equal, attention within the bound kv8ref.attention derives."""
import ctypes

import numpy as np
import pytest

import kv8ref
from kv8ref import E4M3, INT8

pytestmark = pytest.mark.gpu

BAD_BLOCK, NONFINITE = 64, 128


def error_word():
    """Read and clear the device error word."""
    import vxb200
    code = ctypes.c_uint(0)
    vxb200.lib().vxc_check_device_error(ctypes.byref(code))
    return code.value


@pytest.fixture(autouse=True)
def no_device_error(cuda):
    error_word()
    yield
    assert error_word() == 0


class Dev:
    """A kv8ref.Cache and its copy on the device."""

    def __init__(self, torch, kind, nb, bs, kh, hd, seed=0, fill=True):
        import vxb200
        self.torch = torch
        self.ref = kv8ref.Cache(kind, nb, bs, kh, hd)
        rng = np.random.default_rng(seed)
        if fill:   # every byte, codes of what is nowhere live included
            for c in range(2):
                self.ref.code[c][:] = rng.integers(0, 256, self.ref.code[c].shape)
                if kind == E4M3:
                    self.ref.code[c][(self.ref.code[c] & 127) == 127] = 0x7E
                self.ref.scale[c][:] = 2.0 ** rng.integers(-9, -5, (nb, kh))
        self.code = [torch.from_numpy(x.copy()).cuda() for x in self.ref.code]
        self.scale = [torch.from_numpy(x.copy()).cuda() for x in self.ref.scale]
        self.c = vxb200.KV8(kind, nb, bs, kh, hd, self.code[0].data_ptr(), self.code[1].data_ptr(),
                            self.scale[0].data_ptr(), self.scale[1].data_ptr())

    def append(self, k, v, slot, on_device=None):
        """Both sides; k, v [n][kh][hd] numpy."""
        t = self.torch
        kd, vd = t.from_numpy(k).cuda(), t.from_numpy(v).cuda()
        sd = on_device if on_device is not None else t.from_numpy(np.asarray(slot, np.int32)).cuda()
        ld = self.ref.kh * self.ref.hd
        self.c.append(kd.data_ptr(), ld, vd.data_ptr(), ld, sd.data_ptr(), len(slot), t.cuda.current_stream().cuda_stream)
        t.cuda.synchronize()
        self.ref.append(k, v, slot)

    def same(self):
        for c in range(2):
            np.testing.assert_array_equal(self.scale[c].cpu().numpy(), self.ref.scale[c])
            got, want = self.code[c].cpu().numpy(), self.ref.code[c]
            if self.ref.kind == E4M3:   # -0 and 0 are one value
                got, want = np.where(got == 128, 0, got), np.where(want == 128, 0, want)
            np.testing.assert_array_equal(got, want)

    def attn(self, q, scale, table, row0, pos, n_rows=None, most=None, ld_pad=0, guard=3):
        """Device output rows (numpy), `guard` untouched rows of -7 behind the last."""
        t, H = self.torch, q.shape[1]
        n_rows = len(q) if n_rows is None else n_rows
        most = int(np.max(np.diff(row0), initial=1)) if most is None else most
        most = max(most, 1)
        width = H * self.ref.hd
        qd = t.full((len(q) + guard, width + ld_pad), float("nan"), device="cuda")
        qd[:len(q), :width] = t.from_numpy(q.reshape(len(q), -1)).cuda()
        out = t.full((len(q) + guard, width + 2 * ld_pad), -7.0, device="cuda")
        td, rd, pd = (t.from_numpy(np.ascontiguousarray(x, np.int32)).cuda() for x in (table, row0, pos))
        size = self.c.attn_workspace_bytes(H, len(pos), n_rows, most, table.shape[1])
        ws = t.full((size // 4 + 4,), float("nan"), device="cuda")   # nothing in it is initialised
        self.c.attn(qd.data_ptr(), qd.stride(0), H, scale, td.data_ptr(), table.shape[1], rd.data_ptr(), pd.data_ptr(),
                    len(pos), n_rows, most, out.data_ptr(), out.stride(0), ws.data_ptr(), size,
                    t.cuda.current_stream().cuda_stream)
        t.cuda.synchronize()
        got = out.cpu().numpy()
        assert np.all(got[len(q):] == -7.0) and np.all(got[:, width:] == -7.0)
        assert np.all(ws[size // 4:].isnan().cpu().numpy())
        return got[:len(q), :width].reshape(q.shape)


def paged(rng, totals, bs, extra=2):
    """A table of shuffled blocks that holds `totals` tokens per request, -1 behind them."""
    need = [-(-t // bs) if t > 0 else 0 for t in totals]
    nb = sum(need) + extra
    order = rng.permutation(nb).astype(np.int32)
    table = np.full((len(totals), max(need + [1]) + 1), -1, np.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    return table, nb


def check_attn(torch, kind, hd, kh, g, bs, lens, new, seed=0, scale=None, **kw):
    """Ragged requests: lens cached tokens before, `new` rows each."""
    rng = np.random.default_rng(seed)
    totals = [a + b for a, b in zip(lens, new)]
    table, nb = paged(rng, totals, bs)
    d = Dev(torch, kind, nb, bs, kh, hd, seed)
    row0 = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = rng.standard_normal((row0[-1], kh * g, hd)).astype(np.float32)
    scale = 1 / np.sqrt(hd) if scale is None else scale
    got = d.attn(q, scale, table, row0, lens, **kw)
    want, bound = kv8ref.attention(d.ref, q, np.float32(scale), table, row0, lens)
    far = np.abs(got - want) - bound   # rows without tokens: 0, exactly
    assert np.all(far <= 0), (float(far.max()), np.unravel_index(np.argmax(far), far.shape))
    return d


# ---- attention ------------------------------------------------------------------

@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("g", [1, 3, 8])
def test_attn_decode(cuda, kind, hd, g):
    check_attn(cuda, kind, hd, 2, g, 16, [0, 1, 15, 16, 31, 200, 517], [1] * 7)


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("bs", [16, 48, 64, 256])
def test_attn_block_sizes(cuda, kind, bs):
    check_attn(cuda, kind, 128, 1, 4, bs, [0, 63, 64, 255, 300], [2, 1, 3, 5, 1])


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("hd,kh,g,new", [(128, 2, 1, 5), (128, 1, 8, 7), (64, 1, 8, 2), (64, 3, 5, 4), (96, 2, 2, 9),
                                         (32, 1, 4, 16), (128, 1, 16, 1), (128, 1, 24, 1), (64, 1, 33, 2),
                                         (128, 1, 7, 9), (96, 1, 64, 1)])
def test_attn_verify(cuda, kind, hd, kh, g, new):
    check_attn(cuda, kind, hd, kh, g, 32, [0, 100, 301], [new, max(1, new - 1), new])


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("hd,kh,g,lens,new", [(128, 1, 1, [0, 0, 5], [130, 64, 200]), (128, 1, 4, [0, 70], [33, 65]),
                                              (64, 2, 8, [0, 250], [128, 17]), (96, 1, 3, [40], [129]),
                                              (32, 1, 2, [0, 700], [257, 64]), (128, 1, 16, [300], [40]),
                                              (64, 1, 5, [3, 0, 1000], [1, 100, 26]), (128, 2, 2, [511], [513])])
def test_attn_prompt(cuda, kind, hd, kh, g, lens, new):
    check_attn(cuda, kind, hd, kh, g, 64, lens, new)


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("g,new", [(1, 16), (1, 17), (3, 8), (1, 32), (3, 11), (8, 7), (8, 8), (5, 13), (1, 127), (16, 8), (3, 43)])
def test_attn_around_the_tile_sizes(cuda, kind, hd, g, new):
    """16, 32, 64 and 128 queries per kv head, one less and a few more; requests of fewer rows."""
    check_attn(cuda, kind, hd, 2, g, 48, [0, 3, 90, 333], [new, 1, new - 1, new])


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("hd,g,new", [(128, 8, 1), (64, 4, 3), (128, 1, 1), (128, 2, 70), (128, 2, 13), (96, 8, 7)])
def test_attn_long_context_is_split_and_joined(cuda, kind, hd, g, new):
    check_attn(cuda, kind, hd, 1, g, 64, [5000, 0, 2047], [new, new, new])


def test_attn_context_of_over_half_a_million_tokens(cuda):
    """More than 64 splits of 8192 tokens."""
    check_attn(cuda, INT8, 32, 1, 2, 256, [600000, 40], [1, 1])
    check_attn(cuda, E4M3, 32, 1, 1, 256, [550000], [33])


def test_attn_many_requests(cuda):
    rng = np.random.default_rng(3)
    check_attn(cuda, INT8, 64, 2, 2, 16, rng.integers(0, 70, 300).tolist(), rng.integers(0, 3, 300).tolist())
    # begun by length: equal ones and a long one, 128 requests and one more
    for n, kh, new in ((128, 4, 1), (129, 4, 1), (80, 4, 20), (129, 4, 20), (5, 80, 1), (5, 60, 9)):
        lens = rng.integers(0, 4, n)
        lens[n // 2] = 600
        check_attn(cuda, INT8, 32, kh, 3, 16, lens.tolist(), [new] * n)
    # prompts of few tokens: their queries in pieces of 16
    for kind, hd, g, most in ((INT8, 32, 1, 26), (E4M3, 64, 3, 40), (INT8, 32, 5, 30), (E4M3, 32, 16, 9)):
        new = rng.integers(0, most + 1, 90)
        new[0] = most
        check_attn(cuda, kind, hd, 24, g, 16, rng.integers(0, 20, 90).tolist(), new.tolist())
        check_attn(cuda, kind, hd, 24, g, 16, rng.integers(-9, 3, 90).tolist(), np.maximum(new, 10).tolist())


def test_attn_requests_without_rows_and_rows_without_tokens(cuda):
    # request 1 has no rows, request 2 sees nothing (negative positions up to 0), request 4 none at all
    d = check_attn(cuda, INT8, 128, 1, 2, 16, [3, 10, -3, 20, -2], [2, 0, 4, 1, 2])
    rng = np.random.default_rng(0)
    q = rng.standard_normal((3, 2, 128)).astype(np.float32)
    got = d.attn(q, 0.1, np.zeros((1, 2), np.int32), np.array([0, 3]), np.array([-2]))
    assert np.all(got[:2] == 0) and np.any(got[2] != 0)


@pytest.mark.parametrize("hd,new", [(128, 1), (64, 5), (128, 80), (128, 11), (96, 25), (32, 31)])
def test_attn_strides_and_spare_rows(cuda, hd, new):
    check_attn(cuda, E4M3, hd, 2, 2, 32, [50, 7], [new, new], ld_pad=12)
    # the caller's n_rows and max_new are upper bounds
    check_attn(cuda, E4M3, hd, 2, 2, 32, [50, 7], [new, new], n_rows=2 * new + 3, most=new + 11)


@pytest.mark.parametrize("new", [1, 6, 14, 90])
def test_attn_bytes_behind_the_last_token_are_not_used(cuda, new):
    torch = cuda
    rng = np.random.default_rng(5)
    lens, bs = [37, 3], 64
    table, nb = paged(rng, [a + new for a in lens], bs)
    d = Dev(torch, E4M3, nb, bs, 1, 128, 1)
    row0 = np.array([0, new, 2 * new])
    q = rng.standard_normal((2 * new, 4, 128)).astype(np.float32)
    want = d.attn(q, 0.09, table, row0, lens)
    for r, a in enumerate(lens):   # NaN codes from the first token behind the request's last on
        last = table[r, (a + new - 1) // bs]
        for c in d.code:
            c[last, :, (a + new - 1) % bs + 1:] = 0x7F
    free = sorted(set(range(nb)) - set(table.ravel().tolist()))
    for c in range(2):
        d.code[c][free] = 0xFF
        d.scale[c][free] = float("nan")
    np.testing.assert_array_equal(d.attn(q, 0.09, table, row0, lens), want)


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("new", [1, 5, 14, 70])
def test_attn_scales_of_any_size(cuda, kind, new):
    """Blocks whose scales are far apart, zero among them, and far from 1; queries far from 1."""
    torch = cuda
    rng = np.random.default_rng(11)
    bs, hd, lens = 16, 128, [150]
    table, nb = paged(rng, [150 + new], bs)
    d = Dev(torch, kind, nb, bs, 1, hd, 2)
    d.ref.scale[0][:, 0] = 2.0 ** rng.integers(-30, -24, nb)
    d.ref.scale[1][:, 0] = 2.0 ** rng.integers(-12, 13, nb) * (rng.random(nb) < 0.8) * rng.uniform(0.5, 1, nb)
    for c in range(2):
        d.scale[c].copy_(torch.from_numpy(d.ref.scale[c]))
    q = (rng.standard_normal((new, 4, hd)) * 2.0 ** 20).astype(np.float32)
    q[:, 1] *= 1e-6   # a head of its own size, one of zeros
    q[:, 2] = 0
    got = d.attn(q, 0.05, table, np.array([0, new]), lens)
    want, bound = kv8ref.attention(d.ref, q, np.float32(0.05), table, np.array([0, new]), lens)
    # a weight is split with 2^-24 / 2^14 of the largest weight x scale as its last place
    assert np.all(np.abs(got - want) <= bound + 2.0 ** -30 * np.abs(want).max())


@pytest.mark.parametrize("new", [1, 4, 12, 30, 66])
def test_attn_bad_table_entries_are_masked_and_reported(cuda, new):
    rng = np.random.default_rng(2)
    table, nb = paged(rng, [90 + new, 20 + new], 16)
    d = Dev(cuda, INT8, nb, 16, 1, 64, 3)
    table[0, 2], table[0, 4], table[1, 0] = nb, -5, 1 << 30
    row0 = np.array([0, new, 2 * new])
    q = rng.standard_normal((2 * new, 2, 64)).astype(np.float32)
    got = d.attn(q, 0.125, table, row0, [90, 20])
    assert error_word() == BAD_BLOCK
    want, bound = kv8ref.attention(d.ref, q, 0.125, table, row0, [90, 20])
    assert np.all(np.abs(got - want) <= bound)


@pytest.mark.parametrize("new", [2, 12, 30, 70])
def test_attn_lengths_beyond_the_arguments_are_reported(cuda, new):
    rng = np.random.default_rng(2)
    table, nb = paged(rng, [100 + new], 16)
    d = Dev(cuda, INT8, nb, 16, 1, 64, 3)
    q = rng.standard_normal((new, 2, 64)).astype(np.float32)
    # behind the table: these rows are left as they were
    got = d.attn(q, 0.125, table, np.array([0, new]), [table.shape[1] * 16 - 1])
    assert error_word() == BAD_BLOCK
    assert np.all(got[1:] == -7) and np.all(got[0] != -7)
    # more rows than max_new
    got = d.attn(q, 0.125, table, np.array([0, new]), [100], most=new - 1)
    assert error_word() == BAD_BLOCK
    want, bound = kv8ref.attention(d.ref, q, 0.125, table, np.array([0, new]), [100])
    assert np.all(np.abs(got - want)[:new - 1] <= bound[:new - 1]) and np.all(got[new - 1] == -7)
    # more rows than n_rows
    got = d.attn(q, 0.125, table, np.array([0, new]), [100], n_rows=new - 1)
    assert error_word() == BAD_BLOCK
    assert np.all(np.abs(got - want)[:new - 1] <= bound[:new - 1]) and np.all(got[new - 1] == -7)
    # a position next to the largest int
    got = d.attn(q, 0.125, table, np.array([0, new]), [2 ** 31 - 1])
    assert error_word() == BAD_BLOCK and np.all(got == -7)


def test_attn_workspace_too_small_is_refused(cuda):
    import vxb200
    d = Dev(cuda, INT8, 70, 64, 1, 128)
    size = d.c.attn_workspace_bytes(8, 1, 1, 1, 400)
    assert size > 0
    x = cuda.zeros(4096, device="cuda")
    p = x.data_ptr()
    for ws, n in ((p, size - 1), (None, size)):
        rc = vxb200.lib().vxc_kv8_attn(d.c.ref, p, 1024, 8, 0.1, p, 400, p, p, 1, 1, 1, p, 1024, ws, n, None)
        assert rc == -4 and b"workspace" in vxb200.lib().vxc_error_string()


def test_attn_offsets_beyond_32_bits(cuda):
    """A cache of over 4 GiB of K: blocks near its end."""
    torch = cuda
    import vxb200
    kh, bs, hd = 8, 64, 128
    nb = (1 << 32) // (kh * bs * hd) + 40
    k = torch.zeros(nb * kh * bs * hd, dtype=torch.uint8, device="cuda")
    v = torch.zeros_like(k)
    ks, vs = (torch.zeros(nb * kh, device="cuda") for _ in range(2))
    c = vxb200.KV8(INT8, nb, bs, kh, hd, k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr())
    rng = np.random.default_rng(0)
    blocks = np.array([nb - 1, 3, nb - 2, nb // 2], np.int32)
    small = Dev(torch, INT8, 4, bs, kh, hd, fill=False)
    n = 200
    x = rng.standard_normal((2, n, kh, hd)).astype(np.float32)
    p = np.arange(n)
    small.append(x[0], x[1], p)
    xd = torch.from_numpy(x).cuda()
    sd = torch.from_numpy((blocks[p // bs].astype(np.int64) * bs + p % bs).astype(np.int32)).cuda()
    st = torch.cuda.current_stream().cuda_stream
    c.append(xd[0].data_ptr(), kh * hd, xd[1].data_ptr(), kh * hd, sd.data_ptr(), n, st)
    big = k.view(nb, -1)[torch.from_numpy(blocks).long()].cpu().numpy().reshape(small.ref.code[0].shape)
    np.testing.assert_array_equal(big, small.ref.code[0])
    q = rng.standard_normal((1, 16, hd)).astype(np.float32)
    want = small.attn(q, 0.1, np.arange(4, dtype=np.int32)[None], np.array([0, 1]), [n - 1])
    small.c = c
    got = small.attn(q, 0.1, blocks[None], np.array([0, 1]), [n - 1])
    np.testing.assert_array_equal(got, want)


# ---- append ---------------------------------------------------------------------

@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("hd,kh,bs", [(32, 3, 16), (64, 1, 48), (96, 2, 32), (128, 2, 64), (128, 1, 256)])
def test_append_prompt_then_tokens(cuda, kind, hd, kh, bs):
    """A prompt into fresh blocks, then rows of growing and shrinking size one or a few at a time."""
    rng = np.random.default_rng(hd + bs)
    d = Dev(cuda, kind, 6, bs, kh, hd, seed=1)
    blocks = np.array([4, 1, 3, 0])
    p = 0
    for n, size in ((bs + 3, 1.0), (1, 0.1), (1, 30.0), (2, 1e-3), (bs - 5, 2.0), (1, 5e4), (3, 1.0)):
        x = (rng.standard_normal((2, n, kh, hd)) * size).astype(np.float32)
        at = np.arange(p, p + n)
        d.append(x[0], x[1], blocks[at // bs] * bs + at % bs)
        d.same()
        p += n
    # the last three are dropped and written again (a rejected draft)
    at = np.arange(p - 3, p)
    x = rng.standard_normal((2, 3, kh, hd)).astype(np.float32)
    d.append(x[0], x[1], blocks[at // bs] * bs + at % bs)
    d.same()


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("n_req,new", [(40, 1), (9, 7), (3, 400), (2, 700)])
def test_append_many_requests(cuda, kind, n_req, new):
    """Requests at their own places of their blocks; from 513 rows on a CTA goes over several of them."""
    rng = np.random.default_rng(n_req)
    bs, kh, hd = 32, 2, 64
    lens = rng.integers(0, 50, n_req)
    table, nb = paged(rng, lens + new, bs)
    d = Dev(cuda, kind, nb, bs, kh, hd, seed=2)
    slot = np.concatenate([table[r, np.arange(a, a + new) // bs] * bs + np.arange(a, a + new) % bs
                           for r, a in enumerate(lens)])
    x = (rng.standard_normal((2, len(slot), kh, hd)) * 2.0 ** rng.integers(-3, 6, (1, len(slot), 1, 1))).astype(np.float32)
    d.append(x[0], x[1], slot)
    d.same()


@pytest.mark.parametrize("kind", [INT8, E4M3])
def test_append_values_at_the_edges(cuda, kind):
    """Ties, largest codes, zeros, subnormals, the largest floats, and rows that are all zero."""
    d = Dev(cuda, kind, 8, 16, 1, 32, fill=False)
    top = kv8ref.QMAX[kind]
    x = np.zeros((8, 16, 1, 32), np.float32)
    x[0, :, 0] = np.arange(512).reshape(16, 32) / 4 - 64          # ties at halves
    x[0, 0, 0, 0] = top
    x[1, 0, 0, :4] = [1e-45, -1e-40, 2.0 ** -126, 0]
    x[2, 0, 0, :3] = [3.4028235e38, -3.4028235e38, 1]
    x[4, 0, 0, :2] = [np.nextafter(np.float32(top), np.float32(1e9)), 1]
    x[5, 0, 0, :2] = [-top / 64, top / 128]
    x[6, :, 0] = (np.random.default_rng(0).standard_normal((16, 32)) * 1e-3).astype(np.float32)
    x[6, 3, 0, 0] = 1.0
    x[7, :, 0] = -0.0
    for b in range(8):
        d.append(x[b], np.float32(0.75) * x[7 - b], np.arange(16) + 16 * b)   # 0.75: no overflow
    d.same()
    y = np.full((1, 1, 32), 0.5, np.float32)   # into a block whose scale is 0
    d.append(y, y, [16 * 3 + 5])
    d.same()


@pytest.mark.parametrize("kind", [INT8, E4M3])
def test_append_nonfinite_elements_are_zero_and_reported(cuda, kind):
    rng = np.random.default_rng(0)
    d = Dev(cuda, kind, 3, 16, 2, 64)
    x = rng.standard_normal((2, 20, 2, 64)).astype(np.float32)
    x[0, 3, 1, 5], x[0, 4, 0, 0], x[1, 19, 1, 63] = np.nan, np.inf, -np.inf
    d.append(x[0], x[1], np.arange(20))
    assert error_word() == NONFINITE
    d.same()


@pytest.mark.parametrize("n", [40, 600])
def test_append_skipped_rows_bad_slots_and_slots_twice(cuda, n):
    rng = np.random.default_rng(n)
    bs, nb = 16, 64
    d = Dev(cuda, INT8, nb, bs, 2, 64, seed=4)
    slot = np.full(n, -1, np.int32)
    slot[1:8] = 32 + np.arange(7)
    slot[8:20] = 5 * bs + np.array([3, 4, 3, 3, 5, 6, 7, 4, 8, 9, 15, 3])   # one block, slots twice and more
    slot[25:30] = 9 * bs + np.arange(11, 16)
    slot[30:33] = 10 * bs + np.arange(3)
    x = rng.standard_normal((2, n, 2, 64)).astype(np.float32)
    x[:, 10] *= 50
    d.append(x[0], x[1], slot)
    d.same()
    slot[:] = -1
    slot[3], slot[5], slot[7] = nb * bs, 2 ** 31 - 1, -2
    slot[9:12] = 7 + np.arange(3)
    d.append(x[0], x[1], slot)
    assert error_word() == BAD_BLOCK
    d.same()


def test_append_rows_with_strides(cuda):
    torch = cuda
    rng = np.random.default_rng(0)
    d = Dev(torch, E4M3, 3, 16, 2, 32, seed=4)
    qkv = torch.from_numpy(rng.standard_normal((20, 4 * 32 + 2 * 64 + 4)).astype(np.float32)).cuda()   # q, k, v side by side
    slot = torch.arange(20, dtype=torch.int32, device="cuda")
    ld = qkv.stride(0)
    d.c.append(qkv.data_ptr() + 4 * 128, ld, qkv.data_ptr() + 4 * 192, ld, slot.data_ptr(), 20,
               torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    x = qkv.cpu().numpy()
    d.ref.append(x[:, 128:192].reshape(20, 2, 32), x[:, 192:256].reshape(20, 2, 32), np.arange(20))
    d.same()
    d.c.append(0, 0, 0, 0, 0, 0)   # no rows: nothing to do


# ---- tables ---------------------------------------------------------------------

class Tables:
    def __init__(self, torch, n, bs, nb, mb, front=0, seed=0):
        rng = np.random.default_rng(seed)
        self.torch, self.n, self.bs, self.nb, self.mb = torch, n, bs, nb, mb
        self.ref = [np.full((n, mb), -1, np.int32), np.zeros(n, np.int32), rng.permutation(nb).astype(np.int32),
                    np.array([front, nb, 0], np.int32)]
        self.dev = [torch.from_numpy(x.copy()).cuda() for x in self.ref]

    def step(self, length, new, n_rows):
        import vxb200
        t = self.torch
        ld, nd = (t.from_numpy(np.asarray(x, np.int32)).cuda() for x in (length, new))
        row0 = t.full((self.n + 3,), -9, dtype=t.int32, device="cuda")
        slot = t.full((n_rows + 2,), -9, dtype=t.int32, device="cuda")
        vxb200.kv8_tables(ld.data_ptr(), nd.data_ptr(), self.n, self.bs, self.nb, self.mb, *(x.data_ptr() for x in self.dev),
                          n_rows, row0.data_ptr(), slot.data_ptr(), t.cuda.current_stream().cuda_stream)
        t.cuda.synchronize()
        want = kv8ref.tables(length, new, self.bs, self.nb, *self.ref, n_rows)
        np.testing.assert_array_equal(row0.cpu().numpy(), list(want[0]) + [-9, -9])
        np.testing.assert_array_equal(slot.cpu().numpy(), list(want[1]) + [-9, -9])
        for a, b in zip(self.dev, self.ref):
            np.testing.assert_array_equal(a.cpu().numpy(), b)
        return int(self.ref[3][2])


@pytest.mark.parametrize("n,bs,nb,mb,most,rows", [(1, 16, 10, 10, 100, 200), (7, 16, 60, 12, 60, 500),
                                                  (33, 48, 90, 9, 90, 3000), (1500, 32, 4000, 4, 30, 70000),
                                                  (40, 16, 2600, 100, 600, 30000), (8192, 16, 20000, 4, 5, 50000)])
def test_tables_random_steps(cuda, n, bs, nb, mb, most, rows):
    """Lengths that grow, shrink and end; some steps find too few free blocks."""
    rng = np.random.default_rng(n)
    T = Tables(cuda, n, bs, nb, mb, front=nb - 1, seed=n)
    seen = set()
    length = np.zeros(n, np.int64)
    for step in range(12):
        new = rng.integers(0, most + 1, n) * (rng.random(n) < 0.6)
        new = np.minimum(new, mb * bs - length)
        while new.sum() > rows:
            new = new // 2
        status = T.step(length, new, rows)
        seen.add(status)
        if status == 0:
            length = length + new
        u = rng.random(n)
        length = np.where(u < (0.2 if status == 0 else 0.7), 0, np.where(u < 0.8, length * rng.random(n), length)).astype(np.int64)
    assert 0 in seen


def test_tables_refused_calls_change_nothing(cuda):
    T = Tables(cuda, 3, 16, 8, 6, front=5)
    assert T.step([0, 0, 0], [40, 20, 0], 60) == 0
    assert T.step([40, 20, 0], [0, 0, 64], 64) == 1       # 4 blocks, 3 free
    assert error_word() == 0
    assert T.step([40, 20, 0], [0, 0, 97], 200) == 2      # 7 blocks of 6
    assert error_word() == BAD_BLOCK
    for length, new in (([40, -1, 0], [0, 0, 0]), ([40, 20, 0], [0, -7, 0]), ([40, 20, 0], [10, 10, 10])):
        assert T.step(length, new, 29) == 3               # negative; 30 rows of 29
        assert error_word() == BAD_BLOCK
    assert T.step([40, 20, 0], [1, 1, 30], 40) == 0
    for i, bad in ((3, [8, 1, 0]), (3, [-1, 1, 0]), (3, [0, -1, 0]), (3, [0, 9, 0]), (1, [1, 2, 7]), (1, [-1, 0, 0])):
        B = Tables(cuda, 3, 16, 8, 6)
        for side in (B.ref, B.dev):
            side[i][:len(bad)] = cuda.tensor(bad, dtype=cuda.int32).to(side[i].device) if side is B.dev else bad
        before = [x.clone() for x in B.dev]
        import vxb200
        z = cuda.zeros(3, dtype=cuda.int32, device="cuda")
        out = cuda.zeros(8, dtype=cuda.int32, device="cuda")
        vxb200.kv8_tables(z.data_ptr(), z.data_ptr(), 3, 16, 8, 6, *(x.data_ptr() for x in B.dev), 2, out.data_ptr(),
                          out.data_ptr() + 16)
        assert error_word() == BAD_BLOCK
        before[3][2] = 3
        for a, b in zip(B.dev, before):
            assert cuda.equal(a, b), (i, bad)


def test_tables_blocks_outside_the_cache_are_reported(cuda):
    """From the queue, and in a table: their tokens have no slot."""
    import vxb200
    for i, at, bad in ((2, 6, 8), (2, 6, -3), (0, (1, 0), 99)):
        T = Tables(cuda, 2, 16, 8, 4, front=5)   # 4 blocks to the first step: ring entries 5, 6, 7, 0
        if i == 0:
            assert T.step([0, 0], [20, 20], 40) == 0
        T.dev[i][at] = bad
        length, new = ([0, 0], [20, 20]) if i == 2 else ([20, 20], [4, 4])
        ld, nd = (cuda.tensor(x, dtype=cuda.int32, device="cuda") for x in (length, new))
        row0, slot = (cuda.full((n,), -9, dtype=cuda.int32, device="cuda") for n in (3, 40))
        vxb200.kv8_tables(ld.data_ptr(), nd.data_ptr(), 2, 16, 8, 4, *(x.data_ptr() for x in T.dev), 40,
                          row0.data_ptr(), slot.data_ptr())
        want = kv8ref.tables(length, new, 16, 8, *T.ref, 40)
        got = slot.cpu().numpy()
        assert int(T.dev[3][2]) == 0 and np.array_equal(row0.cpu().numpy(), want[0])
        if i == 2:   # the second block taken: the first request's tokens 16 to 19
            assert error_word() == BAD_BLOCK
            assert np.all(got[16:20] == -1)
            keep = np.r_[0:16, 20:40]
            np.testing.assert_array_equal(got[keep], want[1][keep])
        else:        # the second request's first block holds none of its new tokens 20 to 23
            np.testing.assert_array_equal(got, want[1])
            T.dev[0][1, 1] = bad
            vxb200.kv8_tables(ld.data_ptr(), nd.data_ptr(), 2, 16, 8, 4, *(x.data_ptr() for x in T.dev), 40,
                              row0.data_ptr(), slot.data_ptr())
            assert error_word() == BAD_BLOCK
            got = slot.cpu().numpy()
            assert np.all(got[4:8] == -1)
            np.testing.assert_array_equal(got[:4], want[1][:4])


# ---- together ---------------------------------------------------------------------

@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("graph", [False, True])
def test_tables_append_attention_together(cuda, kind, graph):
    """A server's loop on one stream: prompts admitted, verify steps with rejected
    tokens, a request that ends and another in its place; eager or as one
    captured graph replayed for every step."""
    torch = cuda
    import vxb200
    rng = np.random.default_rng(9)
    n, bs, nb, mb, kh, g, hd, rows = 4, 16, 60, 20, 2, 4, 64, 270
    d = Dev(torch, kind, nb, bs, kh, hd, fill=False)
    T = Tables(torch, n, bs, nb, mb, front=50)
    H = kh * g
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        ld, nd = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2))
        row0 = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
        slot = torch.zeros(rows, dtype=torch.int32, device="cuda")
        qkv = torch.zeros(rows, (H + 2 * kh) * hd, device="cuda")
        out = torch.full((rows, H * hd), -7.0, device="cuda")
        most = 128
        size = d.c.attn_workspace_bytes(H, n, rows, most, mb)
        ws = torch.empty(size // 4 + 4, device="cuda")
    scale = 1 / np.sqrt(hd)

    def step():
        w = qkv.stride(0)
        q = qkv.data_ptr()
        vxb200.kv8_tables(ld.data_ptr(), nd.data_ptr(), n, bs, nb, mb, *(x.data_ptr() for x in T.dev), rows,
                          row0.data_ptr(), slot.data_ptr(), st.cuda_stream)
        d.c.append(q + 4 * H * hd, w, q + 4 * (H + kh) * hd, w, slot.data_ptr(), rows, st.cuda_stream)
        d.c.attn(q, w, H, scale, T.dev[0].data_ptr(), mb, row0.data_ptr(), ld.data_ptr(), n, rows, most, out.data_ptr(),
                 H * hd, ws.data_ptr(), size, st.cuda_stream)

    run = step
    if graph:
        with torch.cuda.stream(st):
            step()   # no new rows yet
        st.synchronize()
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg, stream=st):
            step()
        run = cg.replay
    length = np.zeros(n, np.int64)
    plan = [[100, 33, 0, 128], [5, 5, 0, 5], [5, 5, 60, 5], [1, 1, 1, 1], [0, 0, 0, 0], [5, 5, 5, 5], [120, 5, 5, 5]]
    for k, new in enumerate(plan):
        if k in (3, 5):
            length = np.maximum(0, length - 3)   # rejected tokens
        if k == 6:
            length[0] = 0                        # another request in its place
        new = np.array(new)
        m = int(new.sum())
        x = rng.standard_normal((rows, H + 2 * kh, hd)).astype(np.float32)
        with torch.cuda.stream(st):
            ld.copy_(torch.from_numpy(length.astype(np.int32)))
            nd.copy_(torch.from_numpy(new.astype(np.int32)))
            qkv.copy_(torch.from_numpy(x.reshape(rows, -1)))
            out.fill_(-7.0)
            run()
        st.synchronize()
        r0, sl = kv8ref.tables(length, new, bs, nb, *T.ref, rows)
        assert T.ref[3][2] == 0
        np.testing.assert_array_equal(slot.cpu().numpy(), sl)
        np.testing.assert_array_equal(T.dev[0].cpu().numpy(), T.ref[0])
        d.ref.append(x[:, H:H + kh], x[:, H + kh:], sl)
        d.same()
        want, bound = kv8ref.attention(d.ref, x[:m, :H], np.float32(scale), T.ref[0], r0, length)
        got = out.cpu().numpy()
        assert np.all(np.abs(got[:m].reshape(want.shape) - want) <= bound)
        assert np.all(got[m:] == -7)
        length = length + new
    if graph:
        del cg


def test_two_calls_at_once_on_two_streams(cuda):
    """Two caches, two workspaces, two streams: the results are those of each alone."""
    torch = cuda
    rng = np.random.default_rng(1)
    ds, want, args = [], [], []
    for s in range(2):
        table, nb = paged(rng, [3000, 900], 64)
        d = Dev(torch, INT8, nb, 64, 2, 128, seed=s)
        q = rng.standard_normal((2, 8, 128)).astype(np.float32)
        lens = np.array([2999, 899], np.int32)
        want.append(d.attn(q, 0.1, table, np.array([0, 1, 2]), lens))
        size = d.c.attn_workspace_bytes(8, 2, 2, 1, table.shape[1])
        t = [torch.from_numpy(x).cuda() for x in (q.reshape(2, -1), table, np.array([0, 1, 2], np.int32), lens)]
        args.append((d, t, torch.empty(size // 4 + 4, device="cuda"), size, torch.zeros(2, 1024, device="cuda"),
                     torch.cuda.Stream(), table.shape[1]))
        ds.append(d)
    torch.cuda.synchronize()
    for _ in range(20):
        for d, t, ws, size, out, st, mb in args:
            d.c.attn(t[0].data_ptr(), 1024, 8, 0.1, t[1].data_ptr(), mb, t[2].data_ptr(), t[3].data_ptr(), 2, 2, 1,
                     out.data_ptr(), 1024, ws.data_ptr(), size, st.cuda_stream)
    torch.cuda.synchronize()
    for w, a in zip(want, args):
        np.testing.assert_array_equal(a[4].cpu().numpy().reshape(w.shape), w)


@pytest.mark.parametrize("new", [1, 40])
def test_two_calls_at_once_with_records_of_splits(cuda, new):
    """As above with contexts whose splits meet in the workspaces: over 8 splits of a few queries, split tiles."""
    torch = cuda
    rng = np.random.default_rng(new)
    runs = []
    for s in range(2):
        lens = np.array([25600 - new], np.int32)
        table, nb = paged(rng, lens + new, 64)
        d = Dev(torch, E4M3, nb, 64, 1, 64, seed=s)
        q = rng.standard_normal((new, 2, 64)).astype(np.float32)
        row0 = np.array([0, new], np.int32)
        want = d.attn(q, 0.1, table, row0, lens)
        size = d.c.attn_workspace_bytes(2, 1, new, new, table.shape[1])
        assert size > 0
        t = [torch.from_numpy(x).cuda() for x in (q.reshape(new, -1), table, row0, lens)]
        runs.append((d, t, torch.empty(size // 4 + 4, device="cuda"), size, torch.zeros(new, 128, device="cuda"),
                     torch.cuda.Stream(), want, table.shape[1]))
    torch.cuda.synchronize()
    for _ in range(20):
        for d, t, ws, size, out, st, want, mb in runs:
            d.c.attn(t[0].data_ptr(), 128, 2, 0.1, t[1].data_ptr(), mb, t[2].data_ptr(), t[3].data_ptr(), 1, new, new,
                     out.data_ptr(), 128, ws.data_ptr(), size, st.cuda_stream)
    torch.cuda.synchronize()
    for d, t, ws, size, out, st, want, mb in runs:
        np.testing.assert_array_equal(out.cpu().numpy().reshape(want.shape), want)
