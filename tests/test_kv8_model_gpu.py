"""The forward over the paged 8-bit KV cache (vxc_seqs_create_kv8,
vx_model_set_kv_cache) on the GPU.

Logits are compared with a float64 forward whose K and V pass through the
64-bit restatement of the cache (tests/kv8_emulation.py) at the repository's
tolerance for logits, 2e-3 x max|logit|: the forward itself is within about
1e-5 of it, and an element of K or V that the two round to neighbouring codes
(its fp32 value lies on the border between them) moves the logits by far less
than the rounding of the whole cache, about 1e-2 for int8 and 4e-2 for e4m3."""
import ctypes
import os

import numpy as np
import pytest

import fixtures
import kv8_emulation

pytestmark = pytest.mark.gpu
GOLD = os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden")
TOL = 2e-3
INT8, E4M3 = 1, 2


def err(a, b):
    return float(np.max(np.abs(a - b)) / np.max(np.abs(b)))


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("name,n", [("tiny_target", 130), ("tiny_draft", 70), ("d11b_2layer", 40)])
def test_logits_against_the_emulation(cuda, name, n, kind):
    """A prompt in calls of 64 rows, single tokens, a rewind, and the fp32 cache again."""
    import vxb200
    cfg = fixtures.CONFIGS[name]
    ids = np.random.default_rng(3).integers(0, cfg[5], n + 8).astype(np.int32)
    m = vxb200.Model(fixtures.path(name))
    plain = m.forward(ids[:n])
    m.set_kv_cache(kind)
    assert m.cache_len == 0
    ref = kv8_emulation.Model(fixtures.path(name), cfg, kind)
    got = m.forward(ids[:n])
    for i in range(0, n, 64):   # the device's calls
        want = ref.forward(ids[i:min(i + 64, n)])
    assert err(got, want) <= TOL
    assert err(plain, want) > 2 * TOL   # the cache's rounding is there
    for i in range(n, n + 5):
        assert err(m.forward(ids[i:i + 1]), ref.forward(ids[i:i + 1])) <= TOL
    m.cache_len = ref.pos = n + 2       # two tokens dropped, others in their place
    assert err(m.forward(ids[n + 5:n + 8]), ref.forward(ids[n + 5:n + 8])) <= TOL
    m.set_kv_cache(0)
    np.testing.assert_array_equal(m.forward(ids[:n]), plain)
    m.close()


@pytest.mark.parametrize("kind", [INT8, E4M3])
def test_greedy_on_the_device_equals_the_host_loop(cuda, kind):
    import vxb200
    g = np.load(os.path.join(GOLD, "tiny_target.npz"))
    prompt = g["prompt"].astype(np.int32)
    m = vxb200.Model(fixtures.path("tiny_target"))
    m.set_kv_cache(kind)
    got = m.generate_greedy(prompt, 90)   # past a block's end
    m.set_kv_cache(kind)                  # starts anew
    lg, want = m.forward(prompt), []
    for _ in range(90):
        want.append(int(np.argmax(lg)))
        lg = m.forward(np.array([want[-1]], np.int32))
    np.testing.assert_array_equal(got, want)
    m.close()


class Seqs:
    """vxc_seqs over a device-generated net of the tiny target's shape, and vxc_forward."""

    def __init__(self, torch, kind, n_slots, max_ctx, max_rows, bs=16, n_blocks=0):
        import vxb200
        self.t, self.L = torch, vxb200.lib()
        e, layers, h, kv, ff, v, wt, seed, th = fixtures.CONFIGS["tiny_target"]
        c = vxb200.NetConfig(layers, h, kv, e, e // h, ff, v, 4096, th)
        self.net, self.s, self.V = ctypes.c_void_p(), ctypes.c_void_p(), v
        vxb200.check(self.L.vxc_net_create_synth(ctypes.byref(c), wt, seed, None, ctypes.byref(self.net)), "net")
        vxb200.check(self.L.vxc_seqs_create_kv8(self.net, n_slots, max_ctx, max_rows, kind, bs, n_blocks,
                                                ctypes.byref(self.s)), "seqs")

    def forward(self, tokens, slot, pos):
        """tokens [groups][rows]; logits [groups][V] of each group's last row, and the error word."""
        t = self.t
        tokens = np.asarray(tokens, np.int32)
        G, T = tokens.shape
        d = [t.from_numpy(np.ascontiguousarray(x, np.int32)).cuda() for x in (tokens, slot, pos, np.arange(G) * T + T - 1)]
        out = t.zeros(G, self.V, device="cuda")
        st = t.cuda.current_stream().cuda_stream
        rc = self.L.vxc_forward(self.s, d[0].data_ptr(), d[1].data_ptr(), d[2].data_ptr(), G, T, d[3].data_ptr(), G,
                                out.data_ptr(), st)
        assert rc == 0, self.L.vxc_error_string()
        code = ctypes.c_uint(0)
        self.L.vxc_check_device_error(ctypes.byref(code))
        return out.cpu().numpy(), code.value

    def close(self):
        self.L.vxc_seqs_destroy(self.s)
        self.L.vxc_net_destroy(self.net)


@pytest.mark.parametrize("kind", [INT8, E4M3])
def test_slots_share_the_blocks(cuda, kind):
    """Three slots over a pool too small for all contexts: each gives the logits
    it gives alone; a shorter position frees blocks; none free is reported and
    mended by freeing."""
    ids = np.random.default_rng(0).integers(0, 4096, (4, 60))
    one = Seqs(cuda, kind, 1, 256, 64)
    many = Seqs(cuda, kind, 3, 256, 192, n_blocks=10)     # 160 tokens for 3 x 256
    got, e = many.forward(ids[:3, :40], [2, 0, 1], [0, 0, 0])   # 3 x 3 blocks
    assert e == 0
    want = [one.forward(ids[g:g + 1, :40], [0], [0])[0][0] for g in range(3)]
    for g in range(3):
        assert err(got[g], want[g]) <= TOL
    lg, e = many.forward(ids[0:1, 40:56], [2], [40])            # the tenth block
    assert e == 0
    one.forward(ids[0:1, :40], [0], [0])
    assert err(lg[0], one.forward(ids[0:1, 40:56], [0], [40])[0][0]) <= TOL
    assert many.forward(ids[1:2, 40:56], [0], [40])[1] != 0     # none free
    assert many.forward(ids[3:4, :5], [1], [0])[1] == 0         # slot 1 starts anew with one block: two free
    lg, e = many.forward(ids[1:2, 40:56], [0], [40])
    assert e == 0
    one.forward(ids[1:2, :40], [0], [0])
    assert err(lg[0], one.forward(ids[1:2, 40:56], [0], [40])[0][0]) <= TOL
    one.close()
    many.close()


def test_groups_outside_the_set_are_reported(cuda):
    s = Seqs(cuda, INT8, 2, 64, 64)
    ids = np.random.default_rng(0).integers(0, 4096, (2, 8))
    good, e = s.forward(ids[:1], [1], [0])
    assert e == 0
    for slot, pos in (([1, 1], [0, 0]), ([1, 2], [0, 0]), ([1, -1], [0, 0]), ([1, 0], [0, -3]), ([1, 0], [0, 64])):
        lg, e = s.forward(ids, slot, pos)
        assert e != 0
        assert np.all(np.isfinite(lg)) and err(lg[0], good[0]) <= TOL
    lg, e = s.forward(ids, [1, 0], [0, 60])    # runs past the context
    assert e != 0 and err(lg[0], good[0]) <= TOL
    rc = s.L.vxc_forward(s.s, 1, 1, 1, 3, 1, None, 0, None, None)
    assert rc == -4 and b"one group per slot" in s.L.vxc_error_string()
    assert s.forward(ids[1:], [0], [0])[1] == 0
    s.close()


def test_contexts_over_the_limit_are_refused(cuda):
    s = Seqs(cuda, INT8, 1, 64, 64)
    for max_ctx in ((1 << 30) + 1, 2 ** 31 - 1):
        h = ctypes.c_void_p()
        assert s.L.vxc_seqs_create_kv8(s.net, 1, max_ctx, 64, INT8, 64, 4, ctypes.byref(h)) == -4 and not h.value
    s.close()


@pytest.mark.parametrize("kind", [INT8, E4M3])
def test_greedy_ended_by_eos_leaves_the_cache_as_the_host_loop_does(cuda, kind):
    """The replays between eos and the host's next look at the device change nothing: logits after an ended
    generation are those after the same tokens one by one."""
    import vxb200
    m = vxb200.Model(fixtures.path("tiny_target"))
    vocab = fixtures.CONFIGS["tiny_target"][5]
    for seed in range(6):
        ids = np.random.default_rng(seed).integers(0, vocab, 8).astype(np.int32)
        prompt, more = ids[:2 + seed], ids[-2:]
        m.set_kv_cache(kind)
        stream = m.generate_greedy(prompt, 24)
        for end in (1, 3, 6):
            eos = int(stream[end])
            n = int(np.argmax(stream == eos))
            m.set_kv_cache(kind)
            np.testing.assert_array_equal(m.generate_greedy(prompt, 24, eos), stream[:n])
            assert m.cache_len == len(prompt) + n
            got = m.forward(more)
            m.set_kv_cache(kind)
            m.forward(prompt)
            for t in stream[:n]:
                m.forward(np.array([t], np.int32))
            np.testing.assert_array_equal(got, m.forward(more))
    m.close()


@pytest.mark.parametrize("kind", [INT8, E4M3])
def test_greedy_ended_by_eos_needs_no_more_blocks(cuda, kind):
    """eos with the last position at a block's end and no block free."""

    def run(s, prompt, eos, most=20):
        out, n, pos = np.zeros(most, np.int32), ctypes.c_int(-1), ctypes.c_int(-1)
        rc = s.L.vxc_greedy_generate(s.s, 0, 0, prompt.ctypes.data, len(prompt), out.ctypes.data, most, eos,
                                     ctypes.byref(n), ctypes.byref(pos))
        return rc, out[:max(n.value, 0)], pos.value

    cases = 0
    for n in range(1, 7):   # tokens before eos
        prompt = np.random.default_rng(n).integers(0, 4096, 32 - n).astype(np.int32)
        s = Seqs(cuda, kind, 1, 256, 64)
        rc, stream, _ = run(s, prompt, -1)
        s.close()
        assert rc == 0
        if stream[n] in stream[:n]:
            continue
        cases += 1
        s = Seqs(cuda, kind, 1, 256, 64, n_blocks=2)
        rc, got, pos = run(s, prompt, int(stream[n]))
        assert rc == 0, s.L.vxc_error_string()
        np.testing.assert_array_equal(got, stream[:n])
        assert pos == 32
        s.close()
    assert cases


@pytest.mark.parametrize("kind", [INT8, E4M3])
def test_paged_cache_of_a_tensor_parallel_model(cuda, kind):
    """A model made by vx_model_create_tp for one GPU, its exchanges included, gives the plain model's numbers."""
    import vxb200
    ids = np.random.default_rng(3).integers(0, fixtures.CONFIGS["tiny_target"][5], 90).astype(np.int32)
    got = []
    for tp in (None, (0, 1, vxb200.tp_unique_id())):
        m = vxb200.Model(fixtures.path("tiny_target"), tp=tp)
        m.set_kv_cache(kind)
        got.append([m.forward(ids[:80]), m.forward(ids[80:85]), m.generate_greedy(ids[85:], 20), m.forward(ids[:1])])
        m.close()
    for a, b in zip(*got):
        assert err(b, a) <= 1e-5
    np.testing.assert_array_equal(got[0][2], got[1][2])
