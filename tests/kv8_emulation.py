"""A llama forward in float64 over the paged 8-bit cache, from the checkpoint
file (GGUF, Q8_0 or Q4_0 matrices): test infrastructure only.  The arithmetic
is the forward's (csrc/vxc_model.cu): RMSNorm with 1e-5, interleaved RoPE pairs,
causal attention, |silu(gate)| < 0.01 masked to 0; K and V pass through
kv8ref.Cache after rounding to fp32, as the append kernel sees them."""
import struct

import numpy as np

import kv8ref


def read_gguf(path):
    """{tensor name: float64 array [rows, cols] or [cols]} of a GGUF v2/v3 file, and its metadata."""
    b = open(path, "rb").read()
    at = [4]

    def get(fmt):
        v = struct.unpack_from("<" + fmt, b, at[0])[0]
        at[0] += struct.calcsize(fmt)
        return v

    def text():
        n = get("Q")
        v = b[at[0]:at[0] + n].decode()
        at[0] += n
        return v

    kinds = {0: "B", 1: "b", 2: "H", 3: "h", 4: "I", 5: "i", 6: "f", 7: "?", 10: "Q", 11: "q", 12: "d"}

    def val(t):
        if t == 8:
            return text()
        if t == 9:
            u, n = get("I"), get("Q")
            return [val(u) for _ in range(n)]
        return get(kinds[t])

    get("I")
    nt, nk = get("Q"), get("Q")
    meta = {}
    for _ in range(nk):
        k = text()
        meta[k] = val(get("I"))
    infos = []
    for _ in range(nt):
        name = text()
        dims = [get("Q") for _ in range(get("I"))]
        infos.append((name, dims, get("I"), get("Q")))
    base = -(-at[0] // meta.get("general.alignment", 32)) * meta.get("general.alignment", 32)
    out = {}
    for name, dims, t, off in infos:
        cols, rows = int(dims[0]), int(np.prod(dims[1:], dtype=np.int64))
        if t == 0:
            x = np.frombuffer(b, np.float32, rows * cols, base + off).astype(np.float64)
        else:
            size = {2: 18, 8: 34}[t]
            q = np.frombuffer(b, np.uint8, rows * cols // 32 * size, base + off).reshape(-1, size)
            d = q[:, :2].copy().view(np.float16).astype(np.float64)
            if t == 8:
                x = q[:, 2:].view(np.int8).astype(np.float64) * d
            else:   # the reference's interleaved nibbles
                n = np.stack([q[:, 2:] & 15, q[:, 2:] >> 4], 2).reshape(-1, 32)
                x = (n.astype(np.float64) - 8) * d
        out[name] = x.reshape(rows, cols) if len(dims) > 1 else x
    return out, meta


class Model:
    """One sequence; kind None keeps K and V exact (fp32)."""

    def __init__(self, path, cfg, kind, bs=64, n_blocks=16):
        e, self.L, self.H, self.KH, ff, v, wt, seed, self.theta = cfg
        self.w, _ = read_gguf(path)
        self.hd = e // self.H
        self.kind, self.bs = kind, bs
        self.cache = [kv8ref.Cache(kind, n_blocks, bs, self.KH, self.hd) if kind else [[], []] for _ in range(self.L)]
        self.pos = 0

    def rope(self, x, pos):
        f = (1.0 / np.power(np.float32(self.theta), (np.arange(self.hd // 2, dtype=np.float32) * 2) / np.float32(self.hd)))
        a = (pos[:, None].astype(np.float32) * f.astype(np.float32)).astype(np.float64)
        c, s = np.cos(a)[:, None, :], np.sin(a)[:, None, :]
        o = np.empty_like(x)
        o[..., 0::2] = x[..., 0::2] * c - x[..., 1::2] * s
        o[..., 1::2] = x[..., 0::2] * s + x[..., 1::2] * c
        return o

    def forward(self, tokens):
        """Logits of the last token; the tokens are one call (one append per layer)."""
        w, T = self.w, len(tokens)
        pos = np.arange(self.pos, self.pos + T)
        x = w["token_embd.weight"][tokens]
        norm = lambda x, g: x / np.sqrt((x * x).mean(1, keepdims=True) + 1e-5) * g
        for l in range(self.L):
            b = "blk.%d." % l
            h = norm(x, w[b + "attn_norm.weight"])
            q = self.rope((h @ w[b + "attn_q.weight"].T).reshape(T, self.H, self.hd), pos)
            k = self.rope((h @ w[b + "attn_k.weight"].T).reshape(T, self.KH, self.hd), pos)
            v = (h @ w[b + "attn_v.weight"].T).reshape(T, self.KH, self.hd)
            k, v = k.astype(np.float32), v.astype(np.float32)
            c = self.cache[l]
            if self.kind:
                c.append(k, v, pos)
                kk, vv = c.rows(np.arange(-(-(self.pos + T) // self.bs)), self.pos + T)
            else:
                c[0].append(k), c[1].append(v)
                kk, vv = (np.concatenate(y).transpose(1, 0, 2).astype(np.float64) for y in c)
            o = np.zeros((T, self.H, self.hd))
            for i in range(self.H):
                j = i // (self.H // self.KH)
                s = q[:, i] @ kk[j].T / np.sqrt(self.hd)
                s[np.arange(self.pos + T)[None] > pos[:, None]] = -np.inf
                p = np.exp(s - s.max(1, keepdims=True))
                o[:, i] = p / p.sum(1, keepdims=True) @ vv[j]
            x = x + o.reshape(T, -1) @ w[b + "attn_output.weight"].T
            h = norm(x, w[b + "ffn_norm.weight"])
            g, u = h @ w[b + "ffn_gate.weight"].T, h @ w[b + "ffn_up.weight"].T
            g = g / (1 + np.exp(-g))
            x = x + np.where(np.abs(g) < 0.01, 0, g * u) @ w[b + "ffn_down.weight"].T
        self.pos += T
        out = w.get("output.weight", w["token_embd.weight"])
        return (norm(x[-1:], w["output_norm.weight"]) @ out.T)[0]
