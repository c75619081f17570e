"""Cases of the paged 8-bit KV cache: block tables and slot maps built from
request lengths, the append that quantises new K/V rows into blocks with a
scale for each block and head, and the attention that reads them.

`run` computes each operator in plain torch (fp32), or, where `own` is true,
through the library's entry points (vxc_kv8_tables, vxc_kv8_append,
vxc_kv8_attn).  Shapes are those of the models the repository benchmarks: the
7B target (32 heads of 128), the 1.1B draft (32 query / 4 KV heads of 64) and
the 70B target (64 query / 8 KV heads of 128).
"""
import math

import torch

own = False

INT8, E4M3 = 1, 2            # VXC_KV8_INT8, VXC_KV8_E4M3
QMAX = {INT8: 127.0, E4M3: 448.0}


def listed():
    return [
        # one decode step of the 8 sequences of the 7B benchmark: one new token each
        dict(name="tables, 8 decoding", op="tables", n_req=8, ctx=768, new=1, bs=16, pad=0, done=0.0),
        # a server's decode step: 250 requests of any length, some just finished
        dict(name="tables, 250 decoding", op="tables", n_req=250, ctx=16384, new=1, bs=64, pad=6, done=0.1),
        # admission of 32 prompts of up to 4096 tokens into an empty cache
        dict(name="tables, 32 prompts", op="tables", n_req=32, ctx=0, new=4096, bs=32, pad=100, done=0.0),
        # one decode step of one layer of the 7B target, 8 sequences
        dict(name="append, 8 rows", op="append", type=INT8, n_req=8, new=1, ctx=768, kh=32, hd=128, bs=64),
        # a verify step of the 70B target: 32 sequences, 6 drafted tokens and one more
        dict(name="append, 32x7 rows", op="append", type=E4M3, n_req=32, new=7, ctx=4096, kh=8, hd=128, bs=16),
        # the prompt pass of 32 sequences of the 70B target
        dict(name="append, 32 prompts", op="append", type=INT8, n_req=32, new=2047, ctx=0, kh=8, hd=128, bs=64),
        # a draft step of the 1.1B model, 8 sequences
        dict(name="draft step, 8x768", op="attn", type=INT8, n_req=8, new=1, ctx=768, h=32, kh=4, hd=64, bs=16),
        # the 7B target's verify of 4 drafted tokens, 8 sequences
        dict(name="verify, 8x768", op="attn", type=INT8, n_req=8, new=5, ctx=768, h=32, kh=32, hd=128, bs=64),
        # the 70B target's verify of 6 drafted tokens, 32 sequences
        dict(name="verify, 32x4096", op="attn", type=INT8, n_req=32, new=7, ctx=4096, h=64, kh=8, hd=128, bs=32),
        # a decode step of 33 long sequences of the 70B target
        dict(name="decode, 33x16384", op="attn", type=E4M3, n_req=33, new=1, ctx=16384, h=64, kh=8, hd=128, bs=64),
        # the prompt pass of the 7B benchmark: 8 prompts of up to 512 tokens
        dict(name="prompts, 8x512", op="attn", type=INT8, n_req=8, new=512, ctx=512, h=32, kh=32, hd=128, bs=64),
        # the last piece of a long prompt of the 70B target
        dict(name="prompt piece at 12k", op="attn", type=E4M3, n_req=1, new=4096, ctx=16384, h=64, kh=8, hd=128, bs=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "append", "append", "attn", "attn", "attn"])
    bs = rng.choice([16, 32, 48, 64, 128])
    if op == "tables":
        n_req = _log(rng, 1, 600)
        new = min(_log(rng, 1, 4096), 131072 // n_req)
        return dict(op=op, n_req=n_req, ctx=_log(rng, 1, 16384), new=new, bs=bs, pad=rng.choice([0, 1, 57]),
                    done=rng.choice([0.0, 0.1]))
    kind = rng.choice([INT8, E4M3])
    hd = rng.choice([32, 64, 96, 128, 128])
    if op == "append":
        kh = _log(rng, 1, 32)
        n_req = _log(rng, 1, 128)
        new = max(1, min(_log(rng, 1, 4096), 65504 // n_req, 65504 * 1024 // (n_req * kh * hd)))
        return dict(op=op, type=kind, n_req=n_req, new=new, ctx=rng.choice([0, _log(rng, 1, 4096)]), kh=kh, hd=hd, bs=bs)
    g = rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 8, 16])
    kh = _log(rng, 1, max(1, 64 // g))
    ctx = _log(rng, 1, 16384)
    new = min(ctx, rng.choice([1, _log(rng, 1, 16), _log(rng, 1, 2048)]))
    most = min(5.3e8 / (ctx * kh * hd), 4.2e9 / (new * g * kh * ctx), 128)
    return dict(op=op, type=kind, n_req=_log(rng, 1, max(1.0, most)), new=new, ctx=ctx, h=g * kh, kh=kh, hd=hd, bs=bs)


# ---- inputs ------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _lengths(case):
    """(tokens cached before the call, new tokens) of each request, the same for
    every seed: the first request has the full lengths, the others at least half
    of the new tokens and any context; `done` of them have finished."""
    n, new = case["n_req"], case["new"]
    before = max(0, case["ctx"] - (new if case["op"] == "attn" else 0))
    u = torch.rand(3, n, generator=torch.Generator().manual_seed(n + before + new))
    u[:, 0] = 1.0
    length = torch.floor(u[0] * before).to(torch.int32)
    fresh = torch.ceil((0.5 + 0.5 * u[1]) * new).to(torch.int32).clamp(min=1)
    return length, fresh, u[2] < case.get("done", 0.0)


def _ceil(a, b):
    return (a + b - 1) // b


def _paged(need, n_blocks, width, g):
    """A block table [n_req][width] that holds need[r] blocks of a shuffled pool."""
    order = torch.randperm(n_blocks, generator=g, device="cuda").to(torch.int32)
    have = torch.arange(width, device="cuda")[None, :] < need[:, None]
    at = (torch.cumsum(need, 0) - need)[:, None] + torch.arange(width, device="cuda")[None, :]
    table = torch.where(have, order[at.clamp(max=n_blocks - 1).long()], torch.full_like(at, -1).to(torch.int32))
    return table.to(torch.int32).contiguous(), order


def _slots(table, length, fresh, bs):
    """Slot of every new token, request after request."""
    req = torch.repeat_interleave(torch.arange(len(fresh), device="cuda"), fresh.long())
    first = torch.cumsum(fresh, 0) - fresh
    p = length[req] + (torch.arange(len(req), device="cuda") - first[req])
    return (table[req, (p // bs).long()] * bs + p % bs).to(torch.int32)


def _values(rows, kh, hd, g):
    """K or V rows: normal, with channels and tokens of their own size."""
    x = torch.randn(rows, kh, hd, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(1, kh, hd, generator=g, device="cuda"))
    x *= torch.exp(0.3 * torch.randn(rows, 1, 1, generator=g, device="cuda"))
    return x


def prepare(case, seed):
    g = _gen(seed)
    bs = case["bs"]
    length, fresh, gone = (x.to("cuda") for x in _lengths(case))
    if case["op"] == "tables":
        held = _ceil(length, bs)
        length, fresh = length.masked_fill(gone, 0), fresh.masked_fill(gone, 0)
        width = int(_ceil(case["ctx"] + case["new"], bs))
        n_blocks = case["n_req"] * width + 5
        table, order = _paged(held, n_blocks, width, g)
        used = int(held.sum())
        # the queue of free blocks: a ring, its head anywhere
        head = int(torch.randint(0, n_blocks, (1,), generator=g, device="cuda"))
        free = torch.full((n_blocks,), -1, dtype=torch.int32, device="cuda")
        free[(head + torch.arange(n_blocks - used, device="cuda")) % n_blocks] = order[used:]
        state = torch.tensor([head, n_blocks - used, 0], dtype=torch.int32, device="cuda")
        rows = int(fresh.sum()) + case["pad"]
        return dict(case=case, length=length, fresh=fresh, held=held, table=table, free=free, state=state,
                    row0=torch.zeros(case["n_req"] + 1, dtype=torch.int32, device="cuda"),
                    slot=torch.empty(rows, dtype=torch.int32, device="cuda"), n_blocks=n_blocks, width=width)
    kh, hd, kind = case["kh"], case["hd"], case["type"]
    total = length + fresh
    need = _ceil(total, bs)
    width = int(need.max())
    n_blocks = int(need.sum()) + 3
    table, _ = _paged(need, n_blocks, width, g)
    s = dict(case=case, length=length, fresh=fresh, table=table, n_blocks=n_blocks, width=width,
             rows=int(fresh.sum()), most=int(fresh.max()))
    # the cache as earlier appends left it: every block that holds a token is full of values
    for name in ("k", "v"):
        code, scale = [], []
        step = max(1, (1 << 26) // (bs * kh * hd))
        for b in range(0, n_blocks, step):
            x = _values(min(step, n_blocks - b) * bs, kh, hd, g).view(-1, bs, kh, hd).transpose(1, 2)
            e = _scale(x.abs().amax((2, 3)), kind)
            scale.append(e)
            code.append(_code(x, e[:, :, None, None], kind))
        s[name] = torch.cat(code).contiguous()
        s[name + "s"] = torch.cat(scale).contiguous()
        del code, scale
    if case["op"] == "append":
        s["slot"] = _slots(table, length, fresh, bs)
        # rows of the fused projection: K and V of a token side by side
        s["kv"] = torch.stack([_values(s["rows"], kh, hd, g), 1.1 * _values(s["rows"], kh, hd, g)], 1).contiguous()
        return s
    s["row0"] = torch.cat([torch.zeros(1, device="cuda", dtype=torch.int32), torch.cumsum(fresh, 0).to(torch.int32)])
    s["q"] = torch.randn(s["rows"], case["h"], hd, generator=g, device="cuda") * 0.7
    s["scale"] = 1.0 / math.sqrt(hd)
    return s


# ---- the plain forms -----------------------------------------------------------

def _scale(amax, kind):
    """The smallest power of two s with amax <= QMAX s (0 for amax 0, at least 2^-126)."""
    f, e = torch.frexp(amax)
    bits = 7 if kind == INT8 else 9
    e = torch.where(f <= QMAX[kind] / (1 << bits), e - bits, e - bits + 1).clamp(min=-126)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e), torch.zeros_like(amax))


def _code(x, s, kind):
    """Codes (as stored: bytes) of x in units of s, to nearest, ties to even."""
    y = torch.where(s > 0, x / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(x))
    if kind == INT8:
        return torch.round(y).to(torch.int8).view(torch.uint8)
    return y.to(torch.float8_e4m3fn).view(torch.uint8)


def _held_as(code, kind):
    """The stored bytes as the numbers they are, without a copy."""
    return code.view(torch.int8 if kind == INT8 else torch.float8_e4m3fn)


def _plain_tables(s):
    bs, n, nb, width = s["case"]["bs"], s["case"]["n_req"], s["n_blocks"], s["width"]
    length, fresh, held, table, free, state = (s[k] for k in ("length", "fresh", "held", "table", "free", "state"))
    want = _ceil(length + fresh, bs)
    more, less = (want - held).clamp(min=0).long(), (held - want).clamp(min=0).long()
    col = torch.arange(width, device="cuda")[None, :]
    head, count = state[0].long(), state[1].long()
    # surplus blocks to the back of the queue, request after request; new ones from its front
    back = (col >= want[:, None]) & (col < held[:, None])
    to = (head + count + (torch.cumsum(less, 0) - less)[:, None] + col - want[:, None]) % nb
    take = (col >= held[:, None]) & (col < want[:, None])
    at = (head + (torch.cumsum(more, 0) - more)[:, None] + col - held[:, None]) % nb
    got = free[at]
    free[to[back]] = table[back]
    table.copy_(torch.where(take, got, torch.where(back, torch.full_like(table, -1), table)))
    held.copy_(want)
    state.copy_(torch.stack([(head + more.sum()) % nb, count - more.sum() + less.sum(), torch.zeros_like(head)]))
    s["row0"][1:] = torch.cumsum(fresh, 0)
    rows = s["slot"].numel()
    i = torch.arange(rows, device="cuda")
    req = torch.searchsorted(s["row0"][1:].long(), i, right=True).clamp(max=n - 1)
    p = length[req].long() + i - s["row0"][:-1][req].long()
    live = i < s["row0"][-1]
    p = torch.where(live, p, torch.zeros_like(p))
    s["slot"].copy_(torch.where(live, table[req, p // bs].long() * bs + p % bs, torch.full_like(p, -1)))
    return s["row0"], s["slot"], table, held, free, state


def _plain_append(s):
    case = s["case"]
    bs, kind = case["bs"], case["type"]
    slot = s["slot"].long()
    block, off = slot // bs, slot % bs
    fresh_block = torch.zeros(s["n_blocks"], dtype=torch.bool, device="cuda")
    fresh_block[block[off == 0]] = True
    blocks, inv = torch.unique(block, return_inverse=True)
    written = torch.zeros(len(blocks), bs, dtype=torch.bool, device="cuda")
    written[inv, off] = True
    outs = []
    for name, x in (("k", s["kv"][:, 0]), ("v", s["kv"][:, 1])):
        code, scale = s[name], s[name + "s"]
        amax = torch.zeros(len(blocks), case["kh"], device="cuda")
        amax.scatter_reduce_(0, inv[:, None].expand(-1, case["kh"]), x.abs().amax(2), "amax")
        old = scale[blocks].masked_fill(fresh_block[blocks][:, None], 0.0)
        new = torch.maximum(old, _scale(amax, kind))
        held = _held_as(code[blocks], kind).float()
        grown = _code(held * (old / torch.where(new > 0, new, torch.ones_like(new)))[:, :, None, None],
                      torch.ones(1, device="cuda"), kind)
        keep = written[:, None, :, None] | (old <= 0)[:, :, None, None] | (new == old)[:, :, None, None]
        code[blocks] = torch.where(keep, code[blocks], grown)
        scale[blocks] = new
        code[block, :, off] = _code(x, new[inv][:, :, None], kind)
        outs += [_held_as(code, kind), scale]
    return tuple(outs)


def _plain_attn(s):
    case = s["case"]
    n, h, kh, hd, bs, kind = (case[k] for k in ("n_req", "h", "kh", "hd", "bs", "type"))
    g, width, most = h // kh, s["width"], s["most"]
    ctx = width * bs
    table = s["table"].clamp(min=0).long()
    kv = []
    for name in ("k", "v"):
        x = _held_as(s[name][table], kind).float() * s[name + "s"][table][..., None, None]   # [n, width, kh, bs, hd]
        kv.append(x.transpose(1, 2).reshape(n, kh, ctx, hd))
    # rows of a request side by side, padded to the longest
    t = torch.arange(most, device="cuda")
    row = s["row0"][:-1, None].long() + t[None, :]
    live = t[None, :] < s["fresh"][:, None]
    q = s["q"][torch.where(live, row, torch.zeros_like(row))]                # [n, most, h, hd]
    q = q.view(n, most, kh, g, hd).permute(0, 2, 1, 3, 4).reshape(n, kh, most * g, hd)
    a = torch.matmul(q, kv[0].transpose(2, 3)).mul_(s["scale"])
    pos = s["length"][:, None] + t[None, :]                                  # [n, most]
    seen = torch.arange(ctx, device="cuda")[None, None, :] <= pos[:, :, None]
    a = a.view(n, kh, most, g, ctx).masked_fill_(~seen[:, None, :, None, :], float("-inf"))
    a = a.sub_(a.amax(4, keepdim=True)).exp_()
    a = a.div_(a.sum(4, keepdim=True)).view(n, kh, most * g, ctx)
    o = torch.matmul(a, kv[1]).view(n, kh, most, g, hd).permute(0, 2, 1, 3, 4).reshape(n, most, h, hd)
    return o[live]


# ---- the framework's calls ------------------------------------------------------

def _library():
    import os
    import sys
    path = os.path.join(os.getcwd(), "veltrix-engine_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import vxb200
    return vxb200


def _own(s):
    lib = _library()
    case = s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "tables":
        lib.kv8_tables(s["length"].data_ptr(), s["fresh"].data_ptr(), case["n_req"], case["bs"], s["n_blocks"],
                       s["width"], s["table"].data_ptr(), s["held"].data_ptr(), s["free"].data_ptr(),
                       s["state"].data_ptr(), s["slot"].numel(), s["row0"].data_ptr(), s["slot"].data_ptr(), stream)
        return s["row0"], s["slot"], s["table"], s["held"], s["free"], s["state"]
    cache = s.get("cache")
    if cache is None:
        cache = s["cache"] = lib.KV8(case["type"], s["n_blocks"], case["bs"], case["kh"], case["hd"], s["k"].data_ptr(),
                                     s["v"].data_ptr(), s["ks"].data_ptr(), s["vs"].data_ptr())
    if case["op"] == "append":
        kv, ld = s["kv"], 2 * case["kh"] * case["hd"]
        cache.append(kv.data_ptr(), ld, kv.data_ptr() + 2 * ld, ld, s["slot"].data_ptr(), s["rows"], stream)
        return _held_as(s["k"], case["type"]), s["ks"], _held_as(s["v"], case["type"]), s["vs"]
    ws = s.get("ws")
    if ws is None:   # kept from step to step, as a server keeps it
        size = cache.attn_workspace_bytes(case["h"], case["n_req"], s["rows"], s["most"], s["width"])
        ws = s["ws"] = torch.empty(size // 4 + 4, device="cuda")
    ld = case["h"] * case["hd"]
    out = torch.empty_like(s["q"])
    cache.attn(s["q"].data_ptr(), ld, case["h"], s["scale"], s["table"].data_ptr(), s["width"], s["row0"].data_ptr(),
               s["length"].data_ptr(), case["n_req"], s["rows"], s["most"], out.data_ptr(), ld, ws.data_ptr(),
               ws.numel() * 4, stream)
    return out


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return _plain_tables(state) if op == "tables" else _plain_append(state) if op == "append" else _plain_attn(state)


# ---- what a pass cannot do without -----------------------------------------------

def work(case):
    length, fresh, gone = (x.to(torch.int64) for x in _lengths(case))
    n = case["n_req"]
    if case["op"] == "tables":
        length, fresh = length * (1 - gone), fresh * (1 - gone)
    blocks = int((_ceil(length + fresh, case["bs"]) - length // case["bs"]).sum())   # that hold new tokens
    rows = int(fresh.sum())
    if case["op"] == "tables":
        # lengths, new tokens and held blocks read; held blocks, first rows and slots written; the
        # table entries behind the new tokens
        return dict(bytes=4.0 * (5 * n + 1 + rows + case["pad"] + blocks), flops=0.0)
    width = case["kh"] * case["hd"]
    if case["op"] == "append":
        # fp32 K and V rows in, their bytes out, the slot map, the scales of the blocks
        return dict(bytes=rows * (2 * width * 5 + 4.0) + blocks * case["kh"] * 8.0, flops=rows * 4.0 * width)
    tokens = int((length + fresh).sum())
    pairs = int((fresh * length + fresh * (fresh + 1) // 2).sum())   # (row, visible token)
    # K and V bytes once, fp32 queries in and outputs out; a product with K and one with V
    return dict(bytes=tokens * 2.0 * width + rows * case["h"] * case["hd"] * 8.0,
                flops=4.0 * pairs * case["h"] * case["hd"])


# ---- the definition in 64 bits -----------------------------------------------------

def _number(byte, kind):
    """Stored bytes as fp64 numbers."""
    b = byte.to(torch.int64)
    if kind == INT8:
        return torch.where(b > 127, b - 256, b).double()
    sign, e, m = 1.0 - 2.0 * (b >> 7), (b >> 3) & 15, (b & 7).double()
    return sign * torch.where(e > 0, (1 + m / 8) * torch.exp2((e - 7).double()), m / 8 * 2.0 ** -6)


def _rounded(y, kind):
    """fp64 numbers rounded to those that a byte holds."""
    if kind == INT8:
        return torch.round(y)
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    e = torch.where(y.abs() < torch.exp2(e), e - 1, e).clamp(min=-6)
    step = torch.exp2(e - 3)
    return torch.round(y / step) * step


def exact(case, seed):
    if case["op"] == "tables":
        return None   # whole numbers
    s = prepare(case, seed)
    kind, bs, kh, hd = case["type"], case["bs"], case["kh"], case["hd"]
    if case["op"] == "append":
        if s["rows"] // bs + case["n_req"] > 3000:
            return None   # goes block by block
        outs = []
        order = torch.argsort(s["slot"])
        slot = s["slot"][order].long()
        for c, name in ((0, "k"), (1, "v")):
            code, scale = _number(s[name], kind), s[name + "s"].double()
            for block, at in _runs(slot // bs):
                x, off = s["kv"][order[at], c].double(), slot[at] % bs
                old = torch.zeros_like(scale[block]) if int(off[0]) == 0 else scale[block]
                a = x.abs().amax((0, 2))
                e = torch.ceil(torch.log2(a.clamp(min=2.0 ** -150) / QMAX[kind]))
                e = torch.where(a <= QMAX[kind] * torch.exp2(e - 1), e - 1, e)
                e = torch.where(a > QMAX[kind] * torch.exp2(e), e + 1, e).clamp(min=-126)
                new = torch.maximum(old, torch.where(a > 0, torch.exp2(e), torch.zeros_like(a)))
                for i in torch.nonzero((new > old) & (old > 0)).flatten().tolist():
                    code[block, i] = _rounded(code[block, i] * (old[i] / new[i]), kind)
                scale[block] = new
                one = torch.where(new > 0, new, torch.ones_like(new))
                code[block].index_copy_(1, off, _rounded(x / one[None, :, None], kind).transpose(0, 1).contiguous())
            outs += [code if kind == E4M3 else code.to(torch.int8), scale]
        return tuple(outs)
    h, g = case["h"], case["h"] // kh
    out = torch.empty(s["rows"], h, hd, dtype=torch.float64, device="cuda")
    first = s["row0"].tolist()
    for r, past in enumerate(s["length"].tolist()):
        rows = slice(first[r], first[r + 1])
        total = past + first[r + 1] - first[r]
        blocks = s["table"][r, :-(-total // bs)].long()
        seen = torch.arange(total, device="cuda")[None, :] <= past + torch.arange(total - past, device="cuda")[:, None]
        for j in range(kh):
            k, v = ((_number(s[c][blocks, j], kind) * s[c + "s"][blocks, j].double()[:, None, None]).view(-1, hd)[:total]
                    for c in ("k", "v"))
            for i in range(j * g, (j + 1) * g):
                a = s["q"][rows, i].double() @ k.T * s["scale"]
                out[rows, i] = torch.softmax(a.masked_fill(~seen, -math.inf), 1) @ v
    return out


def _runs(block):
    """(block, positions of its rows) of a sorted list of block numbers."""
    ids, counts = torch.unique_consecutive(block, return_counts=True)
    at = 0
    for b, c in zip(ids.tolist(), counts.tolist()):
        yield b, slice(at, at + c)
        at += c
