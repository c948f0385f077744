"""What the operators of the 4-bit paged KV cache are measured on.

The cache (``--kv-cache-dtype mxfp4``) holds keys and values as OCP microscaling FP4: a value is an e2m1 number (a sign and one
of 0, 0.5, 1, 1.5, 2, 3, 4, 6) times a power of two that 32 neighbouring dims of one token and head share. Four operators:

  write    the rotary embedding of queries and keys, and the step's keys and values quantised into the paged cache
           (``rope_cache``; ``splitk_rope_cache`` from the split-K partials that a decode step's projection leaves)
  read     rows of the cache as bf16 (``read_cache``)
  decode   attention of one query per sequence over the cache (``paged_decode``)
  prompt   causal attention of prompt portions over the cache (``prefill_attention``)

the last two with a sliding window beside which the first tokens of a sequence (``sinks``) stay visible. A case that writes also
reads its rows back: those are the values that the bytes stand for.

A cache tensor is uint8 [blocks, kv heads, block_size, 17 D / 32]: per block and head first the codes, block_size D / 2 bytes of
two dims each (the even one in the low half), then one scale byte per token and 32 dims, 2^(byte - 127). Keys: codes by token,
[block_size][D / 2]; scales [D / 32][block_size], where token o of a run of 16 stands at 4 (o % 4) + o / 4. Values: codes by
pair of dims, [D / 2][block_size], scales [D / 32][block_size] in the tokens' order.
"""
import functools
import math

import torch

own = False

GROUP = 32                                          # dims that share a scale
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)   # what the low three bits of a code stand for
SCALE_MIN, SCALE_MAX = 8, 252                       # scale bytes in use: no value of a group is subnormal or above bf16's range
THETA = 500000.0


def listed():
    def write(name, tokens, seqs, nq, nkv, dim, mode, splits):
        return dict(name=name, op="write", tokens=tokens, seqs=seqs, nq=nq, nkv=nkv, dim=dim, mode=mode, splits=splits, block=16)

    def read(name, seqs, ctx, nkv, dim):
        return dict(name=name, op="read", seqs=seqs, ctx=ctx, nkv=nkv, dim=dim, block=16)

    def decode(name, seqs, ctx, nq, nkv, dim, window=0, sinks=0, block=16):
        return dict(name=name, op="decode", seqs=seqs, ctx=ctx, nq=nq, nkv=nkv, dim=dim, window=window, sinks=sinks, block=block)

    def prompt(name, seqs, rows, ctx, nq, nkv, dim, window=0, sinks=0, block=16):
        return dict(name=name, op="prompt", seqs=seqs, rows=rows, ctx=ctx, nq=nq, nkv=nkv, dim=dim, window=window, sinks=sinks,
                    block=block)

    return [
        # one layer of a decode step of four chats, from the projection's partials: latency counts
        write("write 4 chats", 4, 4, 32, 8, 128, 0, 8),
        # a full prompt step of the headline model: 8192 rows of nine prompts, none of a page's length
        write("write prompt step", 8192, 9, 32, 8, 128, 0, 0),
        # a small llama from a GGUF file: heads of 64, rotation of neighbouring dims, one odd prompt
        write("write odd prompt", 701, 1, 32, 4, 64, 1, 0),
        # one chat's rows handed on
        read("read one chat", 1, 1153, 8, 128),
        # a batch of long contexts handed on
        read("read 16 long contexts", 16, 6000, 8, 128),
        # one chat, its context cut over many workgroups: latency counts
        decode("decode one chat", 1, 1152, 32, 8, 128),
        # the headline benchmark's batch
        decode("decode 64 chats", 64, 1152, 32, 8, 128),
        # long contexts: the cache's bytes are all that counts
        decode("decode 16 long contexts", 16, 16384, 32, 8, 128),
        # a model with a window of 4096 whose first tokens stay visible, contexts far behind it
        decode("decode window and sinks", 48, 11000, 32, 8, 128, 4096, 4),
        # short ragged prompts of a model with as many key heads as query heads, heads of 96
        prompt("prompt short ragged", 5, 300, 300, 32, 32, 96),
        # the headline benchmark's prompts: one full step
        prompt("prompt 8 x 1024", 8, 1024, 1024, 32, 8, 128),
        # a portion of a long document behind what is cached already, window and first tokens
        prompt("prompt portion, window and sinks", 1, 4096, 14336, 32, 8, 128, 4096, 4),
    ]


def _spread(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    op = rng.choice(("write", "read", "decode", "decode", "prompt", "prompt"))
    nq, nkv, dim = rng.choice(((32, 8, 128), (32, 8, 128), (40, 8, 128), (28, 4, 128), (8, 1, 128), (16, 16, 128), (32, 4, 64),
                               (14, 2, 64), (32, 32, 96)))
    block = rng.choice((16, 16, 32, 64))
    if op == "write":
        splits = rng.choice((0, 0, 1, 3, 8))
        tokens = _spread(rng, 1, 256 if splits else 8192)
        seqs = tokens if splits else min(tokens, _spread(rng, 1, 12))
        return dict(op=op, tokens=tokens, seqs=seqs, nq=nq, nkv=nkv, dim=dim, mode=rng.choice((0, 1)), splits=splits, block=block)
    window = rng.choice((0, 0, 1, 1)) and _spread(rng, 64, 4096)
    sinks = rng.choice((0, 1, 4, 70)) if window else 0
    if op in ("read", "decode"):
        seqs = _spread(rng, 1, 64)
        ctx = _spread(rng, 1, min(16384, 250000 * 8 // (seqs * nkv)))
        if op == "read":
            return dict(op=op, seqs=seqs, ctx=min(ctx, 96000 * 8 // (seqs * nkv)), nkv=nkv, dim=dim, block=block)
        return dict(op=op, seqs=seqs, ctx=ctx, nq=nq, nkv=nkv, dim=dim, window=window, sinks=sinks, block=block)
    seqs = _spread(rng, 1, 9)
    rows = _spread(rng, 1, 4096 // seqs)
    ctx = rows + rng.choice((0, 0, _spread(rng, 1, 6000)))
    return dict(op=op, seqs=seqs, rows=rows, ctx=ctx, nq=nq, nkv=nkv, dim=dim, window=window, sinks=sinks, block=block)


def _lengths(most, seqs):
    """Lengths of a ragged batch: the first is ``most``, the others go down to two thirds of it."""
    return [max(1, most - (37 * i) % (most // 3 + 1)) for i in range(seqs)]


def _shares(tokens, seqs):
    """The rows of a prompt step by sequence: unequal shares that make up ``tokens``."""
    cut = [tokens * (i * (i + 9)) // (seqs * (seqs + 9)) for i in range(seqs + 1)]
    return [cut[i + 1] - cut[i] for i in range(seqs)]


# ---------------------------------------------------------------- the format, plain

def _quantise(x):
    """Rows [..., D] of bf16 values as (codes uint8 [..., D], scale bytes uint8 [..., D / 32]). The scale is the power of two under
    which a group's largest value is at most 7, and so within a sixth of the largest level; ties go to the even code."""
    g = x.float().unflatten(-1, (-1, GROUP))
    bits = g.abs().amax(-1).to(torch.bfloat16).view(torch.int16).int()
    byte = (((bits + 31) >> 7) - 2).clamp(SCALE_MIN, SCALE_MAX)
    a = torch.ldexp(g.abs(), (127 - byte)[..., None])
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int() + (a >= 3.5).int()
            + (a > 5.0).int() + 8 * torch.signbit(g).int())
    return code.to(torch.uint8).flatten(-2), byte.to(torch.uint8)


def _pack(k, v):
    """Cache tensors of blocks of bf16 rows [blocks, heads, block_size, D]."""
    n, h, bs, d = k.shape

    def tensor(codes, scales):
        return torch.cat((codes.reshape(n, h, -1), scales.reshape(n, h, -1)), -1).view(n, h, bs, 17 * d // 32)

    (kc, ks), (vc, vs) = _quantise(k), _quantise(v)
    ks = ks.view(n, h, bs // 16, 4, 4, d // GROUP).permute(0, 1, 5, 2, 4, 3)
    return (tensor(kc[..., 0::2] | (kc[..., 1::2] << 4), ks),
            tensor((vc[..., 0::2] | (vc[..., 1::2] << 4)).transpose(2, 3), vs.transpose(2, 3)))


def _values(codes, scales):
    """The values, 32 bits [..., D], of packed codes [..., D / 2] and scale bytes [..., D / 32]."""
    level = torch.tensor([s * y for s in (1.0, -1.0) for y in LEVELS], device=codes.device)
    y = level[torch.stack((codes & 15, codes >> 4), -1).int()].flatten(-2)
    return (y.unflatten(-1, (-1, GROUP)) * torch.ldexp(torch.ones_like(scales, dtype=torch.float32), scales.int() - 127)[..., None]).flatten(-2)


def _blocks(cache, blocks, values):
    """The values, 32 bits, of whole blocks [...] of a cache: [..., heads, block_size, D]."""
    n, h, bs, w = cache.shape
    d = w * 32 // 17
    x = cache.view(n, h, -1)[blocks]
    codes, scales = x[..., :bs * d // 2], x[..., bs * d // 2:]
    if values:
        return _values(codes.unflatten(-1, (d // 2, bs)).transpose(-1, -2), scales.unflatten(-1, (d // GROUP, bs)).transpose(-1, -2))
    scales = scales.unflatten(-1, (d // GROUP, bs // 16, 4, 4)).transpose(-1, -2).flatten(-3, -1).transpose(-1, -2)
    return _values(codes.unflatten(-1, (bs, d // 2)), scales)


def _places(cache, slots, values):
    """Where in the flat cache the packed codes [T, heads, D / 2] and the scale bytes [T, heads, D / 32] of slots are."""
    n, h, bs, w = cache.shape
    d = w * 32 // 17
    base = (((slots // bs)[:, None] * h + torch.arange(h, device=slots.device)) * (bs * w))[..., None]
    off = (slots % bs)[:, None, None]
    pair, group = torch.arange(d // 2, device=slots.device), torch.arange(d // GROUP, device=slots.device)
    if values:
        return base + pair * bs + off, base + bs * d // 2 + group * bs + off
    return base + off * (d // 2) + pair, base + bs * d // 2 + group * bs + off // 16 * 16 + 4 * (off % 4) + off % 16 // 4


def _slot_rows(k_cache, v_cache, slots):
    """Keys and values [T, heads, D] of the slots of two caches, as bf16; zeros for a slot below 0."""
    out = []
    for cache, values in ((k_cache, False), (v_cache, True)):
        codes, scales = (cache.view(-1)[at] for at in _places(cache, slots.clamp_min(0), values))
        out.append(torch.where((slots >= 0)[:, None, None], _values(codes, scales), 0.0).to(torch.bfloat16))
    return out


def _scatter(cache, slots, codes, scales, values):
    """Writes rows' packed codes [T, heads, D / 2] and scale bytes [T, heads, D / 32] to their slots, those below 0 nowhere."""
    keep = slots >= 0
    at, scale_at = _places(cache, slots[keep], values)
    cache.view(-1)[at] = codes[keep]
    cache.view(-1)[scale_at] = scales[keep]


def _rotated(x, cos_sin, positions, mode):
    """Rows [T, heads, D] of bf16 rotated and rounded to bf16. The framework's kernels round one product to 32 bits and add the
    other in one fused operation; a key next to a border of the 4-bit grid has to fall to the same side, so this does it likewise,
    the fused operation in 64 bits."""
    d = x.shape[-1]
    cs = cos_sin[positions][:, None]
    c, s = cs[..., :d // 2], cs[..., d // 2:]
    a, b = (x[..., :d // 2], x[..., d // 2:]) if mode == 0 else (x[..., 0::2], x[..., 1::2])
    a, b = a.float(), b.float()
    ra = (a.double() * c.double() - (b * s).double()).float()
    rb = (b.double() * c.double() + (a * s).double()).float()
    y = torch.cat((ra, rb), -1) if mode == 0 else torch.stack((ra, rb), -1).flatten(-2)
    return y.to(torch.bfloat16)


# ---------------------------------------------------------------- inputs

def _normal(shape, gen, std=1.0):
    return torch.empty(shape, device="cuda", dtype=torch.bfloat16).normal_(0.0, std, generator=gen)


def _keys(shape, gen):
    """Keys with a few channels several times as large as the rest, as keys of trained models have them."""
    k = _normal(shape, gen)
    k[..., 5::48] *= 6.0
    return k


def _cos_sin(dim, positions):
    """[positions, dim] fp32: cosines, then sines, of position / THETA^(2 i / dim)."""
    f = THETA ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
    a = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * f
    return torch.cat((a.cos(), a.sin()), -1).float()


def _tables(lens, block, gen):
    """(pages of the pool, block table [sequences, most blocks] int32): every sequence's blocks anywhere in the pool."""
    need = [-(-n // block) for n in lens]
    width, total = max(need), sum(need) + 3
    ids = torch.randperm(total, device="cuda", generator=gen).int()
    table = torch.zeros(len(lens), width, device="cuda", dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    return total, table


def _pool(total, case, gen):
    shape = (total, case["nkv"], case["block"], case["dim"])
    return _pack(_keys(shape, gen), _normal(shape, gen))


def _slots(table, lens, starts, block):
    """Slots of tokens starts[i] .. lens[i] - 1 of every sequence, one after the other."""
    pos = torch.cat([torch.arange(a, n, device="cuda") for a, n in zip(starts, lens)])
    seq = torch.cat([torch.full((n - a,), i, device="cuda") for i, (a, n) in enumerate(zip(starts, lens))])
    return pos, table[seq, pos // block].long() * block + pos % block


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c, op, block, dim, nkv = case, case["op"], case["block"], case["dim"], case["nkv"]
    st = dict(case=case)
    if op == "write":
        shares = [1] * c["tokens"] if c["splits"] else _shares(c["tokens"], c["seqs"])
        # a decode step's rows stand far into their sequences, a prompt step's begin them (the last one goes on)
        starts = [500 + 83 * i % 1500 for i in range(c["seqs"])] if c["splits"] else [0] * (c["seqs"] - 1) + [256 * (c["seqs"] % 3) + 7]
        lens = [a + n for a, n in zip(starts, shares)]
        total, table = _tables(lens, block, gen)
        st["positions"], st["slots"] = _slots(table, lens, starts, block)
        st["cos_sin"] = _cos_sin(dim, max(lens) + 1)
        st["k_cache"], st["v_cache"] = _pool(total, c, gen)
        n = (c["nq"] + 2 * nkv) * dim
        x = _normal((max(1, c["splits"]), c["tokens"], n), gen)
        x[..., 5::48] *= 6.0
        if c["splits"]:   # what the projection of a decode step leaves: 32-bit partial sums (of whole 1/1024: any order of adding is exact)
            x = x.float() + torch.empty(x.shape, device="cuda").normal_(0.0, 0.1, generator=gen)
            st["partials"] = (x * 1024).round() / 1024
            st["qkv"] = torch.empty(c["tokens"], n, device="cuda", dtype=torch.bfloat16)
        else:
            st["rows"] = x[0]
        st["k_rows"], st["v_rows"] = (torch.empty(c["tokens"], nkv, dim, device="cuda", dtype=torch.bfloat16) for _ in "kv")
        return st
    lens = _lengths(c["ctx"], c["seqs"])
    total, table = _tables(lens, block, gen)
    st["k_cache"], st["v_cache"] = _pool(total, c, gen)
    if op == "read":
        _, st["slots"] = _slots(table, lens, [0] * len(lens), block)
        st["k_rows"], st["v_rows"] = (torch.empty(sum(lens), nkv, dim, device="cuda", dtype=torch.bfloat16) for _ in "kv")
        return st
    st["table"], st["ctx"] = table, torch.tensor(lens, device="cuda", dtype=torch.int32)
    nq = c["nq"]
    if op == "decode":
        st["q"] = _normal((c["seqs"], (nq + 2 * nkv) * dim), gen)
        # a user's program keeps the workspace of a split context; its size follows the engine's rule
        wide = c["seqs"] * nkv
        part = 2048 if wide >= 512 or (wide >= 128 and table.shape[1] * block <= 2048) else 512
        parts = -(-table.shape[1] * block // part)
        st["part"] = part
        st["tmp_out"] = torch.empty(c["seqs"], nq, parts, dim, device="cuda")
        st["tmp_ml"] = torch.empty(c["seqs"], nq, parts, 2, device="cuda")
        st["out"] = torch.empty(c["seqs"], nq * dim, device="cuda", dtype=torch.bfloat16)
        return st
    rows = [min(n, r) for n, r in zip(lens, _lengths(c["rows"], c["seqs"]))]
    cu = [sum(rows[:i]) for i in range(len(rows) + 1)]
    # the host's list of 128-row tiles, the ones with the most visible keys first, as the engine dispatches them
    tiles = sorted(((i, r) for i, n in enumerate(rows) for r in range(0, n, 128)), key=lambda t: -(lens[t[0]] - rows[t[0]] + t[1]))
    st["rows"], st["most"] = rows, max(rows)
    st["cu"] = torch.tensor(cu, device="cuda", dtype=torch.int32)
    st["tiles"] = torch.tensor(tiles, device="cuda", dtype=torch.int32)
    st["q"] = _normal((cu[-1], (nq + 2 * nkv) * dim), gen)
    st["out"] = torch.empty(cu[-1], nq * dim, device="cuda", dtype=torch.bfloat16)
    return st


# ---------------------------------------------------------------- one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return _run_own(state, op)
    return {"write": _write, "read": _read, "decode": _decode, "prompt": _prompt}[op](state)


@functools.lru_cache(maxsize=None)
def _ops():
    from hipserve.ops import get_ops

    return get_ops("cuda")


def _run_own(st, op):
    c, ops = st["case"], _ops()
    heads = (c.get("nq"), c["nkv"])
    scale = 1.0 / math.sqrt(c["dim"])
    if op == "write":
        where = (st["positions"], st["slots"], st["cos_sin"], st["k_cache"], st["v_cache"], *heads, c["dim"], c["mode"])
        if c["splits"]:
            qkv = st["qkv"]
            ops.splitk_rope_cache(qkv, st["partials"], c["splits"], *where)
        else:
            qkv = st["rows"].clone()   # the queries are rotated in place
            ops.rope_cache(qkv, *where)
        ops.read_cache(st["k_rows"], st["v_rows"], st["k_cache"], st["v_cache"], st["slots"])
        return dict(q=qkv[:, :c["nq"] * c["dim"]], k=st["k_rows"], v=st["v_rows"])
    if op == "read":
        ops.read_cache(st["k_rows"], st["v_rows"], st["k_cache"], st["v_cache"], st["slots"])
        return dict(k=st["k_rows"], v=st["v_rows"])
    if op == "decode":
        return ops.paged_decode(st["out"], st["q"], st["k_cache"], st["v_cache"], st["table"], st["ctx"], st["tmp_out"], st["tmp_ml"],
                                *heads, st["part"], scale, c["window"], sinks=c["sinks"])
    return ops.prefill_attention(st["out"], st["q"], st["k_cache"], st["v_cache"], st["table"], st["cu"], st["ctx"], st["tiles"],
                                 *heads, scale, c["window"], sinks=c["sinks"])


def _write(st):
    c = st["case"]
    nq, nkv, d = c["nq"], c["nkv"], c["dim"]
    x = st["partials"].sum(0).to(torch.bfloat16) if c["splits"] else st["rows"]
    q, k, v = x.unflatten(-1, (-1, d)).split((nq, nkv, nkv), 1)
    q, k = (_rotated(y, st["cos_sin"], st["positions"], c["mode"]) for y in (q, k))
    for cache, y, values in ((st["k_cache"], k, False), (st["v_cache"], v, True)):
        codes, scales = _quantise(y)
        _scatter(cache, st["slots"], codes[..., 0::2] | (codes[..., 1::2] << 4), scales, values)
    k, v = _slot_rows(st["k_cache"], st["v_cache"], st["slots"])
    return dict(q=q.flatten(1), k=k, v=v)


def _read(st):
    k, v = _slot_rows(st["k_cache"], st["v_cache"], st["slots"])
    return dict(k=k, v=v)


def _context(st):
    """Keys and values of whole block tables, 32 bits: [sequences, heads, tokens, D]."""
    table = st["table"].long()
    return [_blocks(cache, table, values).transpose(1, 2).flatten(2, 3) for cache, values in ((st["k_cache"], False), (st["v_cache"], True))]


def _visible(pos, ctx, tokens, window, sinks):
    """Which of ``tokens`` positions a query at ``pos`` [...] sees in a context of ``ctx`` [...] tokens."""
    j = torch.arange(tokens, device=pos.device)
    p = pos[..., None]
    seen = (j <= p) & (j < ctx[..., None])
    return seen & ((j > p - window) | (j < sinks)) if window else seen


def _attend(q, k, v, seen, scale):
    """q [S, kv heads, n, D], k and v [S, kv heads, tokens, D], seen [S, 1, n or 1, tokens]: softmax over what is seen."""
    s = torch.matmul(q, k.transpose(-1, -2)) * scale
    s = s.masked_fill(~seen, float("-inf"))
    s = (s - s.amax(-1, keepdim=True)).exp()
    return torch.matmul(s, v) / s.sum(-1, keepdim=True)


def _decode(st):
    c = st["case"]
    b, nq, nkv, d = c["seqs"], c["nq"], c["nkv"], c["dim"]
    k, v = _context(st)
    q = st["q"][:, :nq * d].float().view(b, nkv, nq // nkv, d)
    seen = _visible(st["ctx"] - 1, st["ctx"], k.shape[2], c["window"], c["sinks"])[:, None, None]
    return _attend(q, k, v, seen, 1.0 / math.sqrt(d)).reshape(b, nq * d).to(torch.bfloat16)


def _prompt(st):
    c = st["case"]
    n, nq, nkv, d = c["seqs"], c["nq"], c["nkv"], c["dim"]
    g = nq // nkv
    k, v = _context(st)
    cu = st["cu"].long()
    rows = torch.arange(st["most"], device=cu.device)
    at = (cu[:-1, None] + rows).clamp_max(cu[-1] - 1)             # [S, most]: padded rows, the last ones of others
    live = rows < (cu[1:] - cu[:-1])[:, None]
    q = st["q"][:, :nq * d].float()[at].view(n, -1, nkv, g, d).permute(0, 2, 1, 3, 4).reshape(n, nkv, -1, d)
    pos = st["ctx"].long()[:, None] - (cu[1:] - cu[:-1])[:, None] + rows
    seen = _visible(pos, st["ctx"].long()[:, None].expand_as(pos), k.shape[2], c["window"], c["sinks"])
    seen = torch.where(live[..., None], seen, True)               # a padded row is dropped below
    y = _attend(q, k, v, seen[:, None].repeat_interleave(g, 2), 1.0 / math.sqrt(d))
    y = y.view(n, nkv, -1, g, d).permute(0, 2, 1, 3, 4).reshape(n, -1, nq * d).to(torch.bfloat16)
    return y[live]


# ---------------------------------------------------------------- what a pass cannot do without

def _pairs(rows, ctx, window, sinks):
    """Query and key pairs of the last ``rows`` positions of a context."""
    if not window:
        return rows * (2 * ctx - rows + 1) // 2
    return sum(min(p + 1, window) + max(0, min(sinks, p + 1 - window)) for p in range(ctx - rows, ctx))


def work(case):
    c, d, nkv = case, case["dim"], case["nkv"]
    row = 2 * nkv * d * 17 // 32               # cached bytes of a token: keys and values
    plain = 2 * nkv * d * 2                    # the same in bf16
    if c["op"] == "write":
        t, q = c["tokens"], c["nq"] * d
        taken = c["splits"] * 4 * (q + 2 * nkv * d) if c["splits"] else 2 * q + plain
        # in: rows, positions, slots, angles; out: queries, cache; then the rows read back
        return dict(bytes=t * (taken + 16 + 4 * d + 2 * q + row + row + plain), flops=t * (max(1, c["splits"]) + 6) * (q + nkv * d))
    lens = _lengths(c["ctx"], c["seqs"])
    if c["op"] == "read":
        return dict(bytes=sum(lens) * (8 + row + plain), flops=sum(lens) * 2 * nkv * d)
    q = c["nq"] * d
    if c["op"] == "decode":
        seen = [_pairs(1, n, c["window"], c["sinks"]) for n in lens]
        return dict(bytes=sum(seen) * row + c["seqs"] * 4 * q, flops=4 * q * sum(seen))
    rows = [min(n, r) for n, r in zip(lens, _lengths(c["rows"], c["seqs"]))]
    first = [min(n, r + c["window"]) + min(c["sinks"], max(0, n - r - c["window"])) if c["window"] else n for n, r in zip(lens, rows)]
    return dict(bytes=sum(first) * row + sum(rows) * 4 * q, flops=4 * q * sum(_pairs(r, n, c["window"], c["sinks"]) for n, r in zip(lens, rows)))


# ---------------------------------------------------------------- 64 bits

def _stands_for(byte_rows, bs, d, values):
    """The values, 64 bits, of bytes [blocks, heads, 17 bs d / 32] of a cache, written from the format's description: [blocks, heads, bs, d]."""
    n, h, _ = byte_rows.shape
    dev = byte_rows.device
    tok, dims = torch.arange(bs, device=dev)[:, None], torch.arange(d, device=dev)[None, :]
    if values:
        code_at, scale_at = dims // 2 * bs + tok, dims // 32 * bs + tok
    else:
        code_at, scale_at = tok * (d // 2) + dims // 2, dims // 32 * bs + (tok - tok % 16) + 4 * (tok % 4) + tok % 16 // 4
    code = byte_rows[:, :, code_at.reshape(-1)].view(n, h, bs, d)
    code = torch.where(dims % 2 == 1, code >> 4, code & 15)
    low, exponent = (code & 1).double(), ((code >> 1) & 3).double()
    size = torch.where(exponent == 0, low / 2, (1 + low / 2) * torch.exp2(exponent - 1))   # e2m1
    size = torch.where(code >= 8, -size, size)
    scale = torch.exp2(byte_rows[:, :, bs * d // 2 + scale_at.reshape(-1)].view(n, h, bs, d).double() - 127)
    return size * scale


def _nearest(x):
    """bf16 rows [..., D] as the values, 64 bits, that the 4-bit grid keeps of them: the nearest level, the even code of two as near."""
    y = x.double().unflatten(-1, (-1, 32))
    most = y.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(most.clamp_min(2.0 ** -130))) - 2
    e = torch.where(most > 7 * torch.exp2(e), e + 1, e).clamp(SCALE_MIN - 127, SCALE_MAX - 127)
    grid = torch.tensor(LEVELS, device=x.device, dtype=torch.float64)
    a = (y.abs() / torch.exp2(e)).clamp_max(6.0)
    up = torch.searchsorted(grid, a.contiguous()).clamp_max(7)
    down = (up - 1).clamp_min(0)
    to_up, to_down = grid[up] - a, a - grid[down]
    pick = torch.where((to_up < to_down) | ((to_up == to_down) & (up % 2 == 0)), up, down)
    return (torch.sign(y) * grid[pick] * torch.exp2(e)).flatten(-2)


def exact(case, seed):
    st = prepare(case, seed)
    c, op, d, nkv, bs = case, case["op"], case["dim"], case["nkv"], case["block"]
    if op == "write":
        x = (st["partials"].double().sum(0) if c["splits"] else st["rows"]).to(torch.bfloat16).double()
        x = x.view(c["tokens"], c["nq"] + 2 * nkv, d)
        i = torch.arange(d // 2, device=x.device)
        one, two = (i, i + d // 2) if c["mode"] == 0 else (2 * i, 2 * i + 1)
        angle = st["cos_sin"].double()[st["positions"]]
        cos, sin = angle[:, None, :d // 2], angle[:, None, d // 2:]
        turned = x.clone()
        turned[:, :, one] = x[:, :, one] * cos - x[:, :, two] * sin
        turned[:, :, two] = x[:, :, two] * cos + x[:, :, one] * sin
        q, k, v = turned[:, :c["nq"]], turned[:, c["nq"]:c["nq"] + nkv], x[:, c["nq"] + nkv:]
        return dict(q=q.reshape(c["tokens"], -1), k=_nearest(k.to(torch.bfloat16)), v=_nearest(v.to(torch.bfloat16)))
    flat = [t.view(t.shape[0], nkv, -1) for t in (st["k_cache"], st["v_cache"])]
    if op == "read":
        out = []
        for t, values in zip(flat, (False, True)):
            rows = _stands_for(t, bs, d, values).transpose(1, 2).reshape(-1, nkv, d)
            out.append(rows[st["slots"]])
        return dict(k=out[0], v=out[1])
    nq, g, lens = c["nq"], c["nq"] // nkv, st["ctx"].tolist()
    rows = st["rows"] if op == "prompt" else [1] * len(lens)
    out, at = torch.empty(sum(rows), nq, d, device="cuda", dtype=torch.float64), 0
    for i, (n, r) in enumerate(zip(lens, rows)):
        pages = st["table"][i, :-(-n // bs)].long()
        k, v = (_stands_for(t[pages], bs, d, values).transpose(0, 1).reshape(nkv, -1, d)[:, :n] for t, values in zip(flat, (False, True)))
        place, key = torch.arange(n - r, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None, :]
        hidden = key > place
        if c["window"]:
            hidden = hidden | ((key <= place - c["window"]) & (key >= c["sinks"]))
        for h in range(nq):
            q = st["q"][at:at + r, h * d:(h + 1) * d].double()
            p = torch.softmax((q @ k[h // g].t() / math.sqrt(d)).masked_fill(hidden, float("-inf")), -1)
            out[at:at + r, h] = p @ v[h // g]
        at += r
    return out.view(sum(rows), nq * d)
