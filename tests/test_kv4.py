"""The 4-bit paged KV cache (--kv-cache-dtype mxfp4): writers, reader, decode and prompt attention with a window and first tokens
that stay visible, on the CPU engine's operators and (marked gpu) the gfx950 kernels.

The oracle here decodes the cache's bytes from the format's description in 64 bits and attends in 64 bits, without the package's
code. Bytes and read values must be equal. An attention output may be off by what its roundings to bf16 allow: half a step, 2^-8,
of each probability (so 2^-8 of the sum of p |v|) and of the output; the 32-bit sums of up to 2048 products before that are
within 2^-13 of that sum, in the score's exponent included (see ``_check``)."""
import dataclasses
import math

import pytest
import torch

from hipserve.config import PRESETS, EngineConfig
from hipserve.engine.llm_engine import LLMEngine
from hipserve.engine.request import SamplingParams
from hipserve.ops import get_ops, kv4
from hipserve.ops import reference as ref
from hipserve.parallel.comm import TPGroup

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


# ---------------------------------------------------------------- oracle

def _decode_bytes(cache, values):
    """[blocks, heads, block_size, D] float64 from the bytes, element by element of the layout's description."""
    n, h, bs, w = cache.shape
    d = w * 32 // 17
    flat = cache.cpu().reshape(n, h, -1)
    tok, dim = torch.meshgrid(torch.arange(bs), torch.arange(d), indexing="ij")
    code_at = dim // 2 * bs + tok if values else tok * (d // 2) + dim // 2
    place = tok if values else tok // 16 * 16 + 4 * (tok % 4) + tok % 16 // 4
    scale_at = bs * d // 2 + dim // 32 * bs + place
    pick = lambda at: flat[:, :, at.reshape(-1)].view(n, h, bs, d).long()  # noqa: E731
    code, byte = pick(code_at) >> (4 * (dim % 2)) & 15, pick(scale_at)
    y = torch.tensor(LEVELS + [-v for v in LEVELS], dtype=torch.float64)[code] * torch.exp2(byte.double() - 127)
    return torch.where(byte == 255, float("nan"), y)


def _attend(q, k, v, seen, scale):
    """One head, 64 bits: q [r, D], k and v [n, D], seen [r, n] -> (out [r, D], sum of p |v| [r, D])."""
    if not (k.isnan().any() or v.isnan().any()):
        some = seen.any(1, keepdim=True)
        p = torch.softmax((k @ q.T * scale).T.masked_fill(~seen & some, float("-inf")), 1) * some
        return p @ v, p @ v.abs()
    out, size = torch.zeros(len(q), v.shape[1], dtype=torch.float64), torch.zeros(len(q), v.shape[1], dtype=torch.float64)
    for i in range(len(q)):   # row by row, over the seen keys alone
        at = seen[i].nonzero().flatten()
        if len(at):
            p = torch.softmax(k[at] @ q[i] * scale, 0)
            out[i], size[i] = p @ v[at], p @ v[at].abs()
    return out, size


def _oracle(q, kc, vc, tables, rows, ctx, nq, nkv, scale, window, sinks):
    """Sequence i's last rows[i] positions of ctx[i]: (out, size) [sum(rows), nq, D] float64."""
    keys, vals = _decode_bytes(kc, False), _decode_bytes(vc, True)
    nb, _, bs, d = keys.shape
    q, outs, at = q.cpu().double(), [], 0
    for i, (r, n) in enumerate(zip(rows, ctx)):
        j = torch.arange(n)
        page = tables[i].cpu().long()[j // bs] if n else j
        ok = (page >= 0) & (page < nb)
        page = torch.where(ok, page, 0)
        pos = torch.arange(n - r, n)[:, None]
        seen = (j <= pos) & ok
        if window:
            seen &= (j > pos - window) | (j < sinks)
        heads = [_attend(q[at:at + r, h * d:(h + 1) * d], keys[page, h // (nq // nkv), j % bs], vals[page, h // (nq // nkv), j % bs],
                         seen, scale) for h in range(nq)]
        outs.append([torch.stack(x, 1) for x in zip(*heads)])
        at += r
    return [torch.cat(x) for x in zip(*outs)]


def _check(got, want, size):
    """A probability is rounded to bf16 once and the output once: 2^-8 of each (a prompt's sum is that of the rounded probabilities, which
    allows another 2^-8 of the output; held to the same). Scores are sums of 32 bits of up to 128 products of a few
    units, off by under 2^-14 in the exponent, and the sums over the keys add less: together under 2^-11 of the sum of p |v|."""
    got = got.float().cpu().double().view(want.shape)
    assert torch.equal(got.isnan(), want.isnan())
    off = (got - want).abs()
    tol = (2 ** -8 + 2 ** -11) * size + 2 ** -8 * want.abs() + 1e-30
    bad = (off > tol) & ~want.isnan()
    assert not bad.any(), f"off by {(off / tol)[~want.isnan()].max():.3f} of what the roundings allow"


# ---------------------------------------------------------------- inputs

def _random_cache(gen, nb, nkv, bs, d, spread=3):
    """Caches of any codes and of scales around 1."""
    shape = kv4.cache_shape(nb, nkv, bs, d)
    out = []
    for _ in "kv":
        c = torch.randint(0, 256, shape, generator=gen, dtype=torch.uint8).view(nb, nkv, -1)
        c[..., bs * d // 2:] = torch.randint(125 - spread, 125 + spread, (nb, nkv, bs * d // 32), generator=gen).to(torch.uint8)
        out.append(c.view(shape))
    return out


def _tables(gen, ctx, bs, width=None):
    need = [max(1, -(-n // bs)) for n in ctx]
    width = width or max(need)
    nb = sum(need) + 2
    ids = torch.randperm(nb, generator=gen).int()
    t = torch.zeros(len(ctx), width, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = ids[at:at + n]
        at += n
    return nb, t


def _decode(ops, dev, q, kc, vc, bt, ctx, nq, nkv, d, bs, part, window, sinks, out=None, out16=None):
    b = q.shape[0]
    parts = max(1, -(-bt.shape[1] * bs // part))
    to, tm = torch.full((b, nq, parts, d), float("nan"), device=dev), torch.full((b, nq, parts, 2), float("nan"), device=dev)
    out = torch.full((b, nq * d), float("nan"), device=dev, dtype=torch.bfloat16) if out is None else out
    kw = {} if out16 is None else dict(out16=out16)
    ops.paged_decode(out, q.to(dev), kc.to(dev), vc.to(dev), bt.to(dev), torch.as_tensor(ctx, dtype=torch.int32).to(dev), to, tm, nq, nkv,
                     part, 1 / math.sqrt(d), window, sinks=sinks, **kw)
    return out


def _tiles(rows):
    return torch.tensor([(i, r) for i, n in enumerate(rows) for r in range(0, n, 128)], dtype=torch.int32).view(-1, 2)


def _prompt(ops, dev, q, kc, vc, bt, rows, ctx, nq, nkv, d, window, sinks, out=None):
    cu = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], dtype=torch.int32)
    out = torch.full((q.shape[0], nq * d), float("nan"), device=dev, dtype=torch.bfloat16) if out is None else out
    ops.prefill_attention(out, q.to(dev), kc.to(dev), vc.to(dev), bt.to(dev), cu.to(dev), torch.tensor(ctx, dtype=torch.int32).to(dev),
                          _tiles(rows).to(dev), nq, nkv, 1 / math.sqrt(d), window, sinks=sinks)
    return out


def _queries(gen, rows, nq, nkv, d):
    """Rows of a merged projection, as the engine passes them."""
    return torch.randn(rows, (nq + 2 * nkv) * d, generator=gen).to(torch.bfloat16)


# ---------------------------------------------------------------- the format

def test_quantise_takes_the_nearest_level():
    """Every value is within half a step of its neighbours on the grid, or beyond the largest level by at most a sixth; ties go to
    the even code."""
    gen = torch.Generator().manual_seed(0)
    x = (torch.randn(512, 96, generator=gen) * torch.exp2(torch.randint(-60, 60, (512, 1), generator=gen).float())).to(torch.bfloat16)
    codes, scales = kv4.quantise(x)
    s = torch.exp2(scales.double() - 127).repeat_interleave(32, -1)
    levels = torch.tensor(LEVELS, dtype=torch.float64)
    a = x.double().abs() / s
    assert a.max() <= 7 and (a.unflatten(-1, (-1, 32)).amax(-1) > 3).all()
    dist = (a[..., None] - levels).abs()
    assert torch.equal(dist.gather(-1, (codes & 7).long()[..., None]).squeeze(-1), dist.min(-1).values)
    tied = (dist == dist.min(-1, keepdim=True).values).sum(-1) == 2
    assert tied.any() and not (codes[tied] & 1).any()
    assert torch.equal(codes >= 8, torch.signbit(x))
    assert torch.equal(kv4.dequantise(codes, scales).double(), torch.where(codes >= 8, -1.0, 1.0) * levels[(codes & 7).long()] * s)


def test_quantise_at_the_ends_of_the_range():
    big = torch.finfo(torch.bfloat16).max
    x = torch.zeros(7, 64, dtype=torch.bfloat16)
    x[0, 3] = big                     # reads as 6 * 2^125
    x[1, 3] = 2.0 ** -133             # below half of the smallest value, 2^-120: zero
    x[2, 3] = 2.0 ** -118
    x[3, 3], x[3, 40] = float("nan"), 2.0
    x[4, 3], x[4, 40] = float("-inf"), -3.0
    x[5, 3] = 7.0                     # exactly 7 units: stays under the smaller scale and reads as 6
    x[6, 3] = 7.03125                 # the next bf16: the scale doubles
    codes, scales = kv4.quantise(x)
    y = kv4.dequantise(codes, scales)
    assert scales[:, 0].tolist() == [252, 8, 9 - 1, 255, 255, 127, 128]
    assert y[0, 3] == 6 * 2.0 ** 125 and y[1].abs().max() == 0 and y[2, 3] == 2.0 ** -118
    assert y[3:5, :32].isnan().all() and y[3, 40] == 2 and y[4, 40] == -3 and not codes[3:5, :32].any()
    assert y[5, 3] == 6 and y[6, 3] == 8 and not y.isinf().any()


# ---------------------------------------------------------------- writing and reading

def _values(gen, t, n):
    x = torch.randn(t, n, generator=gen)
    x[:, 5::48] *= 6
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("mode", [0, 1])
@pytest.mark.parametrize("nq,nkv,d,bs", [(32, 8, 128, 16), (5, 5, 96, 32), (14, 2, 64, 64), (3, 1, 128, 256)])
@pytest.mark.parametrize("t,order", [(1, "in order"), (37, "anywhere"), (131, "in order"), (260, "aligned"), (703, "in order"),
                                     (720, "aligned")])
def test_write_holds_the_quantised_rows(dev, mode, nq, nkv, d, bs, t, order):
    """The cache's bytes are those of the rows that a bf16 cache holds after the same call, quantised, every other byte is left, and
    the queries are rotated to the same bits; rows in a wider buffer, slots below 0 and behind the cache."""
    gen = torch.Generator().manual_seed(t + d)
    ops, nb = get_ops(dev), 2 + (t + 600) // bs
    wide = _values(gen, t, (nq + 2 * nkv) * d + 16).to(dev)
    pos = torch.randint(0, 4000, (t,), generator=gen).to(dev)
    slots = {"anywhere": torch.randperm(nb * bs, generator=gen)[:t], "in order": torch.arange(t) + bs + 5,
             "aligned": torch.arange(t) + bs}[order].to(dev)
    if t > 20:
        slots[3], slots[17] = -1, nb * bs
    cs = ref.rope_cos_sin(d, 4096, 500000.0).to(dev)
    kc, vc = (c.to(dev) for c in _random_cache(gen, nb, nkv, bs, d))
    before = kc.clone(), vc.clone()
    kb = torch.zeros(nb + 1, nkv, bs, d, device=dev, dtype=torch.bfloat16)
    vb = torch.zeros(nb + 1, nkv, d, bs, device=dev, dtype=torch.bfloat16)
    plain, rows = wide.clone(), wide.clone()
    cols = (nq + 2 * nkv) * d
    ops.rope_cache(plain[:, :cols], pos, slots, cs, kb, vb, nq, nkv, d, mode)
    ops.rope_cache(rows[:, :cols], pos, slots, cs, kc, vc, nq, nkv, d, mode)
    assert torch.equal(rows[:, : nq * d], plain[:, : nq * d])
    assert torch.equal(rows[:, nq * d:], wide[:, nq * d:])
    ok = (slots >= 0) & (slots < nb * bs)
    s = slots[ok].cpu()
    want = before[0].cpu(), before[1].cpu()
    for c, rows_of, values in zip(want, (kb[slots[ok] // bs, :, slots[ok] % bs], vb[slots[ok] // bs, :, :, slots[ok] % bs]), (False, True)):
        codes, scales = kv4.quantise(rows_of.cpu())
        flat = c.view(nb, nkv, -1)
        for i, sl in enumerate(s.tolist()):   # byte by byte of the layout's description
            o, hb = sl % bs, flat[sl // bs]
            packed = codes[i, :, 0::2] | (codes[i, :, 1::2] << 4)
            if values:
                hb[:, o:bs * d // 2:bs] = packed
                hb[:, bs * d // 2 + o::bs] = scales[i]
            else:
                hb[:, o * d // 2:(o + 1) * d // 2] = packed
                hb[:, bs * d // 2 + o // 16 * 16 + 4 * (o % 4) + o % 16 // 4::bs] = scales[i]
    assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("mode", [0, 1])
@pytest.mark.parametrize("nq,nkv,d,bs", [(32, 8, 128, 16), (6, 6, 96, 32), (14, 2, 64, 256), (9, 3, 128, 64)])
@pytest.mark.parametrize("times", [1, 5])
def test_write_and_read_of_ragged_prompts(dev, mode, nq, nkv, d, bs, times):
    """Prompt steps of many rows, few and many of them for the writers: sequences that begin anywhere in the step and in a page, single rows, whole pages, rows of no slot
    between them, pages in any order. Written and read rows are the quantised rows of the same call on a bf16 cache."""
    gen = torch.Generator().manual_seed(bs)
    ops, lens = get_ops(dev), [(0, 70), (5, 6), (0, 1), (3, 100), (16, 48), (0, 131), (9, 10), (0, 16), (250, 300)] * times
    nb = sum(-(-e // bs) for _, e in lens) + 4
    pages = iter(torch.randperm(nb, generator=gen).tolist())
    slots = []
    for first, end in lens:
        own = [next(pages) for _ in range(-(-end // bs))]
        slots += [own[p // bs] * bs + p % bs for p in range(first, end)] + [-1] * (first % 2)
    last = next(pages)
    slots += [last * bs + o for o in (3, 1, 2, 0, 4)]      # backwards and forwards within a page
    t = len(slots)
    assert t > 390 * times
    slots = torch.tensor(slots).to(dev)
    n = (nq + 2 * nkv) * d
    x = _values(gen, t, n).to(dev)
    pos, cs = torch.randint(0, 500, (t,), generator=gen).to(dev), ref.rope_cos_sin(d, 512, 10000.0).to(dev)
    kb = torch.zeros(nb, nkv, bs, d, device=dev, dtype=torch.bfloat16)
    vb = torch.zeros(nb, nkv, d, bs, device=dev, dtype=torch.bfloat16)
    kc, vc = (c.to(dev) for c in _random_cache(gen, nb, nkv, bs, d))
    want = [kc.cpu().clone(), vc.cpu().clone()]
    plain, rows = x.clone(), x.clone()
    ops.rope_cache(plain, pos, slots, cs, kb, vb, nq, nkv, d, mode)
    ops.rope_cache(rows, pos, slots, cs, kc, vc, nq, nkv, d, mode)
    assert torch.equal(rows[:, : nq * d], plain[:, : nq * d])
    ok = slots >= 0
    s = slots[ok]
    held = kb[s // bs, :, s % bs].cpu(), vb[s // bs, :, :, s % bs].cpu()
    for c, r, values in zip(want, held, (False, True)):
        kv4.store(c, s.cpu(), r, values)
    assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1])
    k, v = (torch.full((t, nkv, d), 5.0, device=dev, dtype=torch.bfloat16) for _ in "kv")
    ops.read_cache(k, v, kc, vc, slots)
    for got, r in zip((k, v), held):
        assert torch.equal(got[ok].cpu(), kv4.dequantise(*kv4.quantise(r)))
        assert not got[~ok].any()


@pytest.mark.gpu
@pytest.mark.parametrize("t,splits", [(1, 1), (5, 3), (64, 8), (100, 17)])
@pytest.mark.parametrize("extra", ["plain", "bias", "norm", "neighbours"])
@pytest.mark.parametrize("nq,nkv,d", [(32, 8, 128), (14, 2, 64), (6, 6, 96)])
def test_write_of_partials(t, splits, extra, nq, nkv, d):
    """From a decode step's split-K partials: as the bf16 cache's writer, rounding for rounding."""
    if extra == "norm" and d == 96:
        pytest.skip("no writer takes norms of heads of 96")
    gen = torch.Generator().manual_seed(t)
    ops, bs, nb = get_ops("cuda"), 16, 40
    n = (nq + 2 * nkv) * d
    ws = torch.randn(splits, t, n, generator=gen).cuda()
    pos, slots = torch.randint(0, 4000, (t,), generator=gen).cuda(), torch.randperm(nb * bs, generator=gen)[:t].cuda()
    cs = ref.rope_cos_sin(d, 4096, 10000.0).cuda()
    opts = dict(bias=torch.randn(n, generator=gen).to(torch.bfloat16).cuda()) if extra == "bias" else {}
    if extra == "norm":
        opts = dict(q_w=torch.rand(d, generator=gen).cuda() + 0.5, k_w=torch.rand(d, generator=gen).cuda() + 0.5, eps=1e-6)
    kb = torch.zeros(nb, nkv, bs, d, device="cuda", dtype=torch.bfloat16)
    vb = torch.zeros(nb, nkv, d, bs, device="cuda", dtype=torch.bfloat16)
    kc, vc = (torch.zeros(kv4.cache_shape(nb, nkv, bs, d), device="cuda", dtype=torch.uint8) for _ in "kv")
    got, want = (torch.zeros(t, n, device="cuda", dtype=torch.bfloat16) for _ in "gw")
    mode = 1 if extra == "neighbours" else 0
    ops.splitk_rope_cache(want, ws, splits, pos, slots, cs, kb, vb, nq, nkv, d, mode, **opts)
    ops.splitk_rope_cache(got, ws, splits, pos, slots, cs, kc, vc, nq, nkv, d, mode, **opts)
    assert torch.equal(got[:, : nq * d], want[:, : nq * d])
    for cache, rows, values in ((kc, kb[slots // bs, :, slots % bs], False), (vc, vb[slots // bs, :, :, slots % bs], True)):
        fresh = torch.zeros_like(cache)
        kv4.store(fresh, slots, rows, values)
        assert torch.equal(cache, fresh)


@pytest.mark.gpu
def test_write_quantises_every_bf16_value_as_the_reference():
    """All 65536 values of bf16, NaNs and infinities among them, in groups of neighbours and of strangers, as V rows."""
    ops, nkv, d, bs = get_ops("cuda"), 8, 128, 16
    bits = torch.arange(65536, dtype=torch.int32)
    gen = torch.Generator().manual_seed(3)
    for order in (bits, bits[torch.randperm(65536, generator=gen)], (bits & 0x8000) | 0x3c00 | (bits * 7 & 0x3ff)):
        v = order.to(torch.int16).view(torch.bfloat16).view(-1, nkv * d).cuda()
        t = v.shape[0]
        qkv = torch.cat((torch.zeros(t, nkv * d, device="cuda", dtype=torch.bfloat16), v), 1)
        kc, vc = (torch.zeros(kv4.cache_shape(8, nkv, bs, d), device="cuda", dtype=torch.uint8) for _ in "kv")
        slots = torch.arange(t, device="cuda") + 16
        cs = ref.rope_cos_sin(d, 16, 10000.0).cuda()
        ops.rope_cache(qkv, torch.zeros(t, device="cuda", dtype=torch.long), slots, cs, kc, vc, 0, nkv, d, 0)
        want = torch.zeros(vc.shape, dtype=torch.uint8)
        kv4.store(want, slots.cpu(), v.view(t, nkv, d).cpu(), True)
        assert torch.equal(vc.cpu(), want)
        k, v2 = (torch.empty(t, nkv, d, device="cuda", dtype=torch.bfloat16) for _ in "kv")
        ops.read_cache(k, v2, kc, vc, slots)
        assert torch.equal(v2.cpu().float().nan_to_num(7.0), kv4.load(want, slots.cpu(), True).float().nan_to_num(7.0))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("nkv,d,bs", [(8, 128, 16), (3, 96, 32), (2, 64, 128)])
@pytest.mark.parametrize("t,order", [(0, "in order"), (1, "anywhere"), (16, "aligned"), (100, "anywhere"), (333, "in order")])
def test_read_gives_the_values(dev, nkv, d, bs, t, order):
    gen = torch.Generator().manual_seed(t + bs)
    nb = 2 + 400 // bs
    kc, vc = _random_cache(gen, nb, nkv, bs, d, spread=60)
    kc.view(nb, nkv, -1)[1, 0, bs * d // 2 + 3] = 255
    vc.view(nb, nkv, -1)[1, 0, bs * d // 2 + 5] = 255
    slots = {"anywhere": torch.randint(0, nb * bs, (t,), generator=gen), "in order": torch.arange(t) + 7,
             "aligned": torch.arange(t) + bs}[order]
    if t > 20:
        slots[2], slots[19], slots[20] = -1, nb * bs, slots[5]   # a slot read twice
    k, v = (torch.full((t + 1, nkv * d + 8), 7.0, dtype=torch.bfloat16, device=dev) for _ in "kv")
    ko, vo = (x[:t, :nkv * d].unflatten(1, (nkv, d)) for x in (k, v))
    get_ops(dev).read_cache(ko, vo, kc.to(dev), vc.to(dev), slots.to(dev))
    ok = (slots >= 0) & (slots < nb * bs)
    at = torch.where(ok, slots, 0)
    for got, cache, values in ((ko, kc, False), (vo, vc, True)):
        want = torch.where(ok[:, None, None], _decode_bytes(cache, values)[at // bs, :, at % bs], 0.0)
        assert torch.equal(got.cpu().double().nan_to_num(12345.0), want.nan_to_num(12345.0))
    assert (k[t] == 7).all() and (k[:, nkv * d:] == 7).all()


# ---------------------------------------------------------------- attention

HEADS = [(32, 8, 128, 16), (16, 1, 128, 64), (7, 7, 96, 16), (28, 4, 64, 32), (12, 4, 96, 256)]
WINDOWS = [(0, 0), (100, 0), (100, 4), (64, 70), (1, 1), (1000, 3), (200, 150)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("nq,nkv,d,bs", HEADS)
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("part", [64, 512])
def test_decode(dev, nq, nkv, d, bs, window, sinks, part):
    """Lengths from none to many partitions, odd ones, ones that end inside a page and a chunk; a row of no keys is zeros."""
    gen = torch.Generator().manual_seed(nq + part)
    ctx = [1, 0, 15, 16, 17, 63, 64, 65, 130, 600, 1300, 257]
    nb, bt = _tables(gen, ctx, bs)
    kc, vc = _random_cache(gen, nb, nkv, bs, d)
    q = _queries(gen, len(ctx), nq, nkv, d)
    got = _decode(get_ops(dev), dev, q, kc, vc, bt, ctx, nq, nkv, d, bs, part, window, sinks)
    want, size = _oracle_rows(q, kc, vc, bt, ctx, nq, nkv, d, window, sinks)
    _check(got, want, size)
    assert not got[1].any()


def _oracle_rows(q, kc, vc, bt, ctx, nq, nkv, d, window, sinks):
    """One row a sequence, zeros for those without keys."""
    live = [i for i, n in enumerate(ctx) if n]
    w, s = _oracle(q[live], kc, vc, bt[live], [1] * len(live), [ctx[i] for i in live], nq, nkv, 1 / math.sqrt(d), window, sinks)
    out = [torch.zeros(len(ctx), nq, d, dtype=torch.float64) for _ in "ws"]
    out[0][live], out[1][live] = w, s
    return out


SEQS = [([1], [1]), ([5, 40, 1, 130], [5, 300, 64, 130]), ([64, 128, 33], [64, 129, 500]), ([257, 3], [321, 1000])]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("nq,nkv,d,bs", HEADS + [(6, 2, 128, 16), (8, 1, 64, 16), (10, 2, 128, 16)])
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("rows,ctx", SEQS)
def test_prompt(dev, nq, nkv, d, bs, window, sinks, rows, ctx):
    """Whole prompts and portions behind cached tokens; the rows behind the last sequence are left as they were."""
    if dev == "cpu" and (nq, window) in ((32, 1000), (16, 64), (28, 100)):
        pytest.skip("covered by the other heads")
    gen = torch.Generator().manual_seed(nq + sum(rows))
    nb, bt = _tables(gen, ctx, bs)
    kc, vc = _random_cache(gen, nb, nkv, bs, d)
    q = _queries(gen, sum(rows) + 3, nq, nkv, d)
    out = torch.full((sum(rows) + 3, nq * d + 8), 3.0, device=dev, dtype=torch.bfloat16)
    _prompt(get_ops(dev), dev, q, kc, vc, bt, rows, ctx, nq, nkv, d, window, sinks, out=out[:, :nq * d])
    want, size = _oracle(q, kc, vc, bt, rows, ctx, nq, nkv, 1 / math.sqrt(d), window, sinks)
    _check(out[:sum(rows), :nq * d].reshape(-1, nq, d), want, size)
    assert (out[sum(rows):] == 3).all() and (out[:, nq * d:] == 3).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("nq,nkv,d,bs", [(32, 8, 128, 16), (7, 7, 96, 16), (28, 4, 64, 32), (16, 1, 96, 64)])
@pytest.mark.parametrize("powers", [(0, 0, -24, 24), (20, -12, 0, 8), (-24, 0, 16, -8)])
def test_queries_small_where_keys_are_large(dev, nq, nkv, d, bs, powers):
    """The query's 32 dims of a key's group 2^power, the key's 2^-power: every group says as much of the score as in the other tests.
    Within a group the query's magnitudes are within a factor of 2^8, so a sum of two e4m3 numbers has all their bits and the usual bound holds."""
    gen = torch.Generator().manual_seed(nq + powers[0])
    ctx = [1, 40, 300, 517]
    nb, bt = _tables(gen, ctx, bs)
    kc, vc = _random_cache(gen, nb, nkv, bs, d, spread=1)
    size = torch.rand(404, nq + 2 * nkv, d, generator=gen) * 2 + 2.0 ** -6
    q = size * (torch.randint(0, 2, size.shape, generator=gen) * 2 - 1)
    for g in range(d // 32):
        q[..., 32 * g:32 * g + 32] *= 2.0 ** powers[g]
        by_group = kc.view(nb, nkv, -1)[..., bs * d // 2:].view(nb, nkv, d // 32, bs)
        by_group[:, :, g] -= powers[g] % 256
    q = q.flatten(1).to(torch.bfloat16)
    rows = [1, 3, 300, 100]
    want, size = _oracle(q, kc, vc, bt, rows, ctx, nq, nkv, 1 / math.sqrt(d), 0, 0)
    _check(_prompt(get_ops(dev), dev, q[:404], kc, vc, bt, rows, ctx, nq, nkv, d, 0, 0), want, size)
    want, size = _oracle(q[:4], kc, vc, bt, [1] * 4, ctx, nq, nkv, 1 / math.sqrt(d), 0, 0)
    for part in (64, 1024):
        _check(_decode(get_ops(dev), dev, q[:4], kc, vc, bt, ctx, nq, nkv, d, bs, part, 0, 0), want, size)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("dim", [1, 31, 40, 63])
def test_small_values_of_a_query_beside_a_large_one(dev, d, dim):
    """All 128 mantissas of 2^-8 .. 2^-20 beside a largest value of 1 (the one that leaves the fewest bits) in the same 32 dims: the first key
    meets the small value alone, with a score of 1 to 3, the second one nothing.

    Two e4m3 numbers hold a value within 2^-21 of the largest, exactly from 2^-13 of it on; the score is one product. The output is
    6 / (1 + exp(-score)), of slope 6 / 4 at most."""
    nq, nkv, bs, low = 16, 1, 16, range(8, 21)
    kc, vc = (torch.zeros(kv4.cache_shape(len(low), nkv, bs, d), dtype=torch.uint8) for _ in "kv")
    k, v = kc.view(len(low), -1), vc.view(len(low), -1)
    k[:, bs * d // 2:], v[:, bs * d // 2:] = 127, 127
    k[:, dim // 2] = 7 << 4 * (dim % 2)                        # token 0: 6 of a unit that makes the score
    v[:, :bs * d // 2:bs] = 0x77                               # token 0: 6, token 1: 0
    scale, up = 1 / math.sqrt(d), [r + 1 for r in low]         # 6 2^-r 2^(r + 1) / sqrt(d): from 1.06 on
    for i, b in enumerate(up):
        k[i, bs * d // 2 + dim // 32 * bs] = 127 + b
    x = torch.tensor([[(1 + m / 128) * 2.0 ** -r for m in range(128)] for r in low], dtype=torch.float64)
    n = x.numel() // nq
    q = torch.zeros(n, nq + 2 * nkv, d)
    q[:, :nq, dim] = x.view(n, nq).float()
    q[:, :nq, dim // 32 * 32 + 2] = 1.0
    q = q.flatten(1).to(torch.bfloat16)
    bt = torch.arange(len(low), dtype=torch.int32).repeat_interleave(128 // nq)[:, None]
    unit = 6 * torch.exp2(torch.tensor(up, dtype=torch.float64)) * scale
    want = 6 / (1 + torch.exp(-x * unit[:, None]))
    lost = torch.where(x < 2.0 ** -13, 2.0 ** -21, 0.0) * unit[:, None]
    # beside the lost bits: the probability's and the output's rounding, and the 32-bit steps of _check
    tol = (6 / 4 * lost + (2 ** -8 + 2 ** -11 + 2 ** -8) * want).view(n, nq, 1)
    for got in (_decode(get_ops(dev), dev, q, kc, vc, bt, [2] * n, nq, nkv, d, bs, 64, 0, 0),
                _prompt(get_ops(dev), dev, q, kc, vc, bt, [1] * n, [2] * n, nq, nkv, d, 0, 0)):
        off = (got.float().cpu().double().view(n, nq, d) - want.view(n, nq, 1)).abs()
        assert (off <= tol).all(), f"off by {(off / tol).max():.3f} of what the query's parts allow"


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("power", [127, 126, 0, -100, -111, -117])
def test_queries_from_the_smallest_to_the_largest(dev, d, power):
    """2^power with each of 128 mantissas against one key, 2^power alone against another, all but exact: scores m / sqrt(d) apart, an
    output of 6 / (1 + exp(-m / sqrt(d))) whose only errors are the roundings of probability and output and a few 32-bit steps."""
    nq, nkv, bs = 16, 1, 16
    kc, vc = (torch.zeros(kv4.cache_shape(1, nkv, bs, d), dtype=torch.uint8) for _ in "kv")
    k, v = kc.view(-1), vc.view(-1)
    k[bs * d // 2:], v[bs * d // 2:] = 127 + 8 - power, 127
    k[3 // 2] = 1 << 4                                         # token 0: 0.5 2^(8 - power) of dim 3
    k[d // 2 + 40 // 2] = 1                                    # token 1: of dim 40
    v[:bs * d // 2:bs] = 0x77                                  # token 0: 6, token 1: 0
    m = torch.arange(128, dtype=torch.float64).view(8, nq)
    q = torch.zeros(8, nq + 2 * nkv, d, dtype=torch.float64)
    q[:, :nq, 3], q[:, :nq, 40] = (1 + m / 128) * 2.0 ** power, 2.0 ** power
    q = q.flatten(1).to(torch.bfloat16)
    bt = torch.zeros(8, 1, dtype=torch.int32)
    want = (6 / (1 + torch.exp(-m / math.sqrt(d)))).view(8, nq, 1)
    for got in (_decode(get_ops(dev), dev, q, kc, vc, bt, [2] * 8, nq, nkv, d, bs, 64, 0, 0),
                _prompt(get_ops(dev), dev, q, kc, vc, bt, [1] * 8, [2] * 8, nq, nkv, d, 0, 0)):
        off = (got.float().cpu().double().view(8, nq, d) - want).abs()
        assert (off <= (2 ** -8 + 2 ** -11 + 2 ** -8) * want).all()


def _chunks(n, window, sinks):
    """Chunks of 64 keys that a decode row of n keys takes: those of the first keys, then the window's."""
    lo = max(0, n - window) if window else 0
    return min(-(-min(sinks, lo) // 64), lo // 64) + -(-n // 64) - lo // 64 if n else 0


def _run_chunks(ctx, nkv, parts, window, sinks):
    """Chunks of a decode workgroup's run, a fourth of them a wave's: by what 512 workgroups take, or the workspace's partitions."""
    count = [_chunks(n, window, sinks) for n in ctx]
    slots = max(512 - len(ctx) * nkv // 2, 256)
    return -(-max(sum(count) * nkv // slots + 1, -(-max(count) // parts)) // 4) * 4


def _spoil(caches, bt, bs, d, seq, tok, head, group):
    """A value group's scale byte to that of NaN."""
    v = caches[1].view(caches[1].shape[0], caches[1].shape[1], -1)
    v[int(bt[seq, tok // bs]), head, bs * d // 2 + group * bs + tok % bs] = 255


LONG = [(32, 8, 128, 16), (16, 1, 128, 64), (7, 7, 96, 16), (28, 4, 64, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nkv,d,bs", LONG)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1100, 70), (900, 0)])
def test_decode_of_many_chunks_a_wave(nq, nkv, d, bs, window, sinks):
    """One partition a row: each of the four waves takes up to eight chunks, its two sets of registers in turn; odd ends, and a NaN value and a
    page that is none in late chunks."""
    gen = torch.Generator().manual_seed(nq + d)
    ctx = [1200, 1217, 2000, 770, 0, 1, 1151]
    nb, bt = _tables(gen, ctx, bs)
    kc, vc = _random_cache(gen, nb, nkv, bs, d)
    _spoil((kc, vc), bt, bs, d, 1, 1180, nkv - 1, 1)
    bt[2, 1900 // bs] = -1
    q = _queries(gen, len(ctx), nq, nkv, d)
    assert bt.shape[1] * bs <= 2048 and _chunks(2000, window, sinks) >= 4 * 3
    want, size = _oracle_rows(q, kc, vc, bt, ctx, nq, nkv, d, window, sinks)
    assert want[1].isnan().any()
    _check(_decode(get_ops("cuda"), "cuda", q, kc, vc, bt, ctx, nq, nkv, d, bs, 2048, window, sinks), want, size)


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nkv,d,bs", LONG)
@pytest.mark.parametrize("window,sinks", [(0, 0), (4300, 70)])
def test_decode_of_many_chunks_a_run(nq, nkv, d, bs, window, sinks):
    """Rows in few partitions of many chunks each; a NaN value and pages that are none in the last run and in one between."""
    gen = torch.Generator().manual_seed(nq + d + 1)
    ctx = [8200, 4999, 130]
    nb, bt = _tables(gen, ctx, bs)
    kc, vc = _random_cache(gen, nb, nkv, bs, d)
    _spoil((kc, vc), bt, bs, d, 0, 8150, 0, 0)
    bt[0, 6000 // bs], bt[1, 4900 // bs] = nb, -1
    q = _queries(gen, len(ctx), nq, nkv, d)
    parts = -(-bt.shape[1] * bs // 2048)
    assert _run_chunks(ctx, nkv, parts, window, sinks) >= 4 * 3
    want, size = _oracle(q, kc, vc, bt, [1] * 3, ctx, nq, nkv, 1 / math.sqrt(d), window, sinks)
    assert want[0].isnan().any()
    _check(_decode(get_ops("cuda"), "cuda", q, kc, vc, bt, ctx, nq, nkv, d, bs, 2048, window, sinks), want, size)


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nkv,d,bs,n", [(4, 1, 128, 16, 8300), (16, 1, 96, 32, 10500), (2, 1, 64, 16, 17000)])
def test_decode_of_more_runs_than_the_merge_takes_at_once(nq, nkv, d, bs, n):
    """One kv head: a row's runs are as many as 512 workgroups allow, more than the merge's lanes take four each."""
    gen = torch.Generator().manual_seed(n)
    ctx = [n, 700]
    nb, bt = _tables(gen, ctx, bs)
    kc, vc = _random_cache(gen, nb, nkv, bs, d)
    q = _queries(gen, 2, nq, nkv, d)
    runs = -(-_chunks(n, 0, 0) // _run_chunks(ctx, nkv, -(-bt.shape[1] * bs // 64), 0, 0))
    assert runs > 4 * (256 // (d // 4))
    want, size = _oracle(q, kc, vc, bt, [1, 1], ctx, nq, nkv, 1 / math.sqrt(d), 0, 0)
    _check(_decode(get_ops("cuda"), "cuda", q, kc, vc, bt, ctx, nq, nkv, d, bs, 64, 0, 0), want, size)


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nkv,d,bs", [(4, 1, 128, 16), (4, 2, 64, 32), (3, 3, 96, 16)])
@pytest.mark.parametrize("rows", [65, 130, 256])
@pytest.mark.parametrize("part,window,sinks", [(64, 0, 0), (64, 150, 4), (1024, 0, 0)])
def test_decode_of_many_rows(nq, nkv, d, bs, rows, part, window, sinks):
    """More rows than a wave's lanes work the runs out for at once: ragged lengths, many of them none, one far longer than the others."""
    gen = torch.Generator().manual_seed(rows + part + nq)
    ctx = torch.randint(0, 300, (rows,), generator=gen)
    ctx[torch.rand(rows, generator=gen) < 0.3] = 0
    ctx[rows - 3], ctx[0], ctx[64] = 1000, 0, 290
    ctx = ctx.tolist()
    nb, bt = _tables(gen, ctx, bs)
    kc, vc = _random_cache(gen, nb, nkv, bs, d)
    q = _queries(gen, rows, nq, nkv, d)
    want, size = _oracle_rows(q, kc, vc, bt, ctx, nq, nkv, d, window, sinks)
    got = _decode(get_ops("cuda"), "cuda", q, kc, vc, bt, ctx, nq, nkv, d, bs, part, window, sinks)
    _check(got, want, size)
    assert not got[torch.tensor(ctx) == 0].any()


def _dense(rows, ctx, nq, nkv, bs, width, window, sinks):
    """Whether the prompt kernel takes a call's workgroups tile by tile (else those of a tile come apart, as few rows and split keys have them)."""
    g, tiles = nq // nkv, sum(-(-r // 128) for r in rows)
    heads = next(h for h in (8, 4, 2, 1) if g % h == 0)
    qr, slots = (128, 512) if heads == 1 else (256 // heads, 256)
    wgs = tiles * (128 // qr) * (nq // heads)
    live = min(wgs, (sum(rows) // qr + len(rows)) * (nq // heads))
    seen = min(width * bs, window + sinks + qr + 128) if window else width * bs
    splits = 1 if wgs > 2048 else max(1, min(slots // live, seen // 64 // 8))
    return splits == 1 and 4 * sum(rows) > 3 * 128 * tiles


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nkv,d,bs", [(32, 2, 128, 16), (16, 2, 96, 32), (8, 1, 64, 16), (16, 4, 128, 64), (8, 4, 128, 16), (4, 2, 96, 16),
                                         (6, 6, 128, 16), (5, 1, 64, 32), (10, 2, 96, 16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 70), (130, 0)])
@pytest.mark.parametrize("rows,ctx", [([256, 384, 127], [256, 900, 400]), ([640], [890])])
def test_full_prompt_steps(nq, nkv, d, bs, window, sinks, rows, ctx):
    """Tiles full of rows, behind a cached beginning or not, for 16, 8, 4, 2, 1 and 5 queries a kv head; a NaN value and a page that is none."""
    gen = torch.Generator().manual_seed(nq + d + len(rows))
    nb, bt = _tables(gen, ctx, bs)
    assert _dense(rows, ctx, nq, nkv, bs, bt.shape[1], window, sinks) and sum(-(-r // 128) for r in rows) >= 5
    kc, vc = _random_cache(gen, nb, nkv, bs, d)
    _spoil((kc, vc), bt, bs, d, 0, 250, nkv - 1, d // 32 - 1)
    bt[-1, 300 // bs] = -1
    q = _queries(gen, sum(rows) + 2, nq, nkv, d)
    out = torch.full((sum(rows) + 2, nq * d), 3.0, device="cuda", dtype=torch.bfloat16)
    _prompt(get_ops("cuda"), "cuda", q, kc, vc, bt, rows, ctx, nq, nkv, d, window, sinks, out=out)
    want, size = _oracle(q, kc, vc, bt, rows, ctx, nq, nkv, 1 / math.sqrt(d), window, sinks)
    assert want.isnan().any()
    _check(out[:-2], want, size)
    assert (out[-2:] == 3).all()


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nkv,d,bs", [(32, 8, 128, 16), (16, 1, 128, 64), (7, 7, 96, 16), (14, 7, 64, 32), (28, 4, 96, 256)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (2000, 70), (700, 0)])
@pytest.mark.parametrize("rows,ctx", [([1], [4100]), ([3, 37, 129, 20], [4097, 2500, 700, 20]), ([64, 8, 2], [512, 513, 1100])])
def test_few_rows_over_long_contexts(nq, nkv, d, bs, window, sinks, rows, ctx):
    """Rows whose keys are split over workgroups, beside others that are not; a NaN value and a page that is none in one part alone."""
    gen = torch.Generator().manual_seed(nq + len(rows))
    nb, bt = _tables(gen, ctx, bs)
    kc, vc = _random_cache(gen, nb, nkv, bs, d)
    n = ctx[0]
    bt[0, n // 4 // bs] = -1
    tok = n - 40
    vc.view(nb, nkv, -1)[int(bt[0, tok // bs]), nkv - 1, bs * d // 2 + bs + tok % bs] = 255
    q = _queries(gen, sum(rows) + 1, nq, nkv, d)
    want, size = _oracle(q, kc, vc, bt, rows, ctx, nq, nkv, 1 / math.sqrt(d), window, sinks)
    assert want.isnan().any()
    out = torch.full((sum(rows) + 1, nq * d), 3.0, device="cuda", dtype=torch.bfloat16)
    _prompt(get_ops("cuda"), "cuda", q, kc, vc, bt, rows, ctx, nq, nkv, d, window, sinks, out=out)
    _check(out[:-1], want, size)
    assert (out[-1] == 3).all()


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nkv,d", [(16, 2, 128), (8, 2, 64), (3, 3, 96)])
def test_a_padded_list_of_tiles(nq, nkv, d):
    """Tiles of no sequence behind those of the rows: skipped, and no workspace is taken for their parts (4 GB of them with 16 queries)."""
    gen = torch.Generator().manual_seed(nq)
    bs, rows, ctx = 16, [3], [8192]
    nb, bt = _tables(gen, ctx, bs)
    kc, vc = (c.cuda() for c in _random_cache(gen, nb, nkv, bs, d))
    q = _queries(gen, 3, nq, nkv, d).cuda()
    want, size = _oracle(q, kc, vc, bt, rows, ctx, nq, nkv, 0.1, 0, 0)
    ints = lambda *x: torch.tensor(x, device="cuda", dtype=torch.int32)  # noqa: E731
    tiles = torch.cat((_tiles(rows), torch.tensor([[-1, 0]], dtype=torch.int32).expand(255, -1))).cuda()
    out, bt, cu, ctx = torch.empty(3, nq * d, device="cuda", dtype=torch.bfloat16), bt.cuda(), ints(0, 3), ints(8192)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    get_ops("cuda").prefill_attention(out, q, kc, vc, bt, cu, ctx, tiles, nq, nkv, 0.1)
    assert torch.cuda.max_memory_allocated() - held < 140 << 20
    _check(out, want, size)


@pytest.mark.gpu
def test_two_streams_at_once():
    """Steps of two sequences on streams of their own, at the same time, give what each gives alone."""
    ops, nq, nkv, d, bs = get_ops("cuda"), 16, 2, 128, 16
    streams, jobs = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(2):
        gen = torch.Generator().manual_seed(30 + i)
        rows, ctx = [40 + i], [2500 - 700 * i]
        nb, bt = _tables(gen, ctx, bs)
        kc, vc = (c.cuda() for c in _random_cache(gen, nb, nkv, bs, d))
        slots = (bt[0].long()[torch.arange(ctx[0] - rows[0], ctx[0]) // bs] * bs + torch.arange(ctx[0] - rows[0], ctx[0]) % bs).cuda()
        qkv = _values(gen, rows[0], (nq + 2 * nkv) * d).cuda()
        parts = -(-bt.shape[1] * bs // 512)
        jobs.append(dict(rows=rows, qkv=qkv, kc=kc, vc=vc, bt=bt.cuda(), slots=slots, pos=torch.arange(rows[0]).cuda(),
                         cs=ref.rope_cos_sin(d, 64, 10000.0).cuda(), cu=torch.tensor([0, rows[0]], dtype=torch.int32).cuda(),
                         ctx=torch.tensor(ctx, dtype=torch.int32).cuda(), tiles=_tiles(rows).cuda(),
                         to=torch.empty(1, nq, parts, d, device="cuda"), tm=torch.empty(1, nq, parts, 2, device="cuda")))

    def step(j):
        qkv, kc, vc = j["qkv"].clone(), j["kc"].clone(), j["vc"].clone()
        out, one = (torch.empty(n, nq * d, dtype=torch.bfloat16, device="cuda") for n in (j["rows"][0], 1))
        k, v = (torch.empty(j["rows"][0], nkv, d, dtype=torch.bfloat16, device="cuda") for _ in "kv")
        ops.rope_cache(qkv, j["pos"], j["slots"], j["cs"], kc, vc, nq, nkv, d, 0)
        ops.read_cache(k, v, kc, vc, j["slots"])
        ops.prefill_attention(out, qkv, kc, vc, j["bt"], j["cu"], j["ctx"], j["tiles"], nq, nkv, 0.09)
        ops.paged_decode(one, qkv[-1:], kc, vc, j["bt"], j["ctx"], j["to"], j["tm"], nq, nkv, 512, 0.09)
        return kc, vc, k, v, out, one

    want = [step(j) for j in jobs]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, j in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(step(j))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))


@pytest.mark.gpu
def test_split_rows_replay():
    """The workspace of a captured call is the graph's own: replays beside eager calls of other sizes give the eager result."""
    gen = torch.Generator().manual_seed(8)
    nq, nkv, d, bs, rows, ctx = 32, 8, 128, 16, [17, 2], [3000, 1500]
    nb, bt = _tables(gen, ctx, bs)
    kc, vc = (c.cuda() for c in _random_cache(gen, nb, nkv, bs, d))
    q = _queries(gen, 19, nq, nkv, d).cuda()
    args = (bt.cuda(), torch.tensor([0, 17, 19], dtype=torch.int32).cuda(), torch.tensor(ctx, dtype=torch.int32).cuda(), _tiles(rows).cuda())
    ops, outs = get_ops("cuda"), [torch.empty(19, nq * d, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
    step = lambda i: ops.prefill_attention(outs[i], q, kc, vc, *args, nq, nkv, 0.1)  # noqa: E731
    step(0)
    graphs = []
    for i in (1, 2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(i)
        graphs.append(g)
    for _ in range(3):
        q.copy_(torch.randn_like(q))
        for o in outs:
            o.fill_(7.0)
        step(0)
        for g in graphs:
            g.replay()
        torch.empty(1 << 22, device="cuda").fill_(9.0)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
def test_hidden_nans_stay_hidden_and_seen_ones_show(dev, d, window, sinks):
    """Groups of scale byte 255 (a NaN was written) in tokens behind a row, before its window and behind the context never reach it;
    where a row sees one, a key makes the whole row NaN, a value the 32 dims of its group."""
    gen = torch.Generator().manual_seed(d)
    nq, nkv, bs, n = 4, 2, 16, 150
    nb, bt = _tables(gen, [n, n], bs)
    kc, vc = _random_cache(gen, nb, nkv, bs, d)

    def spoil(cache, seq, tok, head, group, values):
        o = tok % bs
        place = o if values else 4 * (o % 4) + o // 4
        cache.view(nb, nkv, -1)[int(bt[seq, tok // bs]), head, bs * d // 2 + group * bs + place] = 255

    for seq, tok, head, group in ((0, 70, 0, 1), (0, 101, 1, 0), (1, 149, 0, 0), (0, 2, 0, d // 32 - 1)):
        spoil(vc, seq, tok, head, group, True)
    for seq, tok, head, group in ((0, 120, 1, 0), (1, 60, 0, d // 32 - 1)):
        spoil(kc, seq, tok, head, group, False)
    for tok in range(n, -(-n // bs) * bs):   # what is left of the last pages
        for seq in (0, 1):
            for g in range(d // 32):
                for h in range(nkv):
                    spoil(kc, seq, tok, h, g, False)
                    spoil(vc, seq, tok, h, g, True)
    rows = [n, 100]
    q = _queries(gen, sum(rows), nq, nkv, d)
    got = _prompt(get_ops(dev), dev, q, kc, vc, bt, rows, [n, n], nq, nkv, d, window, sinks)
    want, size = _oracle(q, kc, vc, bt, rows, [n, n], nq, nkv, 1 / math.sqrt(d), window, sinks)
    assert want.isnan().any() and not want.isnan().all()
    _check(got.view(-1, nq, d), want, size)
    lens = [n, n, 60, 71, 101, 121, 1]
    pick = [0, 1, 1, 0, 0, 0, 0]
    for part in (64, 256):
        got = _decode(get_ops(dev), dev, q[:7], kc, vc, bt[pick], lens, nq, nkv, d, bs, part, window, sinks)
        want, size = _oracle(q[:7], kc, vc, bt[pick], [1] * 7, lens, nq, nkv, 1 / math.sqrt(d), window, sinks)
        _check(got.view(-1, nq, d), want, size)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("nq,nkv,d", [(8, 2, 64), (3, 3, 96), (16, 2, 128)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_a_query_that_is_no_number(dev, nq, nkv, d, value):
    """A NaN or an infinity in any 32 dims of a query makes that row of that head NaN (a score of infinity has no softmax) and no other."""
    gen = torch.Generator().manual_seed(d)
    bs, n = 16, 200
    nb, bt = _tables(gen, [n], bs)
    kc, vc = _random_cache(gen, nb, nkv, bs, d)
    q = _queries(gen, n, nq, nkv, d)
    spoiled = [(3 + 40 * g, g % nq, 32 * g + 7 * g) for g in range(d // 32)]
    for row, head, dim in spoiled:
        q[row, head * d + dim] = value
    clean = q[:, : nq * d].float().nan_to_num(0.0, 0.0, 0.0).to(torch.bfloat16)
    want, size = _oracle(clean, kc, vc, bt, [n], [n], nq, nkv, 1 / math.sqrt(d), 0, 0)
    for row, head, _ in spoiled:
        want[row, head] = float("nan")
    _check(_prompt(get_ops(dev), dev, q, kc, vc, bt, [n], [n], nq, nkv, d, 0, 0), want, size)
    rows = [r for r, _, _ in spoiled]
    for part in (64, 256):
        got = _decode(get_ops(dev), dev, q[rows], kc, vc, bt.repeat(len(rows), 1), [r + 1 for r in rows], nq, nkv, d, bs, part, 0, 0)
        _check(got, want[rows], size[rows])


@pytest.mark.parametrize("dev", DEVICES)
def test_pages_outside_of_the_cache_are_not_seen(dev):
    """Block ids below 0 and behind the cache: their keys are hidden, a row without any other is zeros; a context longer than its
    table ends with the table."""
    gen = torch.Generator().manual_seed(5)
    nq, nkv, d, bs = 8, 2, 128, 16
    ctx = [200, 90, 40, 33]
    nb, bt = _tables(gen, ctx, bs)
    kc, vc = _random_cache(gen, nb, nkv, bs, d)
    bt[0, 3], bt[0, 12], bt[1, 0], bt[2, :] = -1, nb, 2 ** 31 - 1, -7
    q = _queries(gen, 204, nq, nkv, d)
    got = _decode(get_ops(dev), dev, q[:4], kc, vc, bt, ctx, nq, nkv, d, bs, 64, 0, 0)
    want, size = _oracle(q[:4], kc, vc, bt, [1] * 4, ctx, nq, nkv, 1 / math.sqrt(d), 0, 0)
    _check(got.view(4, nq, d), want, size)
    assert not got[2].any()
    rows = [130, 40, 1, 33]
    got = _prompt(get_ops(dev), dev, q, kc, vc, bt, rows, ctx, nq, nkv, d, 50, 4)
    want, size = _oracle(q, kc, vc, bt, rows, ctx, nq, nkv, 1 / math.sqrt(d), 50, 4)
    _check(got[:204].view(204, nq, d), want, size)
    long = torch.tensor([10 ** 6, 90, 40, 33], dtype=torch.int32)
    got = _decode(get_ops(dev), dev, q[:4], kc, vc, bt, long, nq, nkv, d, bs, 64, 0, 0)
    want, size = _oracle(q[:4], kc, vc, bt, [1] * 4, [bt.shape[1] * bs, 90, 40, 33], nq, nkv, 1 / math.sqrt(d), 0, 0)
    _check(got.view(4, nq, d), want, size)


@pytest.mark.parametrize("dev", DEVICES)
def test_sharp_softmax_and_far_keys(dev):
    """Queries so large that one key takes all, keys of very different scales: the running maximum moves far, early and late."""
    gen = torch.Generator().manual_seed(11)
    nq, nkv, d, bs, n = 8, 2, 128, 16, 700
    nb, bt = _tables(gen, [n, n], bs)
    kc, vc = _random_cache(gen, nb, nkv, bs, d, spread=5)
    q = _queries(gen, 400, nq, nkv, d) * 20
    got = _decode(get_ops(dev), dev, q[:2], kc, vc, bt, [n, n - 1], nq, nkv, d, bs, 128, 0, 0)
    want, size = _oracle(q[:2], kc, vc, bt, [1, 1], [n, n - 1], nq, nkv, 1 / math.sqrt(d), 0, 0)
    # scores of up to 2^11: 32-bit sums of them are off by 2^-12, and so is the exponent
    _check_sharp(got.view(2, nq, d), want, size)
    got = _prompt(get_ops(dev), dev, q, kc, vc, bt, [300, 100], [n, n], nq, nkv, d, 0, 0)
    want, size = _oracle(q, kc, vc, bt, [300, 100], [n, n], nq, nkv, 1 / math.sqrt(d), 0, 0)
    _check_sharp(got.view(400, nq, d), want, size)


def _check_sharp(got, want, size):
    """Scores reach some thousands here: a sum of 128 products in 32 bits is off by up to 2^-24 of the sum of their magnitudes a step,
    2^-24 * 128 * 2^13 = 2^-4 at worst, 2^-8 for errors of either sign; a probability is off by as much, 2^-7 with the two scores of a ratio."""
    off = (got.float().cpu().double() - want).abs()
    assert (off <= (2 ** -8 + 2 ** -7) * 2 * size + 2 ** -8 * want.abs() + 1e-30).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (1, 2 ** 31 - 1), (100, 150), (2 ** 30, 5)])
def test_the_widest_windows(dev, window, sinks):
    """A window or first tokens beyond every context: all keys up to a row's own are seen."""
    gen = torch.Generator().manual_seed(21)
    nq, nkv, d, bs, ctx = 8, 2, 128, 16, [1, 150, 97]
    nb, bt = _tables(gen, ctx, bs)
    kc, vc = _random_cache(gen, nb, nkv, bs, d)
    rows = [1, 150, 40]
    q = _queries(gen, sum(rows), nq, nkv, d)
    want, size = _oracle(q, kc, vc, bt, rows, ctx, nq, nkv, 1 / math.sqrt(d), 0, 0)
    _check(_prompt(get_ops(dev), dev, q, kc, vc, bt, rows, ctx, nq, nkv, d, window, sinks), want, size)
    want, size = _oracle(q[:3], kc, vc, bt, [1] * 3, ctx, nq, nkv, 1 / math.sqrt(d), 0, 0)
    for part in (64, 256):
        _check(_decode(get_ops(dev), dev, q[:3], kc, vc, bt, ctx, nq, nkv, d, bs, part, window, sinks), want, size)


@pytest.mark.parametrize("dev", DEVICES)
def test_a_length_beyond_the_table_ends_with_it(dev):
    """Decode: with a window too, the last keys are the table's last ones."""
    gen = torch.Generator().manual_seed(22)
    nq, nkv, d, bs, n = 8, 2, 128, 16, 160
    nb, bt = _tables(gen, [n, n], bs)
    kc, vc = _random_cache(gen, nb, nkv, bs, d)
    q = _queries(gen, 2, nq, nkv, d)
    want, size = _oracle(q, kc, vc, bt, [1, 1], [n, n], nq, nkv, 1 / math.sqrt(d), 50, 4)
    _check(_decode(get_ops(dev), dev, q, kc, vc, bt, [2 ** 31 - 1, n + 30], nq, nkv, d, bs, 64, 50, 4), want, size)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("nq,nkv,d,bs", [(16, 2, 128, 16), (8, 2, 96, 32), (4, 2, 64, 16), (3, 3, 128, 64)])
@pytest.mark.parametrize("window,sinks", [(100, 4), (100, 0), (1, 70), (100, 1000), (0, 0), (300, 2 ** 31 - 1)])
@pytest.mark.parametrize("held,rows,ctx", [(512, [3, 70, 260, 5], [700, 560, 640, 512]), (4096, [1, 2], [9000, 4100])])
def test_prompt_rows_beyond_their_table(dev, nq, nkv, d, bs, window, sinks, held, rows, ctx):
    """Prompt: positions go on behind the table's keys, so a window may lie wholly behind them; the first tokens are seen all the same."""
    gen = torch.Generator().manual_seed(sum(ctx) + nq)
    nb, bt = _tables(gen, [held] * len(ctx), bs)
    kc, vc = _random_cache(gen, nb, nkv, bs, d)
    q = _queries(gen, sum(rows), nq, nkv, d)
    more = torch.cat((bt, torch.full((len(ctx), -(-max(ctx) // bs)), -1, dtype=torch.int32)), 1)   # no pages there
    want, size = _oracle(q, kc, vc, more, rows, ctx, nq, nkv, 1 / math.sqrt(d), window, sinks)
    assert bool(want[:rows[0]].any()) == (sinks > 0 or window != 100 and window != 1)
    _check(_prompt(get_ops(dev), dev, q, kc, vc, bt, rows, ctx, nq, nkv, d, window, sinks), want, size)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("length", [0, -1, -2 ** 31 + 1, -2 ** 31])
def test_a_prompt_of_no_length_is_zeros(dev, length):
    """Rows before position 0 see nothing, however far before."""
    gen = torch.Generator().manual_seed(24)
    nq, nkv, d, bs = 8, 2, 128, 16
    nb, bt = _tables(gen, [64, 64], bs)
    kc, vc = _random_cache(gen, nb, nkv, bs, d)
    q = _queries(gen, 10, nq, nkv, d)
    for window, sinks in ((0, 0), (20, 4)):
        out = _prompt(get_ops(dev), dev, q, kc, vc, bt, [3, 7], [length, 64], nq, nkv, d, window, sinks)
        want, size = _oracle(q[3:], kc, vc, bt[1:], [7], [64], nq, nkv, 1 / math.sqrt(d), window, sinks)
        assert not out[:3].any()
        _check(out[3:], want, size)


@pytest.mark.gpu
@pytest.mark.parametrize("cu", [[1, -2 ** 31], [2, -2 ** 31 + 1], [0, 2 ** 31 - 1], [-2 ** 31, 5], [-1, 2], [5, 3], [0, 11], [2 ** 31 - 1, -2 ** 31]])
def test_row_offsets_out_of_range_compute_nothing(cu):
    """Offsets that go back, or leave the rows, differences beyond 32 bits among them: no row is written."""
    gen = torch.Generator().manual_seed(25)
    nq, nkv, d, bs = 8, 2, 128, 16
    nb, bt = _tables(gen, [64], bs)
    kc, vc = (c.cuda() for c in _random_cache(gen, nb, nkv, bs, d))
    q = _queries(gen, 10, nq, nkv, d).cuda()
    out = torch.full((10, nq * d), 3.0, device="cuda", dtype=torch.bfloat16)
    ints = lambda *x: torch.tensor(x, device="cuda", dtype=torch.int32)  # noqa: E731
    get_ops("cuda").prefill_attention(out, q, kc, vc, bt.cuda(), ints(*cu), ints(64), ints(0, 0).view(1, 2), nq, nkv, 0.1)
    assert (out == 3).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("d", [64, 96, 128])
def test_scores_at_the_ends_of_the_range(dev, d):
    """Scores around -2^110 (one product each, so exact): the least negative one takes all, wherever it stands; the others' weights are 0,
    so the output is that value within its own rounding, of which a 4-bit value has none."""
    gen = torch.Generator().manual_seed(23)
    nq, nkv, bs, n = 8, 2, 16, 300
    nb, bt = _tables(gen, [n, n], bs)
    kc, vc = _random_cache(gen, nb, nkv, bs, d)
    kc.view(nb, nkv, -1)[..., : bs * d // 2] = 0
    kc.view(nb, nkv, -1)[..., bs * d // 2:] = 127 + 50
    for b in range(nb):   # dim 0 of every key: -6, of token 211: -4
        for t in range(bs):
            kc.view(nb, nkv, -1)[b, :, t * d // 2] = 15
    kc.view(nb, nkv, -1)[int(bt[0, 211 // bs]), :, 211 % bs * d // 2] = 14
    kc.view(nb, nkv, -1)[int(bt[1, 211 // bs]), :, 211 % bs * d // 2] = 14
    q = torch.zeros(600, (nq + 2 * nkv) * d, dtype=torch.bfloat16)
    q[:, ::d] = 2.0 ** 60
    vals = _decode_bytes(vc, True)
    one = torch.stack([vals[int(bt[i, 211 // bs]), :, 211 % bs] for i in (0, 1)]).repeat_interleave(nq // nkv, 1)  # [2, nq, d]
    for part in (64, 512):
        got = _decode(get_ops(dev), dev, q[:2], kc, vc, bt, [n, n], nq, nkv, d, bs, part, 0, 0)
        assert torch.equal(got.view(2, nq, d).cpu().double(), one)
    got = _prompt(get_ops(dev), dev, q, kc, vc, bt, [n, n], [n, n], nq, nkv, d, 0, 0).view(2, n, nq, d)[:, 211:].cpu().double()
    assert torch.equal(got, one[:, None].expand_as(got))


@pytest.mark.parametrize("dev", DEVICES)
def test_slots_outside_of_the_cache_write_and_read_nothing(dev):
    """Slots below 0, behind the cache and at the ends of 64 bits, in runs of 16 too."""
    ops, nq, nkv, d, bs, nb = get_ops(dev), 4, 2, 128, 16, 4
    slots = torch.cat([torch.arange(-16, 0), torch.arange(nb * bs, nb * bs + 32), torch.arange(-2 ** 63, -2 ** 63 + 32),
                       2 ** 63 - 32 + torch.arange(32), torch.arange(2 ** 62, 2 ** 62 + 32)])
    t = len(slots)
    qkv = _values(torch.Generator().manual_seed(3), t, (nq + 2 * nkv) * d)
    kc, vc = _random_cache(torch.Generator().manual_seed(4), nb, nkv, bs, d)
    k, v = kc.to(dev, copy=True), vc.to(dev, copy=True)
    for n in (t, 100):
        ops.rope_cache(qkv[:n].to(dev), torch.arange(n, device=dev), slots[:n].to(dev), ref.rope_cos_sin(d, t, 10000.0).to(dev), k, v, nq, nkv, d, 0)
    assert torch.equal(k.cpu(), kc) and torch.equal(v.cpu(), vc)
    ko, vo = (torch.ones(t, nkv, d, dtype=torch.bfloat16, device=dev) for _ in "kv")
    ops.read_cache(ko, vo, k, v, slots.to(dev))
    assert not ko.any() and not vo.any()


@pytest.mark.gpu
def test_decode_writes_the_f16_copy():
    gen = torch.Generator().manual_seed(2)
    nq, nkv, d, bs, ctx = 16, 4, 128, 16, [700, 1, 0, 300]
    nb, bt = _tables(gen, ctx, bs)
    kc, vc = _random_cache(gen, nb, nkv, bs, d)
    q = _queries(gen, 4, nq, nkv, d)
    for part in (128, 1024):
        out16 = torch.full((4, nq * d), float("nan"), device="cuda", dtype=torch.float16)
        out = _decode(get_ops("cuda"), "cuda", q, kc, vc, bt, ctx, nq, nkv, d, bs, part, 0, 0, out16=out16)
        h = out.float().to(torch.float16).view(4, -1, 8)[:, :, [0, 2, 1, 3, 4, 6, 5, 7]].reshape(4, -1)
        assert torch.equal(out16, h)


@pytest.mark.gpu
@pytest.mark.slow
def test_offsets_past_32_bits():
    """A cache of over 2^32 bytes a tensor: blocks at its end are written, read and attended to like the first ones."""
    nq, nkv, d, bs = 8, 8, 128, 16
    nb = (1 << 32) // (nkv * kv4.row_bytes(d) * bs) + 600
    kc, vc = (torch.empty(kv4.cache_shape(nb, nkv, bs, d), device="cuda", dtype=torch.uint8) for _ in "kv")
    assert kc.numel() > 1 << 32
    ops, n = get_ops("cuda"), 200
    gen = torch.Generator().manual_seed(1)
    qkv = _values(gen, n, (nq + 2 * nkv) * d).cuda()
    cs = ref.rope_cos_sin(d, 512, 10000.0).cuda()
    got = []
    for first in (0, nb - 13):
        bt = torch.arange(first, first + 13, device="cuda", dtype=torch.int32)[None]
        rows, pos = qkv.clone(), torch.arange(n, device="cuda")
        slots = first * bs + pos
        ops.rope_cache(rows, pos, slots, cs, kc, vc, nq, nkv, d, 0)
        k, v = (torch.empty(n, nkv, d, device="cuda", dtype=torch.bfloat16) for _ in "kv")
        ops.read_cache(k, v, kc, vc, slots)
        out, one = torch.empty(n, nq * d, device="cuda", dtype=torch.bfloat16), torch.empty(1, nq * d, device="cuda", dtype=torch.bfloat16)
        ints = lambda *x: torch.tensor(x, device="cuda", dtype=torch.int32)  # noqa: E731
        ops.prefill_attention(out, rows, kc, vc, bt, ints(0, n), ints(n), _tiles([n]).cuda(), nq, nkv, 0.09, 0)
        ws = torch.empty(1, nq, 2, d, device="cuda"), torch.empty(1, nq, 2, 2, device="cuda")
        ops.paged_decode(one, rows[-1:], kc, vc, bt, ints(n), *ws, nq, nkv, 128, 0.09, 0)
        got.append((k, v, out, one))
    assert all(torch.equal(a, b) for a, b in zip(*got)) and got[0][2].float().abs().sum() > 0


# ---------------------------------------------------------------- together, as a step uses them

@pytest.mark.parametrize("dev", DEVICES)
def test_a_sequence_from_prompt_to_decode(dev):
    """A prompt in two portions, then tokens one by one: writes, prompt and decode attention share one cache; every output is the
    oracle's over the bytes, and a token attends to the same values whichever operator reads them."""
    gen = torch.Generator().manual_seed(9)
    nq, nkv, d, bs, n, window, sinks = 8, 2, 128, 16, 150, 60, 4
    ops = get_ops(dev)
    nb, bt = _tables(gen, [n + 10], bs)
    kc, vc = (torch.zeros(kv4.cache_shape(nb, nkv, bs, d), dtype=torch.uint8, device=dev) for _ in "kv")
    cs = ref.rope_cos_sin(d, 512, 10000.0).to(dev)
    x = _values(gen, n + 10, (nq + 2 * nkv) * d)
    scale = 1 / math.sqrt(d)
    at = 0
    for rows in [100, 50] + [1] * 10:
        step = x[at:at + rows].clone().to(dev)
        pos = torch.arange(at, at + rows)
        slots = bt[0, pos // bs].long() * bs + pos % bs
        ops.rope_cache(step, pos.to(dev), slots.to(dev), cs, kc, vc, nq, nkv, d, 0)
        at += rows
        if rows > 1:
            got = _prompt(ops, dev, step, kc, vc, bt, [rows], [at], nq, nkv, d, window, sinks)
        else:
            got = _decode(ops, dev, step, kc, vc, bt, [at], nq, nkv, d, bs, 64, window, sinks)
            again = _prompt(ops, dev, step, kc, vc, bt, [1], [at], nq, nkv, d, window, sinks)
        want, size = _oracle(step, kc, vc, bt, [rows], [at], nq, nkv, scale, window, sinks)
        _check(got.view(rows, nq, d), want, size)
        if rows == 1:
            _check(again.view(1, nq, d), want, size)
    k, v = (torch.empty(n, nkv, d, dtype=torch.bfloat16, device=dev) for _ in "kv")
    pos = torch.arange(n)
    ops.read_cache(k, v, kc, vc, (bt[0, pos // bs].long() * bs + pos % bs).to(dev))
    assert torch.equal(v.cpu(), kv4.dequantise(*kv4.quantise(x[:n, (nq + nkv) * d:].view(n, nkv, d))))


@pytest.mark.gpu
def test_captured_steps_replay():
    """A decode step's write and attention and a prompt's, captured once, replayed for new rows, lengths and tables with eager work in
    between; two graphs that share the workspace, on a side stream."""
    gen = torch.Generator().manual_seed(4)
    nq, nkv, d, bs, b = 8, 2, 128, 16, 6
    ops, n = get_ops("cuda"), (8 + 4) * 128
    nb, width = 200, 16
    kc, vc = (c.cuda() for c in _random_cache(gen, nb, nkv, bs, d))
    cs = ref.rope_cos_sin(d, 512, 10000.0).cuda()
    qkv, pos = torch.zeros(b, n, device="cuda", dtype=torch.bfloat16), torch.zeros(b, device="cuda", dtype=torch.long)
    slots, ctx = torch.zeros(b, device="cuda", dtype=torch.long), torch.ones(b, device="cuda", dtype=torch.int32)
    bt = torch.zeros(b, width, device="cuda", dtype=torch.int32)
    to, tm = torch.empty(b, nq, 4, d, device="cuda"), torch.empty(b, nq, 4, 2, device="cuda")
    out, out_p = (torch.empty(b, nq * d, device="cuda", dtype=torch.bfloat16) for _ in "dp")
    cu, tiles = torch.tensor([0, b], device="cuda", dtype=torch.int32), _tiles([b]).cuda()

    def decode():
        ops.rope_cache(qkv, pos, slots, cs, kc, vc, nq, nkv, d, 0)
        ops.paged_decode(out, qkv, kc, vc, bt, ctx, to, tm, nq, nkv, 64, 0.09, 100, sinks=3)

    def prompt():
        ops.prefill_attention(out_p, qkv, kc, vc, bt[:1], cu, ctx[:1], tiles, nq, nkv, 0.09, 100, sinks=3)
        ops.paged_decode(out, qkv, kc, vc, bt, ctx, to, tm, nq, nkv, 64, 0.09, 0)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graphs = []
        for work in (decode, prompt):
            work()
            side.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                work()
            graphs.append(g)
        for round_ in range(4):
            lens = torch.randint(1, width * bs, (b,), generator=gen)
            lens[0] = max(int(lens[0]), b)
            table = torch.randperm(nb, generator=gen)[: b * width].view(b, width)
            fresh = torch.randn(b, n, generator=gen).to(torch.bfloat16)
            before = kc.clone(), vc.clone()
            for g, work in zip(graphs, (decode, prompt)):
                got = []
                for run in (g.replay, work):
                    kc.copy_(before[0])
                    vc.copy_(before[1])
                    qkv.copy_(fresh)
                    bt.copy_(table)
                    ctx.copy_(lens)
                    pos.copy_(lens - 1)
                    slots.copy_(table.gather(1, ((lens - 1) // bs)[:, None]).squeeze(1) * bs + (lens - 1) % bs)
                    to.fill_(float("nan"))
                    out.fill_(1.0)
                    run()
                    side.synchronize()
                    got.append([x.clone() for x in (out, out_p, kc, vc, qkv)])
                assert all(torch.equal(a, b_) for a, b_ in zip(*got))


# ---------------------------------------------------------------- refusals

@pytest.mark.parametrize("dev", DEVICES)
def test_refusals(dev):
    gen = torch.Generator().manual_seed(1)
    ops, nq, nkv, d, bs = get_ops(dev), 8, 2, 128, 16
    kc, vc = (c.to(dev) for c in _random_cache(gen, 8, nkv, bs, d))
    q = _queries(gen, 2, nq, nkv, d).to(dev)
    out = torch.zeros(2, nq * d, dtype=torch.bfloat16, device=dev)
    bt, ctx = torch.zeros(2, 4, dtype=torch.int32, device=dev), torch.ones(2, dtype=torch.int32, device=dev)
    to, tm = torch.zeros(2, nq, 1, d, device=dev), torch.zeros(2, nq, 1, 2, device=dev)
    cu, tiles = torch.tensor([0, 2], dtype=torch.int32, device=dev), _tiles([2]).to(dev)
    longs, cs = torch.zeros(2, dtype=torch.long, device=dev), ref.rope_cos_sin(d, 16, 10000.0).to(dev)
    bad = (ValueError, RuntimeError)
    for k, v in ((kc[..., :-1], vc), (kc, vc[:4]), (kc, vc.to(torch.int16)), (kc.transpose(0, 1), vc.transpose(0, 1))):
        with pytest.raises(bad):
            ops.paged_decode(out, q, k, v, bt, ctx, to, tm, nq, nkv, 64, 0.1)
        with pytest.raises(bad):
            ops.prefill_attention(out, q, k, v, bt[:1], cu, ctx[:1], tiles, nq, nkv, 0.1)
        with pytest.raises(bad):
            ops.rope_cache(q, longs, longs, cs, k, v, nq, nkv, d, 0)
        with pytest.raises(bad):
            ops.read_cache(*(torch.zeros(2, nkv, d, dtype=torch.bfloat16, device=dev) for _ in "kv"), k, v, longs)
    with pytest.raises(bad):   # other head counts than the cache's
        ops.paged_decode(out, q, kc, vc, bt, ctx, to, tm, nq, 4, 64, 0.1)
    for scale in (-0.1, float("nan")):
        with pytest.raises(bad):
            ops.paged_decode(out, q, kc, vc, bt, ctx, to, tm, nq, nkv, 64, scale)
        with pytest.raises(bad):
            ops.prefill_attention(out, q, kc, vc, bt[:1], cu, ctx[:1], tiles, nq, nkv, scale)
    with pytest.raises(bad):
        ops.read_cache(torch.zeros(3, nkv, d, dtype=torch.bfloat16, device=dev), torch.zeros(2, nkv, d, dtype=torch.bfloat16, device=dev), kc, vc,
                       longs)
    # first tokens beside a window: the other caches' operators have none
    kb = torch.zeros(8, nkv, bs, d, dtype=torch.bfloat16, device=dev)
    vb = torch.zeros(8, nkv, d, bs, dtype=torch.bfloat16, device=dev)
    with pytest.raises(ValueError):
        ops.paged_decode(out, q, kb, vb, bt, ctx, to, tm, nq, nkv, 512, 0.1, 16, sinks=4)
    with pytest.raises(ValueError):
        ops.prefill_attention(out, q, kb, vb, bt[:1], cu, ctx[:1], tiles, nq, nkv, 0.1, 16, sinks=4)


@pytest.mark.gpu
def test_kernel_refusals():
    """What only the kernels need: devices, alignment, workspaces, types."""
    gen = torch.Generator().manual_seed(1)
    ops, nq, nkv, d, bs = get_ops("cuda"), 8, 2, 128, 16
    kc, vc = (c.cuda() for c in _random_cache(gen, 8, nkv, bs, d))
    q = _queries(gen, 2, nq, nkv, d).cuda()
    n = q.shape[1]
    out = torch.zeros(2, nq * d, dtype=torch.bfloat16, device="cuda")
    bt, ctx = torch.zeros(2, 4, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    to, tm = torch.zeros(2, nq, 1, d, device="cuda"), torch.zeros(2, nq, 1, 2, device="cuda")
    longs, cs = torch.zeros(2, dtype=torch.long, device="cuda"), ref.rope_cos_sin(d, 16, 10000.0).cuda()
    odd = torch.zeros(2, n + 4, dtype=torch.bfloat16, device="cuda")

    def decode(**kw):
        a = dict(out=out, q=q, k=kc, v=vc, bt=bt, ctx=ctx, to=to, tm=tm, nq=nq, nkv=nkv, part=64, scale=0.1, window=0, sinks=0)
        a.update(kw)
        ops.paged_decode(a["out"], a["q"], a["k"], a["v"], a["bt"], a["ctx"], a["to"], a["tm"], a["nq"], a["nkv"], a["part"], a["scale"],
                         a["window"], sinks=a["sinks"])

    decode()
    for kw in (dict(q=q.float()), dict(q=q.cpu()), dict(q=odd[:, :n]), dict(q=odd[:, 4:]), dict(bt=bt.long()), dict(bt=bt.cpu()), dict(ctx=ctx.cpu()),
               dict(ctx=ctx[:1]), dict(part=96), dict(part=0), dict(part=32768), dict(to=to[:1]), dict(tm=tm.half()), dict(bt=torch.zeros(2, 5, dtype=torch.int32, device="cuda")),
               dict(window=-1), dict(sinks=-1, window=4), dict(nq=7), dict(out=out[:, :64]), dict(out=out[:1]), dict(v=vc.cpu()), dict(nq=64)):
        with pytest.raises(RuntimeError):
            decode(**kw)
    with pytest.raises(RuntimeError):
        ops.rope_cache(q, longs[:1], longs, cs, kc, vc, nq, nkv, d, 0)
    with pytest.raises(RuntimeError):
        ops.rope_cache(q, longs, longs.int(), cs, kc, vc, nq, nkv, d, 0)
    with pytest.raises(RuntimeError):
        ops.rope_cache(q, longs, longs, cs[:, :64], kc, vc, nq, nkv, d, 0)
    with pytest.raises(RuntimeError):
        ops.rope_cache(q, longs, longs, cs, kc, vc, nq, nkv, d, 2)
    with pytest.raises(RuntimeError):
        ops.rope_cache(q[:, :n - 8], longs, longs, cs, kc, vc, nq, nkv, d, 0)
    with pytest.raises(RuntimeError):
        ops.splitk_rope_cache(q, torch.zeros(1, 2, n - 1, device="cuda"), 1, longs, longs, cs, kc, vc, nq, nkv, d, 0)
    with pytest.raises(RuntimeError):
        ops.splitk_rope_cache(q, torch.zeros(1, 2, n, device="cuda"), 1, longs, longs, cs, kc, vc, nq, nkv, d, 1, q_w=cs[0], k_w=cs[0])
    # views that do not begin at a multiple of 16 bytes, tables of more than 2^30 tokens
    off = torch.zeros(kc.numel() + 8, dtype=torch.uint8, device="cuda")[8:].view(kc.shape)
    wide = torch.zeros(2, nq * d + 2, device="cuda").view(-1)[2:2 + to.numel()].view(to.shape)
    k256 = torch.zeros(kv4.cache_shape(1, nkv, 256, d), dtype=torch.uint8, device="cuda")
    long = torch.zeros(2, 2 ** 22 + 1, dtype=torch.int32, device="cuda")
    for kw in (dict(k=off), dict(v=off), dict(to=wide), dict(k=k256, v=k256, bt=long, window=64)):
        with pytest.raises(RuntimeError):
            decode(**kw)
    with pytest.raises(RuntimeError):
        ops.rope_cache(q, longs, longs, cs, off, vc, nq, nkv, d, 0)
    with pytest.raises(RuntimeError):
        ops.splitk_rope_cache(q, torch.zeros(2 * n + 2, device="cuda")[2:], 1, longs, longs, cs, kc, vc, nq, nkv, d, 0)
    cu = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError):
        ops.prefill_attention(out, q, k256, k256, long, cu, ctx[:1], _tiles([2]).cuda(), nq, nkv, 0.1)


@pytest.mark.gpu
def test_decode_refuses_more_keys_than_it_counts():
    """Rows that share one long table: 2^24 chunks of 64 tokens each, 2^31 of them together."""
    nq, nkv, d, rows = 1, 1, 64, 128
    kc = torch.zeros(kv4.cache_shape(1, nkv, 256, d), dtype=torch.uint8, device="cuda")
    bt = torch.zeros(1, 2 ** 22, dtype=torch.int32, device="cuda").expand(rows, -1)
    q = torch.zeros(rows, nq * d, dtype=torch.bfloat16, device="cuda")
    ctx, to, tm = torch.ones(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, nq, 1, d, device="cuda"), torch.zeros(rows, nq, 1, 2, device="cuda")
    with pytest.raises(RuntimeError, match="chunks of 64 tokens in all"):
        get_ops("cuda").paged_decode(q.clone(), q, kc, kc, bt, ctx, to, tm, nq, nkv, 16384, 0.1)


# ---------------------------------------------------------------- the engine

def _model(heads=2, kv_heads=1, dim=64, window=0, layers=2):
    cfg = PRESETS["tiny-llama"].replace(name="tiny-kv4", hidden_size=heads * dim, num_heads=heads, num_kv_heads=kv_heads, head_dim=dim, num_layers=layers)
    return cfg.replace(sliding_window=window, layer_windows=(window,) * layers) if window else cfg


def _engine(device, mcfg, dtype, **kw):
    base = dict(model=mcfg.name, load_format="dummy", device=device, dtype=dtype, max_num_seqs=8, max_num_batched_tokens=48, num_kv_blocks=256,
                max_model_len=512)
    dev = torch.device("cuda", 0) if device == "cuda" else None
    return LLMEngine(EngineConfig(**{**base, **kw}), tp=TPGroup(0, 1, None, dev) if dev else TPGroup(), model_cfg=mcfg)


def _dense_logits(model, ids, window, sinks):
    """The whole sequence at once, 32 bits, keys and values rounded to the 4-bit grid, no cache."""
    cfg = model.cfg
    x = model.embed[torch.tensor(ids)].float()
    t, d, nq, nkv = len(ids), cfg.head_dim, cfg.num_heads, cfg.num_kv_heads
    pos = torch.arange(t)
    j = pos[None, :]
    seen = j <= pos[:, None]
    if window:
        seen = seen & ((j > pos[:, None] - window) | (j < sinks))
    for lw in model.layers:
        h = ref.rmsnorm(x, lw.ln1, cfg.rms_norm_eps)
        q, k, v = (h @ lw.wqkv.float().T).view(t, -1, d).split((nq, nkv, nkv), 1)
        q, k = (ref.apply_rope(y, pos, model.cos_sin, cfg.rope_mode) for y in (q, k))
        k, v = (kv4.dequantise(*kv4.quantise(y.to(torch.bfloat16))).float().repeat_interleave(nq // nkv, 1) for y in (k, v))
        s = torch.einsum("qhd,khd->hqk", q, k) / math.sqrt(d)
        o = torch.einsum("hqk,khd->qhd", torch.softmax(s.masked_fill(~seen, float("-inf")), -1), v).reshape(t, nq * d)
        x = x + o @ lw.wo.float().T
        gu = ref.rmsnorm(x, lw.ln2, cfg.rms_norm_eps) @ lw.wgu.float().T
        g, u = gu.chunk(2, -1)
        x = x + (torch.nn.functional.silu(g) * u) @ lw.wd.float().T
    return ref.rmsnorm(x, model.norm, cfg.rms_norm_eps)[-1] @ model.lm_head.float().T


@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 0), (24, 4)])
def test_engine_matches_dense(window, sinks):
    """Chunked prompts and paged decode through the CPU engine against the whole sequence at once."""
    mcfg = _model(window=window)
    eng = _engine("cpu", mcfg, "float32", kv_cache_dtype="mxfp4", attention_sinks=sinks)
    m = eng.runner.model
    assert eng.runner.kv[0][0].dtype == torch.uint8
    assert m.kv_bytes_per_block(16) * 32 == 17 * 2 * mcfg.num_layers * mcfg.num_kv_heads * 16 * 64
    assert sum(c.numel() for kv in eng.runner.kv for c in kv) == m.kv_bytes_per_block(16) * 256
    prompts = [[1, 5, 9, 33, 70], list(range(3, 100)), list(range(200, 261))]
    for p, (toks, _, reason) in zip(prompts, eng.generate(prompts, SamplingParams(temperature=0.0, max_tokens=8, ignore_eos=True))):
        assert reason == "length"
        ids = list(p)
        for t in toks:
            lg = _dense_logits(m, ids, window, sinks)
            assert lg[t] >= lg.max() - 1e-4
            ids.append(t)


def test_engine_reuses_cached_prompts():
    """A prompt whose beginning is in the cache: the same tokens, with a window and first tokens that stay visible in it."""
    prompt, sp = list(range(3, 100)), SamplingParams(temperature=0.0, max_tokens=8, ignore_eos=True)
    want = None
    for caching in (False, True):
        eng = _engine("cpu", _model(window=24), "float32", kv_cache_dtype="mxfp4", attention_sinks=4, enable_prefix_caching=caching)
        got = [eng.generate([p], sp)[0][0] for p in (prompt, prompt, prompt[:70] + [1, 2, 3], prompt)]
        assert got[0] == got[1] == got[3]
        want = want or got
        assert got == want


def test_tensor_parallel_engine(tmp_path):
    """Each of two ranks keeps its kv heads' blocks: the tokens of one rank alone."""
    from hipserve.weights.safetensors_loader import random_hf_tensors, save_hf_checkpoint
    from tests import test_tp_cpu as tp

    cfg, ckpt = _model(heads=4, kv_heads=2), str(tmp_path / "kv4")
    save_hf_checkpoint(ckpt, cfg, random_hf_tensors(cfg, seed=7))
    eng = LLMEngine(tp._cfg(ckpt, 1, "mxfp4"), tp=TPGroup())
    assert eng.runner.kv[0][0].dtype == torch.uint8
    want = [r[0] for r in eng.generate(tp.PROMPTS, SamplingParams(temperature=0.0, max_tokens=8, ignore_eos=True))]
    assert tp._run_tp(ckpt, 2, "mxfp4") == want


def test_engine_refusals():
    with pytest.raises(ValueError):
        EngineConfig(kv_cache_dtype="mxfp4", attention_sinks=-1)
    with pytest.raises(ValueError):
        EngineConfig(attention_sinks=4)
    with pytest.raises(ValueError):
        EngineConfig(kv_cache_dtype="fp8", attention_sinks=4)
    with pytest.raises(ValueError):   # heads of 32
        _engine("cpu", PRESETS["tiny-llama"], "float32", kv_cache_dtype="mxfp4")
    with pytest.raises(ValueError):   # 17 queries per kv head
        _engine("cpu", _model(heads=17), "float32", kv_cache_dtype="mxfp4")
    with pytest.raises(ValueError):   # a design with caches of its own
        _engine("cpu", PRESETS["tiny-kesirax"], "float32", kv_cache_dtype="mxfp4")


def test_first_tokens_need_a_windowed_layer():
    """Without one the flag would change nothing; one windowed layer among others will do."""
    with pytest.raises(ValueError, match="no layer"):
        _engine("cpu", _model(), "float32", kv_cache_dtype="mxfp4", attention_sinks=4)
    with pytest.raises(ValueError, match="no layer"):
        _engine("cpu", _model().replace(layer_windows=(0, 0)), "float32", kv_cache_dtype="mxfp4", attention_sinks=4)
    mixed = _model(window=24).replace(layer_windows=(24, 0))
    assert _engine("cpu", mixed, "float32", kv_cache_dtype="mxfp4", attention_sinks=4).runner.model.attention_sinks == 4


def test_command_line():
    from hipserve.server import cli

    cfg = cli.config_from_args(cli.build_parser().parse_args(["--model", "llama-3-8b", "--kv-cache-dtype", "mxfp4", "--attention-sinks", "4"]))
    assert cfg.kv_mxfp4 and cfg.attention_sinks == 4


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(0, 0), (128, 4)])
def test_engine_graph_equals_eager(window, sinks):
    """Llama-3's heads, two layers: captured decode equals eager decode token for token, and the cache takes 17 / 64 of bf16's bytes."""
    mcfg = PRESETS["llama-3-8b"].replace(name="llama-3-kv4", num_layers=2, hidden_size=1024, intermediate_size=3584, num_heads=8,
                                         num_kv_heads=2, vocab_size=32000, max_position_embeddings=2048)
    if window:
        mcfg = mcfg.replace(sliding_window=window, layer_windows=(window, 0))
    prompts = [[1] + list(range(100, 400)), [1, 5, 6, 7], list(range(50, 90))]
    sp = SamplingParams(temperature=0.0, max_tokens=12, ignore_eos=True)
    toks = {}
    for kvd, eager in (("mxfp4", False), ("mxfp4", True), ("auto", False)):
        eng = _engine("cuda", mcfg, "bfloat16", kv_cache_dtype=kvd, attention_sinks=sinks if kvd == "mxfp4" else 0, enforce_eager=eager,
                      max_num_batched_tokens=256, max_model_len=1024)
        toks[kvd, eager] = [r[0] for r in eng.generate(prompts, sp)], eng.runner.model.kv_bytes_per_block(16)
        assert (eng.runner.stats["graph_steps"] > 0) != eager
        eng.shutdown()
        del eng
        torch.cuda.synchronize()
    assert toks["mxfp4", False] == toks["mxfp4", True]
    assert toks["mxfp4", False][1] * 64 == toks["auto", False][1] * 17
