"""The 4-bit paged KV cache (``--kv-cache-dtype mxfp4``) in plain PyTorch: the CPU engine's operators and what the kernels' are tested
against.

OCP microscaling FP4: a value is an e2m1 number times 2^(byte - 127), the byte shared by 32 neighbouring dims of a token and head.
A cache tensor is uint8 [blocks, kv heads, block_size, 17 D / 32]; within a block and head the codes come first (two dims a byte,
the even one in the low half), then the scale bytes:

  keys    codes [block_size][D / 2]; scales [D / 32][block_size], token o of a run of 16 at 4 (o % 4) + o // 4
  values  codes [D / 2][block_size]; scales [D / 32][block_size]

The scale of a group is the power of two under which its largest magnitude is at most 7 (within a sixth of the largest level, 6),
kept within [2^-119, 2^125]; values round to the nearest level, ties to the even code, magnitudes above 6 to 6. A group that holds
a NaN or an infinity has scale byte 255 and reads as NaN.
"""
from __future__ import annotations

import torch

GROUP = 32
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BORDERS = ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False))  # and who keeps a tie
SCALE_MIN, SCALE_MAX, SCALE_NAN = 8, 252, 255
DTYPE = torch.uint8
HEAD_DIMS = (64, 96, 128)


def row_bytes(D: int) -> int:
    """Cached bytes of one token of one kv head, keys or values."""
    return D * 17 // 32


def cache_shape(blocks: int, nkv: int, block_size: int, D: int) -> tuple:
    if D not in HEAD_DIMS:
        raise ValueError(f"the mxfp4 cache holds heads of 64, 96 or 128, not {D}")
    return blocks, nkv, block_size, row_bytes(D)


def is_kv4(cache: torch.Tensor) -> bool:
    return cache.dtype == DTYPE


def head_dim(cache: torch.Tensor) -> int:
    return cache.shape[3] * 32 // 17


def check(k_cache, v_cache, nkv: int):
    ok = all(c.dtype == DTYPE and c.dim() == 4 and c.is_contiguous() and c.shape[3] % 17 == 0 and head_dim(c) in HEAD_DIMS
             for c in (k_cache, v_cache)) and k_cache.shape == v_cache.shape
    if not ok or k_cache.shape[1] != nkv:
        raise ValueError(f"mxfp4 caches are contiguous uint8 [blocks, {nkv}, block_size, 17 head_dim / 32], K and V alike: got "
                         f"{tuple(k_cache.shape)} {k_cache.dtype} and {tuple(v_cache.shape)} {v_cache.dtype}")


def _pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e, 64 bits, for whole e: from its bits, since a power computed in floating point need not be exact."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def quantise(x: torch.Tensor):
    """bf16 rows [..., D] -> (codes uint8 [..., D], scale bytes uint8 [..., D / 32])."""
    g = x.to(torch.bfloat16).unflatten(-1, (-1, GROUP))
    top = (g.view(torch.int16).int() & 0x7fff).amax(-1)    # magnitudes of bf16 order as their bits do
    byte = (((top + 31) >> 7) - 2).clamp(SCALE_MIN, SCALE_MAX)
    lost = top >= 0x7f80
    a = g.double().abs() * _pow2(127 - byte)[..., None]
    code = sum((a >= b if keeps else a > b).int() for b, keeps in BORDERS)
    code = torch.where(lost[..., None], 0, code + 8 * torch.signbit(g).int())
    return code.to(DTYPE).flatten(-2), torch.where(lost, SCALE_NAN, byte).to(DTYPE)


def dequantise(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The values, bf16 (exact), of codes [..., D] under scale bytes [..., D / 32]."""
    level = torch.tensor([s * v for s in (1.0, -1.0) for v in LEVELS], dtype=torch.float64, device=codes.device)
    y = level[codes.long()].unflatten(-1, (-1, GROUP)) * _pow2(scales.long() - 127)[..., None]
    return torch.where((scales == SCALE_NAN)[..., None], float("nan"), y).to(torch.bfloat16).flatten(-2)


def _places(cache, slots, values: bool):
    """Flat indices of slots' packed codes [T, heads, D / 2] and scale bytes [T, heads, D / 32]."""
    _, h, bs, w = cache.shape
    D, dev = head_dim(cache), cache.device
    base = (((slots // bs)[:, None] * h + torch.arange(h, device=dev)) * (bs * w))[..., None]
    off = (slots % bs)[:, None, None]
    pair, group = torch.arange(D // 2, device=dev), torch.arange(D // GROUP, device=dev)
    if values:
        return base + pair * bs + off, base + bs * D // 2 + group * bs + off
    return base + off * (D // 2) + pair, base + bs * D // 2 + group * bs + off // 16 * 16 + 4 * (off % 4) + off % 16 // 4


def _inside(cache, slots):
    return (slots >= 0) & (slots < cache.shape[0] * cache.shape[2])


def store(cache, slots, x, values: bool):
    """Quantises rows x [T, heads, D] into their slots; a slot outside of the cache writes nothing."""
    keep = _inside(cache, slots)
    codes, scales = quantise(x[keep])
    at, scale_at = _places(cache, slots[keep], values)
    flat = cache.view(-1)
    flat[at] = codes[..., 0::2] | (codes[..., 1::2] << 4)
    flat[scale_at] = scales


def load(cache, slots, values: bool) -> torch.Tensor:
    """The rows of slots as bf16 [T, heads, D]; zeros for a slot outside of the cache."""
    keep = _inside(cache, slots)
    at, scale_at = _places(cache, torch.where(keep, slots, 0), values)
    flat = cache.view(-1)
    packed = flat[at]
    codes = torch.stack((packed & 15, packed >> 4), -1).flatten(-2)
    return torch.where(keep[:, None, None], dequantise(codes, flat[scale_at]), 0)


def context(k_cache, v_cache, block_table, n: int):
    """(keys, values, page present) of the first n tokens of a sequence: a block id outside of the cache is no page."""
    bs = k_cache.shape[2]
    j = torch.arange(max(0, min(n, block_table.shape[0] * bs)), device=k_cache.device)
    page = block_table[j // bs].long()
    ok = (page >= 0) & (page < k_cache.shape[0])
    slots = torch.where(ok, page * bs + j % bs, -1)
    return load(k_cache, slots, False), load(v_cache, slots, True), ok


def attend(q, k, v, seen, scale: float) -> torch.Tensor:
    """q [rows, heads, D], k and v [n, kv heads, D], seen [rows, n] -> [rows, heads, D]: softmax over what is seen, zeros for a row that
    sees nothing. What a hidden key or value holds, NaN or not, never enters."""
    if not scale >= 0:
        raise ValueError(f"scale >= 0, got {scale}")
    rows, nq, D = q.shape
    g = nq // k.shape[1]
    q = q.float().unflatten(1, (-1, g)).transpose(0, 1)                   # [kv heads, rows, g, D]
    k, v = (x.float().transpose(0, 1) for x in (k, v))                    # [kv heads, n, D]
    s = torch.matmul(q.flatten(1, 2), k.transpose(1, 2)).unflatten(1, (rows, g)) * scale
    s = s.masked_fill(~seen[None, :, None], float("-inf"))
    some = seen.any(-1)
    p = torch.softmax(torch.where(some[None, :, None, None], s, 0.0), -1)
    p = torch.where(seen[None, :, None], p, 0.0)
    bad = ~torch.isfinite(v)
    out = torch.matmul(p.flatten(1, 2), torch.where(bad, 0.0, v))
    if bad.any():
        hit = torch.matmul(seen.float(), bad.float()) > 0                 # [kv heads, rows, D]: dims that a row sees a NaN of
        out = torch.where(hit.repeat_interleave(g, 1), float("nan"), out)
    return out.unflatten(1, (rows, g)).transpose(0, 1).flatten(1, 2)


def sees(pos, tokens, window: int, sinks: int):
    """[rows, tokens]: key j is seen from position pos if it is not after it and, with a window, is among its last ``window``
    keys or the first ``sinks``."""
    j = torch.arange(tokens, device=pos.device)
    seen = j <= pos[:, None]
    return seen & ((j > pos[:, None] - window) | (j < sinks)) if window > 0 else seen


def paged_decode(q, k_cache, v_cache, block_tables, context_lens, nq, nkv, scale, window=0, sinks=0):
    """q [B, nq * D (+ extra)] -> [B, nq, D]. A length beyond the block table's tokens counts as those."""
    check(k_cache, v_cache, nkv)
    D = head_dim(k_cache)
    out = torch.empty(q.shape[0], nq, D, dtype=q.dtype, device=q.device)
    for b in range(q.shape[0]):
        n = max(0, min(int(context_lens[b]), block_tables.shape[1] * k_cache.shape[2]))
        k, v, ok = context(k_cache, v_cache, block_tables[b], n)
        seen = sees(torch.tensor([n - 1], device=q.device), k.shape[0], window, sinks) & ok
        out[b] = attend(q[b:b + 1, : nq * D].view(1, nq, D), k, v, seen, scale)[0].to(q.dtype)
    return out


def prefill_attention(q, k_cache, v_cache, block_tables, cu_q, ctx_lens, nq, nkv, scale, window=0, sinks=0):
    """q [T, nq * D (+ extra)] -> [cu_q[-1], nq, D]."""
    check(k_cache, v_cache, nkv)
    D = head_dim(k_cache)
    out = torch.empty(int(cu_q[-1]), nq, D, dtype=q.dtype, device=q.device)
    for s in range(len(cu_q) - 1):
        r0, r1, ctx = int(cu_q[s]), int(cu_q[s + 1]), int(ctx_lens[s])
        k, v, ok = context(k_cache, v_cache, block_tables[s], ctx)
        seen = sees(torch.arange(ctx - (r1 - r0), ctx, device=q.device), k.shape[0], window, sinks) & ok
        out[r0:r1] = attend(q[r0:r1, : nq * D].view(r1 - r0, nq, D), k, v, seen, scale).to(q.dtype)
    return out


def read_cache(k_out, v_out, k_cache, v_cache, slots):
    check(k_cache, v_cache, k_cache.shape[1] if k_cache.dim() == 4 else 0)
    shape = (slots.numel(), k_cache.shape[1], head_dim(k_cache))
    if any(tuple(o.shape) != shape for o in (k_out, v_out)):
        raise ValueError(f"read_cache: outputs are bf16 {list(shape)}")
    k_out.copy_(load(k_cache, slots, False))
    v_out.copy_(load(v_cache, slots, True))
