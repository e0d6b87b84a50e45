"""Block tables, the store into a paged cache of 8-bit codes, and attention over it: the definitions in 64 bits, token by token.

CPU tensors in, CPU tensors out; nothing here is shared with the kernels. Codes are int8 or the bits of e4m3 values (uint8);
a code c of a block with scale s stands for c * s.
"""
from __future__ import annotations

import math

import torch

NO_SLOT = -(1 << 31)


def e4m3_values() -> torch.Tensor:
    """The 256 values of the e4m3 codes (4 exponent bits, bias 7, 3 mantissa bits, no infinities, NaN at 0x7f and 0xff)."""
    out = []
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = math.ldexp(m, -9) if e == 0 else math.ldexp(8 + m, e - 10)
        out.append(float("nan") if c & 127 == 127 else (-v if c & 128 else v))
    return torch.tensor(out, dtype=torch.float64)


_E4M3 = e4m3_values()
_E4M3_UP = _E4M3[:127]


def decode(codes: torch.Tensor) -> torch.Tensor:
    return codes.double() if codes.dtype == torch.int8 else _E4M3[codes.long()]


def encode(y: torch.Tensor, e4m3: bool) -> torch.Tensor:
    """The nearest code to each value, ties to the even one; out-of-range values saturate; NaN becomes 0 or NaN."""
    if not e4m3:
        r = torch.nan_to_num(y, nan=0.0, posinf=127.0, neginf=-127.0).round().clamp(-127, 127)
        return r.to(torch.int8)
    a = torch.nan_to_num(y, nan=0.0, posinf=448.0, neginf=-448.0).abs().clamp(max=448.0).contiguous()
    hi = torch.searchsorted(_E4M3_UP, a).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = _E4M3_UP[hi] - a, a - _E4M3_UP[lo]
    c = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    c = c + torch.where(torch.signbit(y), 128, 0)
    return torch.where(torch.isnan(y), torch.full_like(c, 127), c).to(torch.uint8)


def fresh_scale(amax: float, e4m3: bool) -> float:
    if not amax > 0:
        return 0.0
    if not e4m3:
        return max(float(torch.tensor(amax, dtype=torch.float32) * torch.tensor(1 / 127, dtype=torch.float32)), 2.0 ** -126)
    k = -126
    while amax > 448.0 * 2.0 ** k:
        k += 1
    return 2.0 ** k


def build_block_table(block_table, cached, new, free_blocks, free_start, block_size, T, wide=None):
    """Returns (block_table, slot_map, new_start, seq_lens, free_next, wide); lists of ints and int64 tensors."""
    table = block_table.clone().long()
    cap = table.shape[1] * block_size
    at, slots, starts, lens = max(int(free_start), 0), [], [0], []
    n_free = len(free_blocks)
    wide = None if wide is None else wide.clone().long()
    for i, (c, n) in enumerate(zip(cached.tolist(), new.tolist())):
        c, n = min(max(c, 0), cap), max(n, 0)
        fits = min(n, cap - c)
        for j in range(-(-c // block_size), -(-(c + fits) // block_size)):
            table[i, j] = int(free_blocks[at]) if at < n_free else -1
            at += 1

        def slot(p):
            b = int(table[i, p // block_size])
            return NO_SLOT if b < 0 else b * block_size + p % block_size
        slots += [slot(c + t) if t < fits else NO_SLOT for t in range(n)]
        starts.append(starts[-1] + n)
        lens.append(c + fits)
        if wide is not None:
            for p in range(max(0, lens[-1] - wide.shape[1]), lens[-1]):
                wide[i, wide.shape[1] - lens[-1] + p] = slot(p)
    slots = slots[:T] + [NO_SLOT] * (T - len(slots))
    return table, torch.tensor(slots, dtype=torch.int64), torch.tensor(starts), torch.tensor(lens, dtype=torch.int64), min(at, max(n_free, int(free_start))), wide


def quantized_copy(x, block_table, cached, new_start, cache, scale):
    """One of the two matrices: x [T, H, D] into clones of cache [blocks, bs, H, D] and scale [blocks, H]; returns both."""
    cache, scale = cache.clone(), scale.clone()
    e4m3, bs = cache.dtype == torch.uint8, cache.shape[1]
    for i, c in enumerate(cached.tolist()):
        t, end = int(new_start[i]), min(int(new_start[i + 1]), x.shape[0])
        pos = c
        while t < end and pos < block_table.shape[1] * bs:
            b, p = int(block_table[i, pos // bs]), pos % bs
            m = min(bs - p, end - t)
            rows = x[t:t + m].double()
            t, pos = t + m, pos + m
            if not 0 <= b < cache.shape[0]:
                continue
            for h in range(x.shape[1]):
                r = rows[:, h]
                finite = r[torch.isfinite(r)]
                s = fresh_scale(float(finite.abs().max()) if finite.numel() else 0.0, e4m3)
                old = float(scale[b, h])
                if p > 0 and old > 0:
                    need, s, k = s, old, 0
                    while s < need:
                        s, k = s * 2, k + 1
                    if k:
                        cache[b, :p, h] = encode(decode(cache[b, :p, h]) * 2.0 ** -k, e4m3)
                scale[b, h] = s
                y = r / s if s > 0 else torch.where(torch.isnan(r), r, torch.zeros_like(r))
                cache[b, p:p + m, h] = encode(y, e4m3)
    return cache, scale


def quantized_paged_attention(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, softmax_scale):
    """q [B, n, H, D]. Returns (out, (weight, reach, logit)) in fp64: the result, and what error bounds go by: the same sum with |v|
    in the place of v, the sum of |v| alone (both [B, n, H, D]), and the largest softmax_scale * sum |q| |k| ([B, n, H])."""
    B, n, H, D = q.shape
    bs, Hkv = k_cache.shape[1], k_cache.shape[2]
    out, weight, reach = [torch.zeros(B, n, H, D, dtype=torch.float64) for _ in range(3)]
    logit = torch.zeros(B, n, H, dtype=torch.float64)
    for i, L in enumerate(seq_lens.tolist()):
        L = min(max(L, 0), block_table.shape[1] * bs)
        pos = torch.arange(L)
        blk = block_table[i].long()[pos // bs]
        ok = (blk >= 0) & (blk < k_cache.shape[0])
        blk = torch.where(ok, blk, torch.zeros_like(blk))
        for h in range(Hkv):
            k = decode(k_cache[blk, pos % bs, h]) * k_scale[blk, h].double()[:, None]
            v = decode(v_cache[blk, pos % bs, h]) * v_scale[blk, h].double()[:, None]
            for g in range(h * (H // Hkv), (h + 1) * (H // Hkv)):
                for t in range(n):
                    see = ok & (pos < L - (n - 1 - t))
                    if not bool(see.any()):
                        continue
                    x = softmax_scale * (k[see] @ q[i, t, g].double())
                    p = torch.softmax(x, 0)
                    out[i, t, g] = p @ v[see]
                    weight[i, t, g] = p @ v[see].abs()
                    reach[i, t, g] = v[see].abs().sum(0)
                    logit[i, t, g] = (softmax_scale * (k[see].abs() @ q[i, t, g].double().abs())).max()
    return out, (weight, reach, logit)
