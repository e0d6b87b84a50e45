"""The operators of serving from a paged key/value cache held in 8 bits: their cases, plain forms and exact values.

Three operators that a serving loop calls one after the other:

  tables   diopiBuildBlockTable: from the lengths of a batch, the blocks that its new tokens need, their slots, the
           offsets of the packed tokens, and (where asked) the right-aligned table of one slot for each token
  copy     diopiQuantizedCopyKV: new keys and values into cache blocks of 8-bit codes with one scale for each (block, head)
  attend   diopiQuantizedPagedAttention: attention of the newest tokens over those blocks

A code c in a block with scale s stands for c * s. Codes are int8 (c in -127..127, s = amax / 127) or e4m3 (s a power of
two, the smallest with amax / s <= 448). Lengths are spread evenly over [lo, hi] and dealt to the requests by the seed,
so that the work of a case does not depend on the seed.
"""
import math

import torch

own = False

FLT_MIN = 2.0 ** -126
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of a batch of 64: every request gets one more token
        dict(name="tables step", op="tables", batch=64, cached_lo=511, cached_hi=4095, new_lo=1, new_hi=1, block=16, wide=False),
        # 64 prompts of any length up to 8192 enter an empty cache
        dict(name="tables prompts", op="tables", batch=64, cached_lo=0, cached_hi=0, new_lo=1, new_hi=8192, block=64, wide=False),
        # a large batch that also feeds the ops which take one slot for each token
        dict(name="tables wide", op="tables", batch=1024, cached_lo=0, cached_hi=8188, new_lo=0, new_hi=4, block=16, wide=True),
        # one decode step: one token each into a block that is partly filled
        dict(name="copy step", op="copy", batch=64, cached_lo=511, cached_hi=4095, new_lo=1, new_hi=1, heads=8, dim=128, block=16, dtype="bf16", code="e4m3"),
        # the prompts of a prefill batch: 8 requests of 1024 to 8192 tokens, 32 heads
        dict(name="copy prompts", op="copy", batch=8, cached_lo=0, cached_hi=0, new_lo=1024, new_hi=8192, heads=32, dim=128, block=16, dtype="fp16", code="int8"),
        # pieces of prompts behind what is cached already, odd sizes, 32-bit inputs
        dict(name="copy pieces", op="copy", batch=19, cached_lo=0, cached_hi=1001, new_lo=0, new_hi=517, heads=5, dim=80, block=48, dtype="fp32", code="int8"),
        # a single short request: all latency
        dict(name="attend one", op="attend", batch=1, lo=37, hi=37, tokens=1, heads=32, kv_heads=8, dim=128, block=16, dtype="bf16", code="e4m3"),
        # the grouped decode batch: 64 query heads over 8 key/value heads
        dict(name="attend grouped", op="attend", batch=64, lo=512, hi=4096, tokens=1, heads=64, kv_heads=8, dim=128, block=16, dtype="bf16", code="e4m3"),
        # the decode batch with a key/value head for each query head
        dict(name="attend heads", op="attend", batch=64, lo=512, hi=4096, tokens=1, heads=32, kv_heads=32, dim=128, block=16, dtype="fp16", code="int8"),
        # few requests with long histories: the split over the tokens carries it
        dict(name="attend long", op="attend", batch=4, lo=30011, hi=131072, tokens=1, heads=32, kv_heads=4, dim=128, block=64, dtype="fp16", code="e4m3"),
        # four drafted tokens each are checked at once; some requests hold fewer tokens than that
        dict(name="attend drafts", op="attend", batch=32, lo=1, hi=2048, tokens=4, heads=32, kv_heads=8, dim=64, block=32, dtype="bf16", code="int8"),
        # odd head counts and width, empty requests, 32-bit activations
        dict(name="attend odd", op="attend", batch=23, lo=0, hi=1403, tokens=1, heads=14, kv_heads=2, dim=80, block=48, dtype="fp32", code="e4m3"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["tables", "copy", "attend", "attend"])
    block = rng.choice([16, 16, 32, 48, 64, 128])
    if op == "tables":
        batch = log(1, 1024)
        new_hi = rng.choice([1, 1, 4, log(1, 8192)])
        hi = min(8192, max(new_hi, 8 << 20) // batch)
        new_hi = min(new_hi, hi)
        cached_hi = rng.randint(0, hi - new_hi)
        return dict(op=op, batch=batch, cached_lo=rng.randint(0, cached_hi), cached_hi=cached_hi, new_lo=rng.randint(0, new_hi), new_hi=new_hi, block=block,
                    wide=rng.random() < 0.5)
    dtype, code, dim = rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.choice(["e4m3", "int8"]), rng.choice([64, 80, 96, 128, 128, 128, 256])
    if op == "copy":
        heads = rng.choice([1, 2, 4, 5, 8, 8, 16, 32])
        most = (30000 * 32 * 128) // (heads * dim * (2 if dtype == "fp32" else 1))   # tokens: no more data than the prompts of the list
        batch = log(1, 256)
        if rng.random() < 0.4:
            return dict(op=op, batch=batch, cached_lo=0, cached_hi=log(1, 4096), new_lo=1, new_hi=1, heads=heads, dim=dim, block=block, dtype=dtype, code=code)
        new_hi = max(1, min(log(2, 8192), most // batch))
        return dict(op=op, batch=batch, cached_lo=0, cached_hi=rng.choice([0, rng.randint(0, 1500)]), new_lo=rng.randint(0, new_hi), new_hi=new_hi, heads=heads,
                    dim=dim, block=block, dtype=dtype, code=code)
    kv = rng.choice([1, 2, 3, 4, 8, 8, 16, 32])
    group = rng.choice([1, 2, 4, 7, 8, 16] if kv <= 8 else [1, 2, 4])
    batch = log(1, 256)
    most = (140000 * 32 * 128) // (kv * dim)
    hi = max(1, min(log(1, 100000), most // batch))
    return dict(op=op, batch=batch, lo=rng.randint(0, hi), hi=hi, tokens=rng.choice([1, 1, 1, 2, 4]), heads=kv * group, kv_heads=kv, dim=dim, block=block, dtype=dtype,
                code=code)


def spread(lo, hi, batch, gen):
    """batch lengths spread evenly over [lo, hi], in an order of the generator's."""
    n = [lo + ((hi - lo) * i) // max(1, batch - 1) if batch > 1 else hi for i in range(batch)]
    return torch.tensor(n, dtype=torch.int64)[torch.randperm(batch, generator=gen)]


def lengths_of(lo, hi, batch):
    return [lo + ((hi - lo) * i) // max(1, batch - 1) if batch > 1 else hi for i in range(batch)]


def work(case):
    B, bs = case["batch"], case["block"]
    if case["op"] == "tables":
        cached, new = lengths_of(case["cached_lo"], case["cached_hi"], B), lengths_of(case["new_lo"], case["new_hi"], B)
        blocks = sum(new) / bs                      # entries written, each read from the free list
        return {"bytes": 4.0 * (2 * B + sum(new) + 2 * B + 1 + 2 * blocks + (sum(cached) + sum(new) if case["wide"] else 0)), "flops": 0.0}
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "copy":
        new = sum(lengths_of(case["new_lo"], case["new_hi"], B))
        row = case["heads"] * case["dim"]
        return {"bytes": 2.0 * new * row * (e + 1) + 2 * 4.0 * case["heads"] * (new / bs + B) + 12.0 * B, "flops": 4.0 * new * row}
    total = sum(lengths_of(case["lo"], case["hi"], B))
    row = case["kv_heads"] * case["dim"]
    q = B * case["tokens"] * case["heads"] * case["dim"]
    return {"bytes": 2.0 * total * row + 2 * 4.0 * case["kv_heads"] * total / bs + 2.0 * q * e + 4.0 * total / bs + 4.0 * B,
            "flops": 4.0 * total * case["tokens"] * case["heads"] * case["dim"]}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def normal(shape, std, dtype, gen):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * std).to(dtype)


def tables_for(lens, block, width, blocks, gen):
    """A table of `width` blocks for each request: blocks of a shuffled pool for what it holds, -1 behind them."""
    perm = torch.randperm(blocks, generator=gen)
    held = (lens + block - 1) // block
    at = torch.arange(width)[None, :] + (torch.cumsum(held, 0) - held)[:, None]
    keep = torch.arange(width)[None, :] < held[:, None]
    table = torch.where(keep, perm[at.clamp(max=blocks - 1)], torch.tensor(-1))
    return table.to(torch.int32), perm[int(held.sum()):].to(torch.int32)


def prepare(case, seed):
    cpu = torch.Generator().manual_seed(int(seed))
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    B, bs = case["batch"], case["block"]
    s = dict(case)
    if case["op"] in ("tables", "copy"):
        cached = spread(case["cached_lo"], case["cached_hi"], B, cpu)
        new = spread(case["new_lo"], case["new_hi"], B, cpu)
        after = cached + new
        width = max(1, int((case["cached_hi"] + case["new_hi"] + bs - 1) // bs))
        pool = int(after.sum()) // bs + B + 8
    if case["op"] == "tables":
        table, free = tables_for(cached, bs, width, pool + 5, cpu)
        T = int(new.sum())
        i32 = dict(dtype=torch.int32, device="cuda")
        s.update(cached=cached.to(**i32), new=new.to(**i32), table=table.cuda(), free=free.cuda(), start=torch.tensor([3], **i32),
                 slot_map=torch.empty(T, **i32), new_start=torch.empty(B + 1, **i32), seq_lens=torch.empty(B, **i32), next=torch.empty(1, **i32),
                 tokens_wide=torch.zeros(B, case["cached_hi"] + case["new_hi"], **i32) if case["wide"] else None)
        return s
    dt, H, D = DTYPES[case["dtype"]], case["heads"], case["dim"]
    if case["op"] == "copy":
        table, _ = tables_for(after, bs, width, pool, cpu)
        T = int(new.sum())
        starts = torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)])
        k, v = normal((T, H, D), 0.5, dt, gen), normal((T, H, D), 0.5, dt, gen)
        # what earlier tokens left: codes of values a little smaller than the new ones, so that some scales have to grow
        codes, scales = [], []
        for _ in range(2):
            c, sc = encoded((pool + 1, bs, H, D), 0.45, case["code"], gen)   # the last block belongs to nobody
            codes.append(c)
            scales.append(sc)
        s.update(k=k, v=v, table=table.cuda(), cached=cached.to(torch.int32).cuda(), starts=starts.to(torch.int32).cuda(), k_cache=codes[0], v_cache=codes[1],
                 k_scale=scales[0], v_scale=scales[1])
        return s
    lens = spread(case["lo"], case["hi"], B, cpu)
    pool = int(((lens + bs - 1) // bs).sum()) + 8
    table, _ = tables_for(lens, bs, max(1, (case["hi"] + bs - 1) // bs), pool, cpu)
    kc, ks = encoded((pool, bs, case["kv_heads"], D), 0.5, case["code"], gen)
    vc, vs = encoded((pool, bs, case["kv_heads"], D), 0.5, case["code"], gen)
    q = normal((B, case["tokens"], H, D), 1.0, dt, gen)
    s.update(q=q, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, table=table.cuda(), lens=lens.to(torch.int32).cuda(), scale=1.0 / math.sqrt(D))
    return s


def encoded(shape, std, code, gen):
    """Codes and scales of normal values, as earlier calls have left them in the cache."""
    blocks, bs, H, D = shape
    out = torch.empty(shape, dtype=torch.int8 if code == "int8" else torch.float8_e4m3fn, device="cuda")
    scale = torch.empty(blocks, H, dtype=torch.float32, device="cuda")
    step = max(1, (1 << 27) // (bs * H * D))
    for b in range(0, blocks, step):
        n = min(step, blocks - b)
        x = torch.randn((n, bs, H, D), generator=gen, device="cuda") * std
        sc = scale_for(x.abs().amax((1, 3)), code)
        x = x / sc[:, None, :, None]
        out[b:b + n] = x.round().to(torch.int8) if code == "int8" else x.to(torch.float8_e4m3fn)
        scale[b:b + n] = sc
    return out, scale


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------------
def scale_for(amax, code):
    """The scale of a block that begins anew, from the largest magnitude in it (fp32)."""
    if code == "int8":
        s = (amax / 127.0).clamp(min=FLT_MIN)
    else:
        m, e = torch.frexp(amax)                                   # amax = m * 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
        e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-126)
        s = torch.ldexp(torch.ones_like(amax), e)
    return torch.where(amax > 0, s, torch.zeros_like(s))


def grown(old, amax, code):
    """The scale of a block that holds tokens already: old * 2^k with the smallest k >= 0 that covers amax."""
    s = scale_for(amax, code)
    ratio = torch.where((s > old) & (old > 0), s.double() / old.double().clamp(min=1e-300), torch.ones_like(old, dtype=torch.float64))
    m, e = torch.frexp(ratio)                                      # ratio = m * 2^e, 0.5 <= m < 1
    up = torch.where(m == 0.5, e - 1, e)
    return torch.where(old > 0, (old.double() * torch.exp2(up.double())).float(), s)


def plain_tables(s):
    bs, table = s["block"], s["table"]
    c, n = s["cached"].long(), s["new"].long()
    have = (c + bs - 1) // bs
    need = (c + n + bs - 1) // bs - have
    first = torch.cumsum(need, 0) - need + s["start"].long()
    j = torch.arange(table.shape[1], device=table.device)[None, :]
    taken = (j >= have[:, None]) & (j < (have + need)[:, None])
    at = (first[:, None] + j - have[:, None]).clamp(0, s["free"].shape[0] - 1)
    table.copy_(torch.where(taken, s["free"][at], table))
    starts = torch.cat([torch.zeros(1, dtype=torch.int64, device=c.device), torch.cumsum(n, 0)])
    who = torch.repeat_interleave(torch.arange(c.shape[0], device=c.device), n, output_size=s["slot_map"].shape[0])
    pos = torch.arange(who.shape[0], device=c.device) - starts[who] + c[who]
    s["slot_map"].copy_(table[who, pos // bs].long() * bs + pos % bs)
    s["new_start"].copy_(starts)
    s["seq_lens"].copy_(c + n)
    s["next"].copy_(s["start"] + need.sum())
    if s["tokens_wide"] is not None:
        wide = s["tokens_wide"]
        p = torch.arange(wide.shape[1], device=c.device)[None, :] - (wide.shape[1] - (c + n))[:, None]
        slots = torch.gather(table, 1, (p.clamp(min=0) // bs)) * bs + (p % bs).int()
        wide.copy_(torch.where(p >= 0, slots, wide))
    return [table, s["slot_map"], s["new_start"], s["seq_lens"], s["next"], s["tokens_wide"]]


def plain_copy_one(s, x, cache, scale, pos, blk):
    """The new rows of one of the two caches; the cache and its scales are written."""
    bs, code = s["block"], s["code"]
    c, nobody = s["cached"].long(), cache.shape[0] - 1
    n = s["starts"].long().diff()
    row_max = x.float().abs().amax(2)                                                       # [T, H]
    amax = torch.zeros_like(scale).scatter_reduce(0, blk[:, None].expand_as(row_max), row_max, "amax")
    # a block whose first position is written begins anew; the one that a request had begun before keeps its tokens
    partial = (n > 0) & (c % bs > 0)
    tail = torch.gather(s["table"].long(), 1, (c // bs).clamp(max=s["table"].shape[1] - 1)[:, None])[:, 0]
    tail = torch.where(partial, tail, torch.full_like(tail, nobody))
    old = scale[tail]                                                                       # [B, H]
    new_tail = torch.where(partial[:, None], grown(old, amax[tail], code), old)
    touched = torch.zeros(scale.shape[0], dtype=torch.bool, device=x.device)
    touched[blk] = True
    scale.copy_(torch.where(touched[:, None], scale_for(amax, code), scale))
    scale[tail] = new_tail
    # the codes that were there, in the grown scale
    shrink = torch.where(new_tail > 0, old.double() / new_tail.double().clamp(min=1e-300), torch.ones_like(old, dtype=torch.float64))
    shrink = torch.where(old > 0, shrink, torch.ones_like(shrink))
    held = cache[tail]                                                                      # [B, bs, H, D]
    kept = held.float() * shrink.float()[:, None, :, None]
    kept = kept.round().to(cache.dtype) if code == "int8" else kept.to(cache.dtype)
    before = (torch.arange(bs, device=x.device)[None, :] < (c % bs)[:, None]) & partial[:, None]
    raw, raw_kept = cache.view(torch.int8), kept.view(torch.int8)
    raw[tail] = torch.where(before[:, :, None, None], raw_kept, held.view(torch.int8))
    # the new rows: the quotient to the nearest code, ties to the even one
    sx = scale[blk].double()[:, :, None]
    y = torch.where(sx > 0, x.double() / sx.clamp(min=1e-300), torch.zeros((), dtype=torch.float64, device=x.device))
    y = y.round().clamp(-127, 127).to(torch.int8) if code == "int8" else y.clamp(-448, 448).float().to(cache.dtype)
    raw[blk, pos % bs] = y.view(torch.int8)


def plain_copy(s):
    starts, c = s["starts"].long(), s["cached"].long()
    T = s["k"].shape[0]
    who = torch.repeat_interleave(torch.arange(c.shape[0], device=c.device), starts.diff(), output_size=T)
    pos = torch.arange(T, device=c.device) - starts[who] + c[who]
    blk = s["table"][who, pos // s["block"]].long()
    plain_copy_one(s, s["k"], s["k_cache"], s["k_scale"], pos, blk)
    plain_copy_one(s, s["v"], s["v_cache"], s["v_scale"], pos, blk)
    return [s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]]


def plain_attend(s):
    q, table, lens = s["q"], s["table"].long(), s["lens"].long()
    B, n, H, D = q.shape
    bs, Hkv, width = s["block"], s["kv_heads"], table.shape[1]
    at = table.clamp(min=0)
    k = s["k_cache"][at].float() * s["k_scale"][at][:, :, None, :, None]
    k = k.reshape(B, width * bs, Hkv, D).permute(0, 2, 3, 1)
    x = torch.matmul(q.float().reshape(B, n, Hkv, H // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, n * (H // Hkv), D), k) * s["scale"]
    del k
    limit = lens[:, None] - (n - 1) + torch.arange(n, device=q.device)[None, :]                       # tokens that new token t sees
    seen = torch.arange(width * bs, device=q.device)[None, None, :] < limit[:, :, None]              # [B, n, tokens]
    seen = seen[:, None, :, None, :].expand(B, 1, n, H // Hkv, width * bs).reshape(B, 1, n * (H // Hkv), width * bs)
    x = torch.where(seen, x, torch.full((), -math.inf, device=q.device))
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    x = x / x.sum(-1, keepdim=True).clamp(min=1e-37)
    v = s["v_cache"][at].float() * s["v_scale"][at][:, :, None, :, None]
    v = v.reshape(B, width * bs, Hkv, D).permute(0, 2, 1, 3)
    o = torch.matmul(x, v)
    return o.reshape(B, Hkv, n, H // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B, n, H, D).to(q.dtype)


def run(s):
    if own:
        from diopi_b200 import functions as F
        from diopi_b200.runtime import default_context
        ctx = default_context()
        ctx.release()
        if s["op"] == "tables":
            F.build_block_table(s["table"], s["cached"], s["new"], s["free"], s["start"], s["block"], slot_map=s["slot_map"], new_start=s["new_start"],
                                seq_lens=s["seq_lens"], free_next=s["next"], token_table=s["tokens_wide"], ctx=ctx)
            return [s["table"], s["slot_map"], s["new_start"], s["seq_lens"], s["next"], s["tokens_wide"]]
        if s["op"] == "copy":
            F.quantized_copy_kv(s["k"], s["v"], s["table"], s["cached"], s["starts"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], ctx=ctx)
            return [s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]]
        return F.quantized_paged_attention(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"], s["lens"], s["scale"], ctx=ctx)
    if s["op"] == "tables":
        return plain_tables(s)
    return plain_copy(s) if s["op"] == "copy" else plain_attend(s)


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits, request by request
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        return exact_attend(s)
    if case["op"] == "copy":
        return exact_copy(s)
    return None  # whole numbers: they are equal or wrong


def exact_attend(s):
    q = s["q"]
    B, n, H, D = q.shape
    bs, Hkv = s["block"], s["kv_heads"]
    out = torch.zeros(B, n, H, D, dtype=torch.float64, device=q.device)
    for i, L in enumerate(s["lens"].tolist()):
        used = s["table"][i, :(L + bs - 1) // bs].long()
        for h in range(Hkv):
            keys = (s["k_cache"][used, :, h].double() * s["k_scale"][used, h].double()[:, None, None]).reshape(-1, D)[:L]
            vals = (s["v_cache"][used, :, h].double() * s["v_scale"][used, h].double()[:, None, None]).reshape(-1, D)[:L]
            group = slice(h * (H // Hkv), (h + 1) * (H // Hkv))
            for t in range(n):
                m = L - (n - 1 - t)
                if m > 0:
                    out[i, t, group] = torch.softmax(q[i, t, group].double() @ keys[:m].T * s["scale"], -1) @ vals[:m]
    return out


def exact_copy(s):
    bs, code, most = s["block"], s["code"], 127 if s["code"] == "int8" else 448
    out = []
    cached, starts, table = s["cached"].tolist(), s["starts"].tolist(), s["table"].tolist()
    for x, cache, scale in ((s["k"], s["k_cache"], s["k_scale"]), (s["v"], s["v_cache"], s["v_scale"])):
        values, sc = cache.double(), scale.double()
        if sum((b - a) // bs + 2 for a, b in zip(starts, starts[1:])) > 8000:
            return None
        for i, c in enumerate(cached):
            t, end = starts[i], starts[i + 1]
            while t < end:
                pos = c + t - starts[i]
                b, p = table[i][pos // bs], pos % bs
                m = min(bs - p, end - t)
                rows = x[t:t + m].double()
                top = rows.abs().amax((0, 2))
                if code == "int8":
                    need = (top / 127).float().double()
                else:
                    need = torch.exp2(torch.ceil(torch.log2((top / 448).clamp(min=FLT_MIN)) - 1e-9))
                need = torch.where(top > 0, need.clamp(min=FLT_MIN), torch.zeros_like(need))
                if p > 0:
                    had = sc[b]
                    steps = torch.ceil(torch.log2((need / had.clamp(min=1e-300)).clamp(min=1)) - 1e-12)
                    need = torch.where(had > 0, had * torch.exp2(steps), need)
                    ratio = torch.where((had > 0) & (need > 0), had / need.clamp(min=1e-300), torch.ones_like(need))
                    values[b, :p] = nearest(values[b, :p] * ratio[None, :, None], code)
                sc[b] = need
                values[b, p:p + m] = nearest((rows / need.clamp(min=1e-300)[None, :, None]).clamp(-most, most), code)
                t += m
        out += [values, sc]
    return [None if code == "int8" else out[0], None if code == "int8" else out[2], out[1], out[3]]


def nearest(y, code):
    """The nearest value that a code can hold, ties to even."""
    if code == "int8":
        return y.round()
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return (y / step).round() * step
