"""The 8-bit cache operators at the ends of their ranges: logits far beyond fp16, values near the largest fp32, scales that
are no powers of two. Same oracle as the other tests of these operators."""
import math

import pytest
import torch

from oracle import quantized_cache as O
from test_gpu_quantized_cache import DT, LENS, F, attention_inputs, bound_of, check_attention, check_copy, ctx, paged, take_status  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_status(F):  # noqa: F811
    """No kernel of these tests meets anything that it has to report."""
    assert take_status(F) is None
    yield
    assert take_status(F) is None


# ---------------------------------------------------------------------------------------------------
# logits
# ---------------------------------------------------------------------------------------------------
def small_integers(shape, e4m3, g):
    """Codes of -3 .. 3."""
    v = torch.randint(-3, 4, shape, generator=g)
    return O.encode(v.double(), e4m3)


@pytest.mark.parametrize("scale", [3e4, 1e5, 1e6, 1e9, 1e20, 1e27])
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n,e4m3,bs,D", [(1, True, 16, 64), (3, True, 16, 128), (1, False, 24, 128), (3, False, 16, 256), (2, True, 16, 80)])
def test_attention_of_huge_logits(F, ctx, n, e4m3, bs, D, dt, scale):  # noqa: F811
    """Queries and keys of small integers, key scales of powers of two: every q . k * ks is a small multiple of 1/4, exact in
    fp32, and logits of different ones are at least scale / 4 > 2^12 apart. So the weights are 1 / (number of tokens that share
    the largest), 0 for the others, however the logits are rounded (by 2^-20 of themselves at most, and the largest is below
    9 * D * 2 * 2^2 / 4 < 2^15 of those steps; equal products are rounded alike, as they only differ by powers of two in
    their factors). What is left is the sum over equal weights (exact), one rounding of the quotient and of the value times
    its scale, and the result's own."""
    g = torch.Generator().manual_seed(n * 100 + D)
    lens = LENS + [90, 400]
    q, kc, vc, ks, vs, table, lens_t = attention_inputs(lens, n=n, e4m3=e4m3, bs=bs, D=D, dt=dt, seed=D + n)
    q = torch.randint(-3, 4, q.shape, generator=g).to(DT[dt])
    kc = small_integers(kc.shape, e4m3, g)
    ks = 2.0 ** torch.randint(-2, 1, ks.shape, generator=g)
    for sign in (1, -1):   # -1: every logit of some rows is far below zero
        kk = kc
        if sign < 0:
            kk = small_integers(kc.shape, e4m3, g)
            kk = O.encode(-O.decode(kk).abs() - 1, e4m3)
        qq = q if sign > 0 else (q.abs() + 1)
        want, (weight, _, _) = O.quantized_paged_attention(qq, kk, vc, ks, vs, table, lens_t, scale)
        got = F.quantized_paged_attention(qq.cuda(), kk.cuda(), vc.cuda(), ks.cuda(), vs.cuda(), table.cuda(), lens_t.cuda(), scale, ctx=ctx).cpu().double()
        ctx.release()
        tiny = 2.0 ** -25 if dt == "fp16" else 1e-38
        bound = weight * 2.0 ** -18 + want.abs() * torch.finfo(DT[dt]).eps / 2 + tiny
        ok = (got - want).abs() <= bound
        assert bool(ok.all()), f"{int((~ok).sum())} of {ok.numel()} values off, {int((~torch.isfinite(got)).sum())} not finite, first {(~ok).nonzero()[0].tolist()}"


# ---------------------------------------------------------------------------------------------------
# values
# ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("factor", [1e18, 1e25, 1e32, 1e35, 1e-30])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("n,e4m3,D", [(1, True, 64), (1, False, 128), (3, True, 128), (2, True, 256), (2, True, 40)])
def test_attention_of_huge_values(F, ctx, n, e4m3, D, dt, factor):  # noqa: F811
    """Values that only the 8-bit exponent of bf16 and fp32 reaches, next to ordinary ones; logits that grow along the request,
    so that the running maximum rises a little with almost every tile. The bounds are those of any other value: all of
    them are relative to sum p |v|, but the one of the weights' last bits, which goes by the value itself (sum |v|). (The 2^-18 to
    which weights of such values are held are far below what logits of hundreds may be off by.)"""
    lens = [1, 17, 40, 333, 700, 0]
    q, kc, vc, ks, vs, table, lens_t = attention_inputs(lens, n=n, e4m3=e4m3, D=D, dt=dt, seed=D)
    for i, L in enumerate(lens):
        blocks = table[i, :-(-L // 16)]
        ks[blocks] = 0.01 * torch.arange(1, len(blocks) + 1)[:, None] / 4
    vs = vs.clamp(max=0.3) * factor / 3     # 448 * 0.1 * 1e35 < 3.4e38
    check_attention(F, ctx, (q, kc, vc, ks, vs, table, lens_t))
    ctx.release()
    mixed = vs.clone()
    mixed[::2] /= factor
    check_attention(F, ctx, (q, kc, vc, ks, mixed, table, lens_t))
    ctx.release()


@pytest.mark.parametrize("factor", [1e13, 1e20, 1e34])
@pytest.mark.parametrize("n,e4m3,D", [(1, True, 64), (3, True, 128), (1, False, 256), (2, False, 40)])
def test_attention_of_huge_values_and_small_logits(F, ctx, n, e4m3, D, factor):  # noqa: F811
    """fp32 queries so small that logits hardly matter: what is left is how exactly weights of such values are held. A weight is
    2^(x - r) with x - r rounded at a magnitude below 128, by 2^-18, and its normaliser is a sum of such: 2 ln 2 * 2^-18 < 2^-17."""
    lens = [1, 17, 40, 333, 700, 0]
    q, kc, vc, ks, vs, table, lens_t = attention_inputs(lens, n=n, e4m3=e4m3, D=D, dt="fp32", seed=D, std=1e-4)
    vs = vs.clamp(max=0.3) * factor / 3
    vs[::2] /= factor
    args = (q, kc, vc, ks, vs, table, lens_t)
    want, sums = O.quantized_paged_attention(*args, 0.1)
    got = F.quantized_paged_attention(*[t.cuda() for t in args], 0.1, ctx=ctx).cpu().double()
    assert bool(((got - want).abs() <= bound_of(want, sums, 700, D, torch.float32) + sums[0] * 2.0 ** -17).all())


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("n,e4m3,D", [(1, True, 64), (3, True, 128), (1, False, 256), (2, False, 40)])
def test_attention_where_the_sum_of_the_values_is_infinite(F, ctx, n, e4m3, D, dt):  # noqa: F811
    """Equal weights over values just below the largest fp32: their mean is finite, their sum is not."""
    lens = [1, 40, 700, 0]
    q, kc, vc, ks, vs, table, lens_t = attention_inputs(lens, n=n, e4m3=e4m3, D=D, dt=dt, seed=D)
    vc = vc & 0x7f if e4m3 else vc.abs()
    vc = torch.where(vc == 0x7f, 0x7e, vc) if e4m3 else vc
    check_attention(F, ctx, (torch.zeros_like(q), kc, vc.to(kc.dtype), ks, torch.full_like(vs, 3.2e38 / (448 if e4m3 else 127)), table, lens_t))


# ---------------------------------------------------------------------------------------------------
# scales of the store
# ---------------------------------------------------------------------------------------------------
def store_both(F, ctx, x, table, cached, starts, cache, scale, wide):  # noqa: F811
    """The store's codes and scales; `wide`: in a cache whose rows are one byte too far apart for the vector kernel."""
    dc = []
    for _ in range(2):
        c = cache.cuda()
        if wide:
            big = torch.zeros(*cache.shape[:-1], cache.shape[-1] + 1, dtype=cache.dtype, device="cuda")
            big[..., :-1] = c
            c = big[..., :-1]
        dc.append(c)
    ds = [scale.cuda() for _ in range(2)]
    F.quantized_copy_kv(x.cuda(), x.cuda(), table.cuda(), cached.cuda(), starts.cuda(), *dc, *ds, ctx=ctx)
    return dc, ds


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_copy_into_blocks_of_any_scale(F, ctx, D, dt, e4m3, wide):  # noqa: F811
    """Blocks that someone else began, with scales of any mantissa (amax / 448 for one): the new values sit on the borders
    between two codes of the scale that the block has or grows to, and one step of their type beside them."""
    g = torch.Generator().manual_seed(D)
    B, H, bs = 24, 3, 16
    table = torch.randperm(B + 2, generator=g)[:B, None]
    cached = torch.randint(1, 8, (B,), generator=g)
    new = torch.randint(1, 8, (B,), generator=g)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)])
    scale = torch.rand(B + 2, H, generator=g) + 0.5
    scale[::3] = torch.randint(65, 128, scale[::3].shape, generator=g) / 64.0       # ties that bf16 holds
    scale *= 2.0 ** torch.randint(-20, 20, scale.shape, generator=g)
    grow = torch.randint(0, 4, (B, H), generator=g)
    who = torch.repeat_interleave(torch.arange(B), new)
    s = scale[table[who, 0]].double() * 2.0 ** grow[who]          # the scale that each block ends with
    # The value that makes it grow to that: a fresh block's scale for it is above s / 2 and not above s.
    top = 448.0 * 2.0 ** torch.floor(torch.log2(s)) if e4m3 else 127.0 * 0.75 * s
    v = O.e4m3_values()[:127] if e4m3 else torch.arange(0, 96, dtype=torch.float64)
    border = (v[:-1] + v[1:]) / 2
    border = border[border < (220 if e4m3 else 95)]
    T = int(new.sum())
    pick = border[torch.randint(0, len(border), (T, H, D), generator=g)] * (1 - 2.0 * torch.randint(0, 2, (T, H, D), generator=g))
    pick = pick * s[:, :, None]
    pick[:, :, 0] = top
    x = pick.to(DT[dt])
    eps = torch.finfo(DT[dt]).eps
    beside = torch.randint(-1, 2, (T, H, D), generator=g)
    beside[:, :, 0] = 0
    x = torch.where(beside == 0, x, (x.double() * (1 + eps * beside)).to(DT[dt]))
    cache = torch.randint(0, 120, (B + 2, bs, H, D), generator=g).to(torch.uint8 if e4m3 else torch.int8)
    want = O.quantized_copy(x, table, cached, starts, cache, scale)
    dc, ds = store_both(F, ctx, x, table, cached, starts, cache, scale, wide)
    for m in range(2):
        assert torch.equal(ds[m].cpu(), want[1])
        diff = dc[m].cpu() != want[0]
        assert not bool(diff.any()), f"{int(diff.sum())} of {T * H * D} codes differ, first at {diff.nonzero()[0].tolist()}"


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("e4m3", [True, False])
def test_copy_into_blocks_of_the_largest_scales(F, ctx, e4m3, wide):  # noqa: F811
    """Scales whose reciprocal is no normal fp32 number, and subnormal ones."""
    g = torch.Generator().manual_seed(1)
    scale = torch.tensor([[2.0 ** 125, 2.0 ** 126], [2.0 ** 127, 1.5 * 2.0 ** 126], [1.9 * 2.0 ** 127, 2.0 ** -127], [2.0 ** -140, 2.0 ** -126]])
    x = (torch.randn(8, 2, 64, generator=g) * 2.0 ** 125).float()
    x[6:, 0] *= 0.0
    x[4:6, 1] *= 2.0 ** -251
    x[6:, 1] *= 2.0 ** -251
    table, cached, starts = torch.arange(4)[:, None], torch.full((4,), 5), torch.arange(0, 9, 2)
    cache = torch.randint(0, 120, (4, 16, 2, 64), generator=g).to(torch.uint8 if e4m3 else torch.int8)
    want = O.quantized_copy(x, table, cached, starts, cache, scale)
    dc, ds = store_both(F, ctx, x, table, cached, starts, cache, scale, wide)
    for m in range(2):
        assert torch.equal(ds[m].cpu(), want[1])
        assert torch.equal(dc[m].cpu(), want[0])


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_copy_of_zeros_of_both_signs(F, ctx, dt, e4m3, wide):  # noqa: F811
    """A block of nothing but zeros has scale 0 and codes 0, whatever their signs; in a block with a scale a negative zero keeps its sign."""
    g = torch.Generator().manual_seed(4)
    x = torch.zeros(40, 2, 64)
    x[torch.rand(x.shape, generator=g) < 0.5] = -0.0
    x[20:, 1, 5] = 3.0
    x = x.to(DT[dt])
    table, cached, starts = torch.tensor([[0, 1], [2, 3]]), torch.tensor([0, 9]), torch.tensor([0, 20, 40])
    cache, scale = torch.zeros(5, 16, 2, 64, dtype=torch.uint8 if e4m3 else torch.int8), torch.zeros(5, 2)
    want = O.quantized_copy(x, table, cached, starts, cache, scale)
    dc, ds = store_both(F, ctx, x, table, cached, starts, cache, scale, wide)
    assert bool((want[0][:2] == 0).all()) and (not e4m3 or bool((want[0][2:4, :, 1] == 0x80).any()))
    for m in range(2):
        assert torch.equal(dc[m].cpu(), want[0]) and torch.equal(ds[m].cpu(), want[1])


# ---------------------------------------------------------------------------------------------------
# views
# ---------------------------------------------------------------------------------------------------
def test_slices_of_one_fused_tensor(F, ctx):  # noqa: F811
    """q and out are slices of one projection; lengths, offsets and slots are columns of one tensor."""
    args = attention_inputs(LENS, D=64, n=2)
    fused = torch.full((len(LENS), 2, 3, 8, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    views = {"q": fused[:, :, 0], "out": fused[:, :, 2]}
    check_attention(F, ctx, args, view=lambda kind, t: views[kind].copy_(t) if kind in views else t)
    assert bool((fused[:, :, 1] == 7).all()) and torch.equal(fused[:, :, 0].cpu(), args[0])
    i32 = dict(dtype=torch.int32, device="cuda")
    t = torch.full((8, 5), -3, **i32)
    t[:3, 0], t[:3, 1] = torch.tensor([4, 0, 9], **i32), torch.tensor([1, 5, 2], **i32)
    table = torch.full((3, 4), -1, **i32)
    table[0, 0], table[2, :3] = 0, torch.tensor([1, 2, 3], **i32)
    F.build_block_table(table, t[:3, 0], t[:3, 1], torch.arange(20, 0, -1, **i32), torch.zeros(1, **i32), 4, slot_map=t[:, 2], new_start=t[:4, 3], seq_lens=t[:3, 4],
                        free_next=torch.zeros(1, **i32), ctx=ctx)
    assert t[:, 0].tolist() == [4, 0, 9] + [-3] * 5 and t[:, 1].tolist() == [1, 5, 2] + [-3] * 5
    assert t[:, 3].tolist() == [0, 1, 6, 8] + [-3] * 4 and t[:, 4].tolist() == [5, 5, 11] + [-3] * 5
    # blocks taken: 20 | 19, 18 | none
    assert t[:, 2].tolist() == [80, 76, 77, 78, 79, 72, 13, 14]


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n,e4m3,D", [(1, True, 64), (3, True, 128), (2, False, 256), (1, False, 40)])
def test_attention_of_infinite_queries(F, ctx, n, e4m3, D, dt):  # noqa: F811
    """An infinity in a row of q makes every logit of that row infinite or NaN, hence the row NaN, also where all of them are -inf;
    rows that see no token stay zeros, and no other row is touched."""
    lens = [0, 1, 40, 16, 700, 300]
    q, kc, vc, ks, vs, table, lens_t = attention_inputs(lens, n=n, e4m3=e4m3, D=D, dt=dt, seed=D)
    kc[..., 5] = 0x30 if e4m3 else 17          # every key is positive here
    clean = q.clone()
    bad = torch.zeros(q.shape[:3], dtype=torch.bool)
    for i, (t, h, x) in enumerate(((0, 0, -math.inf), (n - 1, 1, -math.inf), (0, 2, math.inf), (n - 1, 3, -math.inf), (n - 1, 7, -math.inf), (0, 4, math.inf))):
        q[i, t, h, 5] = x
        clean[i, t, h, 5] = 0
        bad[i, t, h] = lens[i] - (n - 1 - t) > 0
    got = F.quantized_paged_attention(q.cuda(), kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(), table.cuda(), lens_t.cuda(), 0.1, ctx=ctx).cpu()
    assert torch.equal(torch.isnan(got), bad[..., None].expand_as(got))
    want, sums = O.quantized_paged_attention(clean, kc, vc, ks, vs, table, lens_t, 0.1)
    ok = (got.double() - want).abs() <= bound_of(want, sums, 700, D, q.dtype)
    assert bool((ok | bad[..., None]).all())
