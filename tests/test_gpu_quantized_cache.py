"""The block-paged cache in 8 bits on the GPU, through the C ABI: tables and slots exactly, codes and scales exactly, and the
attention against the definition in 64 bits within bounds derived from its roundings."""
import math

import pytest
import torch

from oracle import quantized_cache as O

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def F(built_libs):
    from diopi_b200 import functions
    return functions


@pytest.fixture()
def ctx():
    from diopi_b200.runtime import Context
    return Context()


@pytest.fixture(autouse=True)
def no_status_left(F):
    """Each test starts and ends without a kernel status of another one: a housekeeping-sized op takes it."""
    yield
    torch.cuda.synchronize()
    take_status(F)


def take_status(F):
    """The status an earlier kernel left, as text, or None."""
    from diopi_b200.runtime import DiopiError
    torch.cuda.synchronize()
    z = torch.zeros(1, 1, 1, device="cuda")
    try:
        F.destindex_copy_kv(z, torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, 1, 1, device="cuda"))
    except DiopiError as e:
        torch.cuda.synchronize()
        return str(e)
    torch.cuda.synchronize()
    return None


# ---------------------------------------------------------------------------------------------------
# tables
# ---------------------------------------------------------------------------------------------------
def run_tables(F, cached, new, bs, cols, *, start=0, spare=6, T=None, wide=None, dt=torch.int32, seed=0, n_free=None):
    g = torch.Generator().manual_seed(seed)
    cached, new = torch.tensor(cached, dtype=torch.int64), torch.tensor(new, dtype=torch.int64)
    B = cached.shape[0]
    held = (cached.clamp(0, cols * bs) + bs - 1) // bs
    perm = torch.randperm(int(held.sum()) + 4 * B * cols + spare, generator=g)
    table = torch.full((B, cols), -7, dtype=torch.int64)
    at = 0
    for i in range(B):
        table[i, :held[i]] = perm[at:at + int(held[i])]
        at += int(held[i])
    free = perm[at:] if n_free is None else perm[at:at + n_free]
    T = int(new.clamp(min=0).sum()) if T is None else T
    wide_t = None if wide is None else torch.full((B, wide), -9, dtype=torch.int64)
    want = O.build_block_table(table, cached, new, free, start, bs, T, wide_t)
    dev = lambda t: None if t is None else t.to(dt).cuda()  # noqa: E731
    d_table, d_wide = dev(table), dev(wide_t)
    out = dict(slot_map=torch.full((T,), 5, dtype=dt, device="cuda"), new_start=torch.full((B + 1,), 5, dtype=dt, device="cuda"),
               seq_lens=torch.full((B,), 5, dtype=dt, device="cuda"), free_next=torch.full((1,), 5, dtype=dt, device="cuda"))
    F.build_block_table(d_table, dev(cached), dev(new), dev(free), dev(torch.tensor([start])), bs, token_table=d_wide, **out)
    got = (d_table, out["slot_map"], out["new_start"], out["seq_lens"], out["free_next"], d_wide)
    for name, a, b in zip(("table", "slots", "starts", "lens", "next", "wide"), got, want):
        if b is not None:
            b = torch.tensor([b]) if isinstance(b, int) else b
            assert torch.equal(a.cpu().long(), b.long()), name


@pytest.mark.parametrize("bs", [1, 3, 16, 64])
@pytest.mark.parametrize("dt", [torch.int32, torch.int64])
def test_tables_of_lengths_around_blocks(F, bs, dt):
    edge = [0, 1, bs - 1, bs, bs + 1, 3 * bs]
    cached = [c for c in edge for _ in edge]
    new = [n for _ in edge for n in edge]
    run_tables(F, cached, new, bs, 7, dt=dt, wide=7 * bs, start=2)
    assert take_status(F) is None


@pytest.mark.parametrize("B", [1, 31, 257, 1500])
def test_tables_of_a_decode_step(F, B):
    g = torch.Generator().manual_seed(B)
    run_tables(F, torch.randint(0, 200, (B,), generator=g).tolist(), [1] * B, 16, 14, wide=224)
    assert take_status(F) is None


def test_tables_of_long_prompts(F):
    run_tables(F, [0, 5, 0], [30001, 0, 12345], 32, 1000, T=43000, wide=30100)
    assert take_status(F) is None


def test_tables_of_an_empty_batch(F):
    run_tables(F, [], [], 16, 3, T=4, start=3)


def test_tables_when_blocks_run_out(F):
    run_tables(F, [3, 16, 9], [20, 40, 30], 16, 6, n_free=4, wide=96)
    assert "status 4" in take_status(F)


def test_tables_of_requests_beyond_their_row(F):
    run_tables(F, [30, 70, 5, -3], [40, 2, 7, 4], 16, 4)
    assert "status 4" in take_status(F)


def test_tables_of_slots_beyond_the_slot_map(F):
    bs, i32 = 16, dict(dtype=torch.int32, device="cuda")
    slot_map, guard = torch.full((8,), 77, **i32), torch.full((2, 8), 77, **i32)
    slot_map = guard[0]
    F.build_block_table(torch.zeros(2, 4, **i32), torch.zeros(2, **i32), torch.tensor([6, 9], **i32), torch.arange(8, **i32), torch.zeros(1, **i32), bs,
                        slot_map=slot_map, new_start=torch.zeros(3, **i32), seq_lens=torch.zeros(2, **i32), free_next=torch.zeros(1, **i32))
    assert slot_map.tolist() == [0, 1, 2, 3, 4, 5, 16, 17] and guard[1].tolist() == [77] * 8
    assert "status 4" in take_status(F)


def test_tables_of_strided_tensors(F):
    """A table, lengths and a slot map that are columns or slices of wider tensors."""
    i32 = dict(dtype=torch.int32, device="cuda")
    big = torch.full((3, 20), -1, **i32)
    lens = torch.tensor([[4, 1], [0, 5], [17, 2]], **i32)
    slots = torch.full((8, 3), 9, **i32)
    F.build_block_table(big[:, 2:14:3], lens[:, 0], lens[:, 1], torch.arange(20, 0, -1, **i32)[::2], torch.tensor([1], **i32), 4, slot_map=slots[:, 1],
                        new_start=torch.zeros(8, **i32)[::2], seq_lens=torch.zeros(6, **i32)[::2], free_next=torch.zeros(1, **i32))
    # held: 1, 0, 5 > 4 columns (17 tokens are cut to 16, so nothing fits any more)
    assert big[0, 2:14:3].tolist() == [-1, 18, -1, -1] and big[1, 2:14:3].tolist() == [16, 14, -1, -1]
    assert slots[:, 1].tolist() == [72, 64, 65, 66, 67, 56, O.NO_SLOT, O.NO_SLOT] and slots[:, 0].tolist() == [9] * 8
    assert "status 4" in take_status(F)


def test_slots_that_do_not_fit_32_bits(F):
    i32, i64 = dict(dtype=torch.int32, device="cuda"), dict(dtype=torch.int64, device="cuda")
    for kind, want in ((i32, O.NO_SLOT), (i64, (1 << 30) * 16)):
        slot_map = torch.zeros(1, **kind)
        F.build_block_table(torch.zeros(1, 2, **i32), torch.zeros(1, **i32), torch.ones(1, **i32), torch.tensor([1 << 30], **i32), torch.zeros(1, **i32), 16,
                            slot_map=slot_map, new_start=torch.zeros(2, **i32), seq_lens=torch.zeros(1, **i32), free_next=torch.zeros(1, **i32))
        assert slot_map.tolist() == [want]
        assert (take_status(F) is None) == (kind is i64)


# ---------------------------------------------------------------------------------------------------
# the store
# ---------------------------------------------------------------------------------------------------
def paged(B, lens, bs, cols, blocks, g):
    """A block table that names distinct blocks for what the requests hold, and nonsense behind that."""
    perm = torch.randperm(blocks, generator=g)
    table = torch.full((B, cols), 1 << 29, dtype=torch.int64)
    at = 0
    for i, L in enumerate(lens):
        n = -(-L // bs)
        assert at + n <= blocks
        table[i, :n] = perm[at:at + n]
        at += n
    return table


def random_codes(shape, e4m3, g):
    c = torch.randint(-127, 128, shape, generator=g)
    if not e4m3:
        return c.to(torch.int8)
    c = torch.where((c & 127) == 127, torch.zeros_like(c), c)
    return (c & 255).to(torch.uint8)


def check_copy(F, ctx, cached, new, *, bs=16, H=3, D=64, dt="bf16", e4m3=True, fix=None, view=None, T_extra=0, idx=torch.int32, std=0.6, seed=0):
    g = torch.Generator().manual_seed(seed)
    B, after = len(cached), [c + n for c, n in zip(cached, new)]
    cols = max(-(-a // bs) for a in after) + 1
    blocks = sum(-(-a // bs) for a in after) + 3
    table = paged(B, after, bs, cols, blocks, g)
    T = sum(new) + T_extra
    starts = torch.tensor([0] + new).cumsum(0)
    xs, caches, scales = [], [], []
    for m in range(2):
        xs.append((torch.randn(T, H, D, generator=g) * std).to(DT[dt]))
        caches.append(random_codes((blocks, bs, H, D), e4m3, g))
        # some blocks' scales are far too small, some are far too large, some fit
        s = torch.tensor([2.0 ** -9, 2.0 ** -12, 2.0 ** -6, 0.0, 2.0])[torch.randint(0, 5, (blocks, H), generator=g)]
        if not e4m3:
            s = s * (1 + torch.rand(blocks, H, generator=g))
        scales.append(s)
    if fix is not None:
        fix(xs, starts)
    want = [O.quantized_copy(x, table, torch.tensor(cached), starts, c, s) for x, c, s in zip(xs, caches, scales)]
    view = view or (lambda kind, t: t)
    dx = [view("x", x.cuda()) for x in xs]
    dc, ds = [view("cache", c.cuda()) for c in caches], [view("scale", s.cuda()) for s in scales]
    F.quantized_copy_kv(dx[0], dx[1], table.to(idx).cuda(), torch.tensor(cached, dtype=idx).cuda(), starts.to(idx).cuda(), dc[0], dc[1], ds[0], ds[1], ctx=ctx)
    for m in range(2):
        assert torch.equal(ds[m].cpu(), want[m][1]), f"scales of {'kv'[m]}"
        diff = dc[m].cpu() != want[m][0]
        assert not bool(diff.any()), f"{int(diff.sum())} codes of {'kv'[m]} differ, first at {diff.nonzero()[0].tolist()}"
    return dc, ds


EDGES = ([0, 0, 5, 16, 15, 31, 40, 0, 7], [1, 16, 11, 1, 2, 33, 0, 50, 9])


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [64, 128, 256, 80, 48, 20])
def test_copy_widths_and_types(F, ctx, D, dt, e4m3):
    check_copy(F, ctx, *EDGES, D=D, dt=dt, e4m3=e4m3, seed=D)
    assert take_status(F) is None


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("bs", [1, 8, 24, 32, 48, 64, 128, 130, 256])
def test_copy_block_sizes(F, ctx, bs, e4m3):
    cached, new = EDGES
    check_copy(F, ctx, cached + [bs, bs - 1, 3], new + [2 * bs + 1, 2, bs], bs=bs, D=64, H=5, e4m3=e4m3, seed=bs, dt="fp16")


@pytest.mark.parametrize("B", [1, 3, 256, 700])
def test_copy_of_a_decode_step(F, ctx, B):
    g = torch.Generator().manual_seed(B)
    check_copy(F, ctx, torch.randint(0, 40, (B,), generator=g).tolist(), [1] * B, H=8, D=64, idx=torch.int64)


def test_copy_ties_and_borders(F, ctx):
    """Values on the borders between codes: x / s exactly between two codes, and one bit beside it."""
    def fix(xs, starts):
        for x in xs:
            x[:, :, 0] = 127.0    # int8: s = 1 exactly
            k = torch.arange(x[:, :, 1:].numel()).reshape(x[:, :, 1:].shape) % 253 - 126
            x[:, :, 1:] = k + 0.5
            x[:, 0, 1::2] *= 1 + 2.0 ** -23
            x[:, 1, 1::2] *= 1 - 2.0 ** -23
    check_copy(F, ctx, [0, 0], [16, 20], dt="fp32", e4m3=False, fix=fix)

    def fix8(xs, starts):
        v = O.e4m3_values()[:127]
        mid = torch.cat([(v[:-1] + v[1:]) / 2, v, -v]).float()
        for x in xs:
            x[:] = mid[torch.arange(x.numel()).reshape(x.shape) % mid.numel()]
            x[:, :, 0] = 448.0
            x[:, 1, 1::2] *= 1 + 2.0 ** -23
    check_copy(F, ctx, [0, 0], [16, 20], dt="fp32", e4m3=True, fix=fix8)


@pytest.mark.parametrize("std", [1e-30, 1e-6, 3e4])
@pytest.mark.parametrize("e4m3", [True, False])
def test_copy_magnitudes(F, ctx, std, e4m3):
    check_copy(F, ctx, *EDGES, dt="fp32", e4m3=e4m3, std=std, H=4)


@pytest.mark.parametrize("D", [64, 20])
@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_copy_zeros_infinities_and_nan(F, ctx, dt, e4m3, D):
    def fix(xs, starts):
        for x in xs:
            x[0] = 0.0                    # a block of zeros
            x[3, 0, 2] = math.inf
            x[4, 1, 3] = -math.inf
            x[5, 0, 4] = math.nan
            x[20:40, 2] = math.nan        # a head with nothing finite in a whole block
            x[int(starts[5])] = math.inf
            x[6, 0] = -0.0
    check_copy(F, ctx, *EDGES, dt=dt, e4m3=e4m3, fix=fix, D=D)


@pytest.mark.parametrize("e4m3", [True, False])
def test_copy_strides(F, ctx, e4m3):
    """Rows that are slices of a fused projection, a head-major cache, scales inside a wider tensor: the vector kernel; then
    an odd offset and a transposed width: the element one."""
    def make(shift):
        def view(kind, t):
            if kind == "x":
                big = torch.full((t.shape[0], 3 * t.shape[1], t.shape[2] + shift), 7.0, dtype=t.dtype, device="cuda")
                v = big[:, t.shape[1]:2 * t.shape[1], shift:]
            elif kind == "cache":
                v = torch.zeros(t.shape[0], t.shape[2], t.shape[1], t.shape[3] + shift, dtype=t.dtype, device="cuda")[..., shift:].transpose(1, 2)
            else:
                v = torch.zeros(t.shape[1], t.shape[0] + 2, device="cuda")[:, 1:-1].t()
            v.copy_(t)
            return v
        return view
    for shift in (0, 3):
        check_copy(F, ctx, *EDGES, view=make(shift), e4m3=e4m3)
    check_copy(F, ctx, *EDGES, view=lambda kind, t: t.transpose(-1, -2).contiguous().transpose(-1, -2) if kind != "scale" else t, e4m3=e4m3)


def test_copy_leaves_rows_behind_the_last_request(F, ctx):
    check_copy(F, ctx, [0, 18], [5, 3], T_extra=9)
    assert take_status(F) is None


def test_copy_skips_blocks_outside_the_cache(F, ctx):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(40, 2, 64, generator=g).half()
    for table in ([[0, -1], [5, 1]], [[2, 99], [1 << 30, 4]]):
        cache, scale = torch.zeros(6, 16, 2, 64, dtype=torch.int8), torch.ones(6, 2)
        args = (torch.tensor(table), torch.tensor([0, 0]), torch.tensor([0, 20, 40]))
        want = O.quantized_copy(x, *args, cache, scale)
        dc, ds = [cache.cuda(), cache.cuda()], [scale.cuda(), scale.cuda()]
        F.quantized_copy_kv(x.cuda(), x.cuda(), *[a.cuda() for a in args], *dc, *ds, ctx=ctx)
        assert torch.equal(dc[0].cpu(), want[0]) and torch.equal(dc[1].cpu(), want[0]) and torch.equal(ds[0].cpu(), want[1])
        assert "status 1" in take_status(F)


def test_copy_of_tokens_beyond_the_table_or_the_rows(F, ctx):
    """cached + new past the row of the table, offsets past the rows of k: what fits is written, the rest is reported or not there."""
    g = torch.Generator().manual_seed(6)
    x = torch.randn(20, 2, 64, generator=g).half()
    table, cached, starts = torch.tensor([[0, 1], [2, 3]]), torch.tensor([25, 3]), torch.tensor([0, 12, 40])
    cache, scale = torch.zeros(6, 16, 2, 64, dtype=torch.int8), torch.zeros(6, 2)
    want = O.quantized_copy(x, table, cached, starts, cache, scale)
    dc, ds = [cache.cuda(), cache.cuda()], [scale.cuda(), scale.cuda()]
    F.quantized_copy_kv(x.cuda(), x.cuda(), table.cuda(), cached.cuda(), starts.cuda(), *dc, *ds, ctx=ctx)
    assert torch.equal(dc[0].cpu(), want[0]) and torch.equal(ds[1].cpu(), want[1])
    assert "status 1" in take_status(F)


@pytest.mark.parametrize("e4m3", [True, False])
def test_copy_token_by_token_stays_near(F, ctx, e4m3):
    """A block filled one token at a time, its scale growing on the way: still near what was written. Each of the at most 12
    growths can add half a step of its own scale, and every scale is at most half the next: 1/2 + 1/4 + ... < 1 final step;
    the last rounding adds half a step (e4m3: half a step of the value, 2^-4 of it, in the place of the grid's)."""
    g = torch.Generator().manual_seed(8)
    H, D = 2, 64
    x = (torch.randn(16, H, D, generator=g) * torch.logspace(-2, 1, 16)[:, None, None]).half()
    cache = [torch.zeros(1, 16, H, D, dtype=torch.uint8 if e4m3 else torch.int8, device="cuda") for _ in range(2)]
    scale = [torch.zeros(1, H, device="cuda") for _ in range(2)]
    table, one = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    for t in range(16):
        F.quantized_copy_kv(x[t:t + 1].cuda(), x[t:t + 1].cuda(), table, torch.tensor([t], dtype=torch.int32, device="cuda"), one, *cache, *scale, ctx=ctx)
    s = scale[0].cpu().double()[0][None, :, None]
    got = O.decode(cache[0].cpu()[0]) * s
    far = (got - x.double()).abs()
    bound = 1.5 * s * (2.0 ** -9 if e4m3 else 1.0) + (x.double().abs() * 2.0 ** -4 if e4m3 else 0)
    assert bool((far <= bound).all())


# ---------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------
def bound_of(out, sums, L, D, dt):
    """What a kernel that is right may be off by. The logits: q is held with 2^-22 of its row's largest value or better and the
    products are summed in fp32, which truncates each partial sum by 2^-22 of the terms' magnitudes at most, D / 16 + 4
    times: e = (D / 16 + 5) * 2^-22 * sum |q||k|. A weight is then off by 2 e (numerator) and its normaliser by as much;
    the exponential adds 2^-21. The weights meet the values in fp16 (2^-11 of each) or, for fp32, as two fp16 parts (2^-21),
    and L / 16 + 16 sums are rounded to fp32. All of it is relative to sum p |v|. fp16 ends at 2^-24: a weight is held in it
    scaled so that the largest one of its 16 tokens is 2^15, hence off by half of 2^-24 * 2^-15 = 2^-40 of that one at most
    (which is 1 at most), and so is the lower one of two parts: 2^-40 * sum |v|. Last, half a step of the result."""
    weight, reach, logit = sums
    e = (D / 16 + 5) * 2.0 ** -22 * logit[..., None]
    w = 4 * e + 2.0 ** -20 + (2.0 ** -21 if dt == torch.float32 else 2.0 ** -11) + (L / 16 + 16) * 2.0 ** -23
    tiny = 2.0 ** -25 if dt == torch.float16 else 1e-38   # half the smallest subnormal of the result's type
    return weight * w + reach * 2.0 ** -40 + out.abs() * torch.finfo(dt).eps / 2 + tiny


def attention_inputs(lens, *, bs=16, Hkv=2, group=4, n=1, D=128, dt="bf16", e4m3=True, seed=0, std=1.0, extra_cols=2):
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    blocks = sum(-(-L // bs) for L in lens) + 2
    cols = max([-(-L // bs) for L in lens] + [0]) + extra_cols
    table = paged(B, lens, bs, cols, blocks, g)
    kc, vc = random_codes((blocks, bs, Hkv, D), e4m3, g), random_codes((blocks, bs, Hkv, D), e4m3, g)
    unit = 1 / 60 if not e4m3 else 1 / 40
    ks, vs = [unit * torch.exp(torch.randn(blocks, Hkv, generator=g)) for _ in range(2)]
    q = (torch.randn(B, n, Hkv * group, D, generator=g) * std).to(DT[dt])
    return q, kc, vc, ks, vs, table, torch.tensor(lens)


def check_attention(F, ctx, args, *, idx=torch.int32, view=None, scale=None, squeeze=False):
    q, kc, vc, ks, vs, table, lens = args
    scale = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    want, sums = O.quantized_paged_attention(*args, scale)
    view = view or (lambda kind, t: t)
    dq = view("q", (q[:, 0] if squeeze else q).cuda())
    got = F.quantized_paged_attention(dq, view("cache", kc.cuda()), view("cache", vc.cuda()), view("scale", ks.cuda()), view("scale", vs.cuda()),
                                      table.to(idx).cuda(), lens.to(idx).cuda(), scale, ctx=ctx, out=view("out", torch.full_like(dq, 9.0)))
    got = (got[:, None] if squeeze else got).cpu().double()
    far = (got - want).abs()
    ok = far <= bound_of(want, sums, int(lens.max()) if lens.numel() else 0, q.shape[-1], q.dtype)
    assert bool(ok.all()), f"{int((~ok).sum())} of {ok.numel()} values off, worst {float((far / (sums[0] + 1e-30)).max()):.3g} of the weight, first {(~ok).nonzero()[0].tolist()}"
    return got


LENS = [0, 1, 2, 15, 16, 17, 31, 33, 64, 100, 257]


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [64, 128, 256, 80, 16, 40, 320])
def test_attention_widths_and_types(F, ctx, D, dt, e4m3):
    check_attention(F, ctx, attention_inputs(LENS, D=D, dt=dt, e4m3=e4m3, seed=D), squeeze=True)
    assert take_status(F) is None


@pytest.mark.parametrize("Hkv,group", [(1, 1), (1, 16), (1, 17), (1, 71), (2, 8), (3, 5), (4, 1), (5, 3), (6, 2), (7, 1), (8, 4), (8, 1), (11, 2), (16, 2), (1, 130), (12, 1), (2, 33)])
def test_attention_head_layouts(F, ctx, Hkv, group):
    check_attention(F, ctx, attention_inputs([0, 1, 40, 333, 16, 129], Hkv=Hkv, group=group, D=64, dt="fp16", seed=Hkv * 100 + group))


@pytest.mark.parametrize("bs", [1, 3, 8, 17, 24, 32, 48, 64, 100, 128, 272])
@pytest.mark.parametrize("e4m3", [True, False])
def test_attention_block_sizes(F, ctx, bs, e4m3):
    args = attention_inputs(LENS + [bs, bs + 1, 2 * bs - 1], bs=bs, D=64, e4m3=e4m3, seed=bs)
    check_attention(F, ctx, args, idx=torch.int64)
    check_attention(F, ctx, attention_inputs(LENS + [bs, 700], bs=bs, D=128, e4m3=e4m3, seed=bs, n=3, group=3))


@pytest.mark.parametrize("bs", [8, 24, 40])
def test_attention_ignores_the_next_block(F, ctx, bs):
    """Blocks that do not fill a tile: what lies behind a block in memory (NaN here) is another block's."""
    lens = [bs, 3 * bs - 1, 5, 0]
    q, kc, vc, ks, vs, table, lens_t = attention_inputs(lens, D=64, bs=bs, dt="fp16")
    used = torch.cat([table[i, :-(-L // bs)] for i, L in enumerate(lens)])
    keep = [c[used].clone() for c in (kc, vc)]
    for c, k in zip((kc, vc), keep):
        c[:] = 0x7f
        c[used] = k
        for i, L in enumerate(lens):
            if L % bs:
                c[table[i, L // bs], L % bs:] = 0x7f
    check_attention(F, ctx, (q, kc, vc, ks, vs, table, lens_t))


@pytest.mark.parametrize("n", [2, 3, 5, 16])
@pytest.mark.parametrize("D,Hkv,group", [(64, 2, 4), (128, 1, 1), (96, 3, 2), (40, 2, 2)])
def test_attention_of_several_new_tokens(F, ctx, n, D, Hkv, group):
    """Rows of requests with fewer tokens than that see none: zeros."""
    args = attention_inputs([0, 1, 2, 4, 5, 16, 17, 18, 47, 300], n=n, D=D, Hkv=Hkv, group=group, seed=n)
    got = check_attention(F, ctx, args)
    assert bool((got[0] == 0).all()) and bool((got[1, :n - 1] == 0).all())


@pytest.mark.parametrize("B,L", [(1, 5000), (3, 2100), (300, 20), (700, 3)])
def test_attention_splits(F, ctx, B, L):
    """One long request over all SMs, and more requests than SMs."""
    g = torch.Generator().manual_seed(B)
    lens = [L] + torch.randint(0, L + 1, (B - 1,), generator=g).tolist()
    check_attention(F, ctx, attention_inputs(lens, D=64, Hkv=2, group=2, seed=B))


def test_attention_large_logits_and_scales(F, ctx):
    """Logits of hundreds, queries far beyond fp16, scales that differ by powers of ten between blocks."""
    q, kc, vc, ks, vs, table, lens = attention_inputs([200, 77, 16, 500], std=30.0, dt="bf16")
    check_attention(F, ctx, (q, kc, vc, ks, vs, table, lens))
    vs = vs * 10.0 ** torch.randint(-4, 4, vs.shape, generator=torch.Generator().manual_seed(1))
    check_attention(F, ctx, (q, kc, vc, ks, vs, table, lens))
    check_attention(F, ctx, ((q.float() * 1e6).bfloat16(), kc, vc, ks * 1e-6, vs, table, lens))
    check_attention(F, ctx, ((q.float() * 1e-8).bfloat16(), kc, vc, ks * 1e8, vs, table, lens))
    ks = ks.clone()
    ks[::2] = 0.0     # blocks that hold nothing but zeros
    vs[::3] = 0.0
    check_attention(F, ctx, (q, kc, vc, ks, vs, table, lens))


@pytest.mark.parametrize("D", [64, 128, 256, 40])
@pytest.mark.parametrize("n", [1, 3])
def test_attention_ignores_what_lies_behind_the_last_token(F, ctx, D, n):
    """NaN codes in positions behind the length, in blocks of nobody, and nonsense in the table's unused columns."""
    lens = [1, 15, 16, 18, 40, 0]
    q, kc, vc, ks, vs, table, lens_t = attention_inputs(lens, D=D, n=n, dt="fp16")
    for c in (kc, vc):
        for i, L in enumerate(lens):
            if L % 16:
                c[table[i, L // 16], L % 16:] = 0x7f
        used = torch.cat([table[i, :-(-L // 16)] for i, L in enumerate(lens)])
        rest = torch.ones(c.shape[0], dtype=torch.bool)
        rest[used] = False
        c[rest] = 0xff
    check_attention(F, ctx, (q, kc, vc, ks, vs, table, lens_t))
    assert take_status(F) is None


def test_attention_hands_nan_on(F, ctx):
    """A NaN in q or in a token that is seen reaches the rows that see it, and no other."""
    q, kc, vc, ks, vs, table, lens = attention_inputs([40, 40, 40], D=64, Hkv=2, group=2, dt="fp16")
    q[0, 0, 1, 3] = math.nan
    kc[table[1, 1], 2, 0, 5] = 0x7f
    vc[table[2, 0], 9, 1, 7] = 0x7f
    got = F.quantized_paged_attention(q.cuda(), kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(), table.cuda(), lens.cuda(), 0.1, ctx=ctx).cpu()
    bad = torch.zeros(3, 1, 4, 64, dtype=torch.bool)
    bad[0, 0, 1] = True
    bad[1, 0, :2] = True
    bad[2, 0, 2:, 7] = True
    assert torch.equal(torch.isnan(got), bad)


@pytest.mark.parametrize("D,group,n", [(64, 2, 3), (128, 1, 2), (128, 5, 4), (256, 2, 3), (40, 2, 3)])
def test_attention_keeps_nan_from_the_tokens_before_it(F, ctx, D, group, n):
    """A NaN value of a new token is seen by that token's rows and those after it, not by the rows of the tokens before it."""
    lens = [40, 33, n, 18]
    q, kc, vc, ks, vs, table, lens_t = attention_inputs(lens, D=D, Hkv=2, group=group, n=n, dt="fp32" if D == 64 else "bf16")
    clean = vc.clone()
    bad = torch.zeros(len(lens), n, 2 * group, D, dtype=torch.bool)
    for i, (L, t, h, d) in enumerate(zip(lens, (n - 1, 0, n - 1, 1), (0, 1, 0, 1), (3, D - 1, 0, D // 2))):
        pos = L - n + t
        vc[table[i, pos // 16], pos % 16, h, d] = 0xff if i % 2 else 0x7f
        clean[table[i, pos // 16], pos % 16, h, d] = 0
        bad[i, t:, h * group:(h + 1) * group, d] = True
    kc[table[3, 1], 1, 0, 5] = 0x7f          # the last token's key, of head 0
    bad[3, n - 1:, :group] = True
    got = F.quantized_paged_attention(q.cuda(), kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(), table.cuda(), lens_t.cuda(), 0.1, ctx=ctx).cpu()
    assert torch.equal(torch.isnan(got), bad)
    kc[table[3, 1], 1, 0, 5] = 0
    want, sums = O.quantized_paged_attention(q, kc, clean, ks, vs, table, lens_t, 0.1)
    ok = (got.double() - want).abs() <= bound_of(want, sums, 40, D, q.dtype)
    assert bool((ok | bad).all())


@pytest.mark.parametrize("e4m3", [True, False])
def test_attention_strides(F, ctx, e4m3):
    """q as a slice of a fused projection, a head-major cache, scales inside a wider tensor, an odd offset of the cache."""
    def make(shift, qshift):
        def view(kind, t):
            if kind in ("q", "out"):
                v = torch.full((*t.shape[:-2], 3 * t.shape[-2], t.shape[-1] + qshift), 7.0, dtype=t.dtype, device="cuda")[..., t.shape[-2]:2 * t.shape[-2], qshift:]
            elif kind == "cache":
                v = torch.zeros(t.shape[0], t.shape[2], t.shape[1], t.shape[3] + shift, dtype=t.dtype, device="cuda")[..., shift:].transpose(1, 2)
            else:
                v = torch.zeros(t.shape[1], t.shape[0] + 2, device="cuda")[:, 1:-1].t()
            return v.copy_(t)
        return view
    args = attention_inputs(LENS, D=64, e4m3=e4m3, n=2)
    for shift, qshift in ((0, 0), (16, 1), (16, 8), (3, 0)):
        check_attention(F, ctx, args, view=make(shift, qshift))
    check_attention(F, ctx, args, view=lambda kind, t: t.transpose(-1, -2).contiguous().transpose(-1, -2) if kind == "cache" else t)


def test_attention_leaves_out_blocks_outside_the_cache(F, ctx):
    for bs, D in ((16, 64), (8, 64), (16, 40)):
        q, kc, vc, ks, vs, table, lens = attention_inputs([100, 40, 30], D=D, bs=bs)
        table[0, 2], table[1, 0], table[2] = -1, kc.shape[0], 1 << 30
        got = check_attention(F, ctx, (q, kc, vc, ks, vs, table, lens))
        assert bool((got[2] == 0).all())
        assert "status 1" in take_status(F)


def test_attention_clamps_lengths_to_the_table(F, ctx):
    q, kc, vc, ks, vs, table, lens = attention_inputs([48, 48], D=64, extra_cols=0)
    check_attention(F, ctx, (q, kc, vc, ks, vs, table, torch.tensor([1000, -5])))


def test_attention_into_its_own_query(F, ctx):
    args = attention_inputs(LENS + [900], D=128, n=2, Hkv=1, group=20)
    q, kc, vc, ks, vs, table, lens = args
    want, sums = O.quantized_paged_attention(*args, 0.1)
    d = q.cuda()
    F.quantized_paged_attention(d, kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(), table.cuda(), lens.cuda(), 0.1, ctx=ctx, out=d)
    assert bool(((d.cpu().double() - want).abs() <= bound_of(want, sums, 900, 128, q.dtype)).all())


def test_attention_empty_calls(F, ctx):
    for B, H in ((0, 8), (2, 8)):
        q = torch.full((B, H, 64), 3.0, dtype=torch.float16, device="cuda")
        c = torch.zeros(0, 16, 2, 64, dtype=torch.int8, device="cuda")
        s = torch.zeros(0, 2, device="cuda")
        out = F.quantized_paged_attention(q, c, c, s, s, torch.zeros(B, 0, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda"), 1.0, ctx=ctx)
        assert out.shape == q.shape and bool((out == 0).all())


def test_attention_offsets_beyond_32_bits(F, ctx):
    """A cache of more than 2^32 bytes whose last blocks are read and written."""
    bs, Hkv, D = 16, 8, 128
    blocks = (1 << 32) // (bs * Hkv * D) + 40
    g = torch.Generator().manual_seed(3)
    cache = [torch.empty(blocks, bs, Hkv, D, dtype=torch.int8, device="cuda") for _ in range(2)]
    scale = [torch.zeros(blocks, Hkv, device="cuda") for _ in range(2)]
    x = [torch.randn(600, Hkv, D, generator=g).half() for _ in range(2)]
    ids = torch.arange(38) + blocks - 38
    table, starts = ids[None].to(torch.int32).cuda(), torch.tensor([0, 600], dtype=torch.int32, device="cuda")
    F.quantized_copy_kv(x[0].cuda(), x[1].cuda(), table, torch.zeros(1, dtype=torch.int32, device="cuda"), starts, *cache, *scale, ctx=ctx)
    local = torch.arange(38)[None]
    want = [O.quantized_copy(t, local, torch.tensor([0]), torch.tensor([0, 600]), torch.zeros(38, bs, Hkv, D, dtype=torch.int8), torch.zeros(38, Hkv)) for t in x]
    for m in range(2):
        assert torch.equal(scale[m][-38:].cpu(), want[m][1])
        assert torch.equal(cache[m][-38:].cpu().reshape(-1, Hkv, D)[:600], want[m][0].reshape(-1, Hkv, D)[:600])
    q = torch.randn(1, 1, 8, D, generator=g).half()
    lens = torch.tensor([600])
    o, sums = O.quantized_paged_attention(q, want[0][0], want[1][0], want[0][1], want[1][1], local, lens, 0.1)
    got = F.quantized_paged_attention(q.cuda(), *cache, *scale, table, lens.cuda(), 0.1, ctx=ctx).cpu().double()
    assert bool(((got - o).abs() <= bound_of(o, sums, 600, D, torch.float16)).all())


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_attention_gives_the_same_bits_again(F, ctx, dt):
    args = [t.cuda() for t in attention_inputs([1000, 3, 0, 517, 64], D=128, dt=dt, n=2)]
    first = F.quantized_paged_attention(*args, 0.1, ctx=ctx)
    for _ in range(5):
        ctx.release()
        assert torch.equal(F.quantized_paged_attention(*args, 0.1, ctx=ctx), first)


def test_plain_kernel_agrees(F, ctx):
    """The switch decode_plain sends every call to the kernel without a split; both are within the bound."""
    args = attention_inputs(LENS + [700], D=128, n=2)
    check_attention(F, ctx, args)
    F.set_option("decode_plain", 1)
    try:
        check_attention(F, ctx, args)
    finally:
        F.set_option("decode_plain", 0)


def test_attention_on_another_stream_and_in_a_graph(F):
    """A captured call reads lengths, table and cache as they are when it is replayed."""
    from diopi_b200.runtime import Context
    st = torch.cuda.Stream()
    args = attention_inputs([300, 40, 1000], D=128)
    q, kc, vc, ks, vs, table, lens = [t.cuda() for t in args]
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        ctx = Context(st)
        out = torch.empty_like(q)
        F.quantized_paged_attention(q, kc, vc, ks, vs, table, lens, 0.1, ctx=ctx, out=out)
        st.synchronize()
        ctx.release()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            F.quantized_paged_attention(q, kc, vc, ks, vs, table, lens, 0.1, ctx=ctx, out=out)
        for new in ([300, 40, 1000], [1, 0, 999], [17, 40, 16]):
            lens.copy_(torch.tensor(new))
            q.neg_()
            out.fill_(5.0)
            graph.replay()
            st.synchronize()
            a = (q.cpu(), *args[1:6], torch.tensor(new))
            want, sums = O.quantized_paged_attention(*a, 0.1)
            assert bool(((out.cpu().double() - want).abs() <= bound_of(want, sums, 1000, 128, q.dtype)).all())


def test_which_kernel_takes_a_call(F, ctx, capfd):
    """The split kernel wherever the width is a multiple of 16 up to 256 and the cache's rows are aligned."""
    F.set_option("log", 1)
    try:
        for kw, kernel in ((dict(), "split"), (dict(D=16), "split"), (dict(D=256, dt="fp32"), "split"), (dict(bs=48), "split"), (dict(bs=24), "split"), (dict(bs=1), "split"), (dict(D=40), "plain"),
                           (dict(D=272), "plain"), (dict(n=3, group=50), "split")):
            args = [t.cuda() for t in attention_inputs([70, 3], **kw)]
            capfd.readouterr()
            F.quantized_paged_attention(*args, 0.1, ctx=ctx)
            assert f"({kernel} kernel)" in capfd.readouterr().err, kw
    finally:
        F.set_option("log", 0)


@pytest.mark.parametrize("Hkv,group,D", [(1, 300, 64), (2, 129, 128), (1, 64, 256)])
def test_attention_of_wide_groups(F, ctx, Hkv, group, D):
    """More query rows on a K/V head than the warps of a CTA take."""
    check_attention(F, ctx, attention_inputs([300, 0, 17], Hkv=Hkv, group=group, D=D, dt="fp16"))


def test_attention_of_thousands_of_requests(F, ctx):
    g = torch.Generator().manual_seed(2)
    lens = torch.randint(0, 20, (4100,), generator=g).tolist()   # more than the split kernel keeps the lengths of
    check_attention(F, ctx, attention_inputs(lens, D=64, Hkv=1, group=2, dt="fp16"))
    check_attention(F, ctx, attention_inputs(lens[:4096], D=64, Hkv=1, group=2, dt="fp16"))


def test_the_next_operation_finds_the_output(F, ctx):
    """Requests that need no merge: the second kernel of a call must not end the call before the first one has."""
    args = [t.cuda() for t in attention_inputs([60] * 40, D=128, Hkv=8, group=2)]
    want = F.quantized_paged_attention(*args, 0.1, ctx=ctx)
    out = torch.empty_like(want)
    for _ in range(200):
        ctx.release()
        out.fill_(7.0)
        F.quantized_paged_attention(*args, 0.1, ctx=ctx, out=out)
        assert torch.equal(out.clone(), want)


def test_calls_on_two_streams_at_once(F):
    """Each stream has a context, hence scratch, of its own."""
    from diopi_b200.runtime import Context
    streams = [torch.cuda.Stream() for _ in range(2)]
    args = [[t.cuda() for t in attention_inputs([2000, 31, 700], seed=s)] for s in range(2)]
    wants = [F.quantized_paged_attention(*a, 0.1, ctx=Context()) for a in args]
    ctxs = [Context(st) for st in streams]
    outs = [[torch.empty_like(w) for _ in range(30)] for w in wants]
    torch.cuda.synchronize()
    for i in range(30):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                F.quantized_paged_attention(*args[s], 0.1, ctx=ctxs[s], out=outs[s][i])
                ctxs[s].release()
    torch.cuda.synchronize()
    for s in range(2):
        assert all(torch.equal(o, wants[s]) for o in outs[s])


def test_a_captured_step_of_all_three(F):
    """Tables, store and attention in one graph, replayed with other lengths: a decode loop without the host."""
    from diopi_b200.runtime import Context
    g = torch.Generator().manual_seed(9)
    B, H, Hkv, D, bs, cols = 4, 8, 2, 64, 16, 6
    i32 = dict(dtype=torch.int32, device="cuda")
    blocks = B * cols
    start_lens = torch.tensor([5, 0, 16, 40])
    o_table = paged(B, start_lens.tolist(), bs, cols, blocks, g)
    o_table = torch.where(o_table > blocks, torch.full_like(o_table, -1), o_table)
    used = set(o_table[o_table >= 0].tolist())
    free = torch.tensor([b for b in range(blocks) if b not in used])
    table, d_free, at, nxt = o_table.to(**i32), free.to(**i32), torch.zeros(1, **i32), torch.zeros(1, **i32)
    cached, new, seq, starts, slots = start_lens.to(**i32), torch.ones(B, **i32), torch.zeros(B, **i32), torch.zeros(B + 1, **i32), torch.zeros(B, **i32)
    o_cache = [random_codes((blocks, bs, Hkv, D), True, g) for _ in range(2)]
    o_scale = [torch.full((blocks, Hkv), 0.125) for _ in range(2)]
    cache, scale = [c.cuda() for c in o_cache], [s.cuda() for s in o_scale]
    k, v, q = [torch.zeros(B, h, D, dtype=torch.float16, device="cuda") for h in (Hkv, Hkv, H)]
    out = torch.zeros_like(q)
    st = torch.cuda.Stream()
    ctx = Context(st)

    def step():
        F.build_block_table(table, cached, new, d_free, at, bs, slot_map=slots, new_start=starts, seq_lens=seq, free_next=nxt, ctx=ctx)
        F.quantized_copy_kv(k, v, table, cached, starts, *cache, *scale, ctx=ctx)
        F.quantized_paged_attention(q, *cache, *scale, table, seq, 0.125, out=out, ctx=ctx)

    keep = [t.clone() for t in (table, *cache, *scale)]
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        step()                       # sizes the scratch outside the capture
        st.synchronize()
        ctx.release()
        for t, was in zip((table, *cache, *scale), keep):
            t.copy_(was)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            step()
            cached.copy_(seq)
            at.copy_(nxt)
        o_cached, o_at = start_lens, 0
        for _ in range(20):
            hk, hv, hq = [torch.randn(t.shape, generator=g).half() for t in (k, v, q)]
            k.copy_(hk), v.copy_(hv), q.copy_(hq)
            graph.replay()
            st.synchronize()
            o_table, _, o_starts, o_lens, o_at, _ = O.build_block_table(o_table, o_cached, torch.ones(B, dtype=torch.int64), free, o_at, bs, B)
            for m, x in enumerate((hk, hv)):
                o_cache[m], o_scale[m] = O.quantized_copy(x, o_table, o_cached, o_starts, o_cache[m], o_scale[m])
                assert torch.equal(cache[m].cpu(), o_cache[m]) and torch.equal(scale[m].cpu(), o_scale[m])
            want, sums = O.quantized_paged_attention(hq[:, None], *o_cache, *o_scale, o_table, o_lens, 0.125)
            assert bool(((out.cpu().double()[:, None] - want).abs() <= bound_of(want, sums, 96, D, torch.float16)).all())
            o_cached = o_lens
    assert take_status(F) is None


# ---------------------------------------------------------------------------------------------------
# the three together
# ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("e4m3", [True, False])
def test_a_prefill_and_decode_steps(F, ctx, e4m3):
    """Prompts enter, then tokens one by one, all lengths on the device. Beside the 8-bit cache a 16-bit pool is fed by the same
    slots and read through the token table and the block table by the operators that take those."""
    g = torch.Generator().manual_seed(21)
    B, H, Hkv, D, bs, cols, N = 5, 4, 4, 64, 16, 8, 128
    i32 = dict(dtype=torch.int32, device="cuda")
    prompts = [37, 1, 0, 64, 20]
    blocks = B * cols
    table, free = torch.full((B, cols), -1, **i32), torch.randperm(blocks, generator=g).to(**i32)
    head = [torch.zeros(1, **i32), torch.zeros(1, **i32)]
    cached, seq, starts = torch.zeros(B, **i32), torch.zeros(B, **i32), torch.zeros(B + 1, **i32)
    cache = [torch.zeros(blocks, bs, Hkv, D, dtype=torch.float8_e4m3fn if e4m3 else torch.int8, device="cuda") for _ in range(2)]
    scale = [torch.zeros(blocks, Hkv, device="cuda") for _ in range(2)]
    pool = [torch.zeros(blocks * bs, Hkv, D, dtype=torch.float16, device="cuda") for _ in range(2)]
    wide = torch.zeros(B, N, **i32)
    o_table, o_cached, o_at = torch.full((B, cols), -1), torch.zeros(B, dtype=torch.int64), 0
    o_cache = [torch.zeros(blocks, bs, Hkv, D, dtype=torch.uint8 if e4m3 else torch.int8) for _ in range(2)]
    o_scale = [torch.zeros(blocks, Hkv) for _ in range(2)]
    for step in range(12):
        new = torch.tensor(prompts if step == 0 else [1, 1, 1, 1, 0 if step % 3 else 1])
        T = int(new.sum())
        k, v = [(torch.randn(T, Hkv, D, generator=g) * (1 + step / 3)).half() for _ in range(2)]
        q = torch.randn(B, H, D, generator=g).half()
        slots = torch.zeros(T, **i32)
        F.build_block_table(table, cached, new.to(**i32), free, head[step % 2], bs, slot_map=slots, new_start=starts, seq_lens=seq, free_next=head[1 - step % 2],
                            token_table=wide, ctx=ctx)
        F.quantized_copy_kv(k.cuda(), v.cuda(), table, cached, starts, *cache, *scale, ctx=ctx)
        F.destindex_copy_kv(k.cuda(), slots, pool[0], ctx=ctx)
        F.destindex_copy_kv(v.cuda(), slots, pool[1], ctx=ctx)
        got = F.quantized_paged_attention(q.cuda(), *cache, *scale, table, seq, 1 / 8, ctx=ctx)
        o16 = torch.zeros(B, H, D, dtype=torch.float16, device="cuda")
        F.token_decode_attention(q.cuda(), *pool, o16, wide, starts[:B], seq, N, ctx=ctx)
        lens = (cached.cpu().long() + new)
        p16 = F.paged_attention(q.cuda().view(B, H * D), pool[0].view(-1, Hkv * D), pool[1].view(-1, Hkv * D), None, lens.tolist(), H, Hkv, D, table, bs, ctx=ctx)
        # the oracle's course of the same steps
        o_table, o_slots, o_starts, o_lens, o_at, _ = O.build_block_table(o_table, o_cached, new, free.cpu(), o_at, bs, T)
        assert torch.equal(table.cpu().long(), o_table) and torch.equal(slots.cpu().long(), o_slots) and torch.equal(seq.cpu().long(), o_lens)
        for m, x in enumerate((k, v)):
            o_cache[m], o_scale[m] = O.quantized_copy(x, o_table, o_cached, o_starts, o_cache[m], o_scale[m])
            bits = cache[m].view(torch.uint8) if e4m3 else cache[m]
            assert torch.equal(bits.cpu(), o_cache[m]) and torch.equal(scale[m].cpu(), o_scale[m])
        want, sums = O.quantized_paged_attention(q[:, None], *o_cache, *o_scale, o_table, o_lens, 1 / 8)
        assert bool(((got.cpu().double()[:, None] - want).abs() <= bound_of(want, sums, 128, D, torch.float16)).all())
        # the 16-bit operators through the same tables: their two forms agree to fp16 of values below 8 standard deviations
        assert torch.allclose(o16.view(B, H * D), p16, rtol=1e-2, atol=1e-2 * (1 + step / 3))
        cached, seq = seq.clone(), seq
        o_cached = o_lens
        ctx.release()
    assert take_status(F) is None
