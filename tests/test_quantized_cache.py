"""The block-paged cache in 8 bits without a GPU: the oracle against what it must satisfy, and every refusal of the three
entry points before any CUDA work (the tensors only pretend to live on a device)."""
import math

import pytest
import torch

from diopi_b200.runtime import DTYPE_NOT_SUPPORTED, ERROR_OCCURRED, DiopiError
from oracle import quantized_cache as O


@pytest.fixture(scope="module")
def F(built_libs):
    from diopi_b200 import functions
    return functions


def fails(code, fn, *args, match=None, **kw):
    with pytest.raises(DiopiError, match=match) as e:
        fn(*args, as_device=True, **kw)
    assert e.value.code == code, e.value


# ---- the oracle ----------------------------------------------------------------------------------
def test_e4m3_codes_agree_with_torch():
    codes = torch.arange(256, dtype=torch.int16).to(torch.uint8)
    want = codes.view(torch.float8_e4m3fn).double()
    assert torch.equal(torch.nan_to_num(O.decode(codes), nan=999.0), torch.nan_to_num(want, nan=999.0))
    x = torch.cat([torch.randn(20000, generator=torch.Generator().manual_seed(3)) * s for s in (1e-3, 1.0, 100.0)]).clamp(-448, 448)
    mid = (O.e4m3_values()[:126] + O.e4m3_values()[1:127]) / 2   # every tie
    x = torch.cat([x.double(), mid, -mid, O.e4m3_values()[:127]])
    assert torch.equal(O.encode(x, True), x.float().to(torch.float8_e4m3fn).view(torch.uint8))


@pytest.mark.parametrize("e4m3", [False, True])
def test_store_is_within_half_a_step(e4m3):
    g = torch.Generator().manual_seed(11)
    x = torch.randn(16, 2, 32, generator=g, dtype=torch.float32)
    cache = torch.zeros(1, 16, 2, 32, dtype=torch.uint8 if e4m3 else torch.int8)
    c, s = O.quantized_copy(x, torch.zeros(1, 1, dtype=torch.int64), torch.tensor([0]), torch.tensor([0, 16]), cache, torch.zeros(1, 2))
    got = O.decode(c[0]) * s[0].double()[None, :, None]
    # int8: half a step of s; e4m3: half a step of a value, 2^-4 of it, or of the smallest step where that is larger
    bound = s[0].double()[None, :, None] * 0.5 if not e4m3 else torch.maximum(x.double().abs() * 2.0 ** -4, s[0].double()[None, :, None] * 2.0 ** -10)
    assert bool(((got - x.double()).abs() <= bound * (1 + 1e-6)).all())


def test_scales():
    assert O.fresh_scale(0.0, True) == 0 and O.fresh_scale(0.0, False) == 0
    assert O.fresh_scale(448.0, True) == 1 and O.fresh_scale(449.0, True) == 2 and O.fresh_scale(224.0, True) == 0.5
    assert O.fresh_scale(1e-45, False) == 2.0 ** -126 == O.fresh_scale(1e-45, True)


# ---- refusals -------------------------------------------------------------------------------------
def table_args(B=2, cols=4, T=6, N=None, dt=torch.int32):
    z = lambda *s: torch.zeros(*s, dtype=dt)  # noqa: E731
    a = dict(block_table=z(B, cols), cached_lens=z(B), new_lens=z(B), free_blocks=z(9), free_start=z(1), block_size=4)
    kw = dict(slot_map=z(T), new_start=z(B + 1), seq_lens=z(B), free_next=z(1), token_table=None if N is None else z(B, N))
    return a, kw


def test_block_table_refusals(F):
    def bad(code, match, pos=(), **over):
        a, kw = table_args(N=8)
        for k, v in over.items():
            (a if k in a else kw)[k] = v(a, kw) if callable(v) else v
        fails(code, F.build_block_table, *a.values(), match=match, **kw)

    i32 = dict(dtype=torch.int32)
    bad(ERROR_OCCURRED, "block_size must be positive", block_size=0)
    bad(ERROR_OCCURRED, "block_size must be positive", block_size=-16)
    bad(ERROR_OCCURRED, "batch \\+ 1", new_start=torch.zeros(2, **i32))
    bad(ERROR_OCCURRED, "batch = 2", seq_lens=torch.zeros(3, **i32))
    bad(ERROR_OCCURRED, "batch = 2", cached_lens=torch.zeros(1, **i32))
    bad(ERROR_OCCURRED, "one entry", free_next=torch.zeros(2, **i32))
    bad(ERROR_OCCURRED, "one entry", free_start=torch.zeros(0, **i32))
    bad(ERROR_OCCURRED, "rows for a batch", token_table=torch.zeros(3, 8, **i32))
    bad(ERROR_OCCURRED, "2 dim", block_table=torch.zeros(8, **i32))
    bad(DTYPE_NOT_SUPPORTED, "int32 or int64", slot_map=torch.zeros(6))
    bad(DTYPE_NOT_SUPPORTED, "int32 or int64", free_blocks=torch.zeros(6, dtype=torch.int16))
    # what is written must not be what is read, nor written twice
    bad(ERROR_OCCURRED, "share memory", seq_lens=lambda a, kw: a["cached_lens"])
    bad(ERROR_OCCURRED, "share memory", free_next=lambda a, kw: a["free_start"])
    bad(ERROR_OCCURRED, "share memory", seq_lens=lambda a, kw: kw["new_start"][:2])
    bad(ERROR_OCCURRED, "share memory", slot_map=lambda a, kw: a["free_blocks"][3:])
    bad(ERROR_OCCURRED, "expanded", block_table=torch.zeros(1, 4, **i32).expand(2, 4))
    bad(ERROR_OCCURRED, "2\\^31", block_table=torch.zeros(2, 4, **i32), block_size=(1 << 29))
    bad(ERROR_OCCURRED, "null handle", slot_map=None)


def cache_args(B=2, T=5, H=4, D=32, bs=8, blocks=6, dt=torch.float16, code=torch.int8):
    return dict(k=torch.zeros(T, H, D, dtype=dt), v=torch.zeros(T, H, D, dtype=dt), block_table=torch.zeros(B, 3, dtype=torch.int32),
                cached_lens=torch.zeros(B, dtype=torch.int32), new_start=torch.zeros(B + 1, dtype=torch.int32), k_cache=torch.zeros(blocks, bs, H, D, dtype=code),
                v_cache=torch.zeros(blocks, bs, H, D, dtype=code), k_scale=torch.zeros(blocks, H), v_scale=torch.zeros(blocks, H))


def test_copy_refusals(F):
    def bad(code, match, **over):
        a = cache_args()
        for k, v in over.items():
            a[k] = v(a) if callable(v) else v
        fails(code, F.quantized_copy_kv, *a.values(), match=match)

    bad(DTYPE_NOT_SUPPORTED, "float64", k=torch.zeros(5, 4, 32, dtype=torch.float64), v=torch.zeros(5, 4, 32, dtype=torch.float64))
    bad(ERROR_OCCURRED, "share a dtype", v=torch.zeros(5, 4, 32))
    bad(ERROR_OCCURRED, "must be \\[tokens, 4, 32\\]", k=torch.zeros(5, 4, 16, dtype=torch.float16))
    bad(ERROR_OCCURRED, "must be \\[tokens, 4, 32\\]", v=torch.zeros(4, 4, 32, dtype=torch.float16))
    bad(DTYPE_NOT_SUPPORTED, "int8, or uint8", k_cache=torch.zeros(6, 8, 4, 32, dtype=torch.float16))
    bad(ERROR_OCCURRED, "share a dtype", v_cache=torch.zeros(6, 8, 4, 32, dtype=torch.uint8))
    bad(ERROR_OCCURRED, "differ in dim 0", v_cache=torch.zeros(7, 8, 4, 32, dtype=torch.int8), v_scale=torch.zeros(7, 4))
    bad(ERROR_OCCURRED, "'k_scale' must be", k_scale=torch.zeros(6, 5))
    bad(DTYPE_NOT_SUPPORTED, "float32", v_scale=torch.zeros(6, 4, dtype=torch.float16))
    bad(ERROR_OCCURRED, "same memory", v_cache=lambda a: a["k_cache"])
    bad(ERROR_OCCURRED, "same memory", v_scale=lambda a: a["k_scale"])
    bad(ERROR_OCCURRED, "expanded", k_scale=torch.zeros(6, 1).expand(6, 4))
    bad(ERROR_OCCURRED, "batch = 2", cached_lens=torch.zeros(3, dtype=torch.int32))
    bad(ERROR_OCCURRED, "batch \\+ 1", new_start=torch.zeros(2, dtype=torch.int32))
    bad(DTYPE_NOT_SUPPORTED, "int32 or int64", block_table=torch.zeros(2, 3))
    bad(ERROR_OCCURRED, "beyond the supported maximum", k_cache=torch.zeros(6, 8, 4, 513, dtype=torch.int8), v_cache=torch.zeros(6, 8, 4, 513, dtype=torch.int8))
    bad(ERROR_OCCURRED, "null handle", v=None)


def test_attention_refusals(F):
    c = cache_args()
    good = dict(q=torch.zeros(2, 8, 32, dtype=torch.float16), k_cache=c["k_cache"], v_cache=c["v_cache"], k_scale=c["k_scale"], v_scale=c["v_scale"],
                block_table=c["block_table"], seq_lens=c["cached_lens"], softmax_scale=0.2)

    def bad(code, match, out=None, **over):
        a = {**good, **over}
        fails(code, F.quantized_paged_attention, *a.values(), match=match, out=out)

    bad(ERROR_OCCURRED, "multiple of the cache's 4", q=torch.zeros(2, 6, 32, dtype=torch.float16))
    bad(ERROR_OCCURRED, "head_dim 16", q=torch.zeros(2, 8, 16, dtype=torch.float16))
    bad(ERROR_OCCURRED, "batch = 3", q=torch.zeros(3, 8, 32, dtype=torch.float16))
    bad(ERROR_OCCURRED, "\\[batch, heads, head_dim\\]", q=torch.zeros(8, 32, dtype=torch.float16))
    bad(DTYPE_NOT_SUPPORTED, "float64", q=torch.zeros(2, 8, 32, dtype=torch.float64))
    bad(ERROR_OCCURRED, "share a dtype", out=torch.zeros(2, 8, 32))
    bad(ERROR_OCCURRED, "differ in dim 1", out=torch.zeros(2, 4, 32, dtype=torch.float16))
    bad(ERROR_OCCURRED, "last dim", q=torch.zeros(2, 8, 64, dtype=torch.float16)[:, :, ::2])
    bad(ERROR_OCCURRED, "expanded", out=torch.zeros(1, 8, 32, dtype=torch.float16).expand(2, 8, 32))
    buf = torch.zeros(2 * 8 * 32 + 32, dtype=torch.float16)
    bad(ERROR_OCCURRED, "not overlap", q=buf[:512].view(2, 8, 32), out=buf[32:].view(2, 8, 32))
    for s in (0.0, -1.0, math.nan, math.inf):
        bad(ERROR_OCCURRED, "softmax_scale", softmax_scale=s)
    bad(DTYPE_NOT_SUPPORTED, "int32 or int64", seq_lens=torch.zeros(2))
    bad(ERROR_OCCURRED, "65535", q=torch.zeros(2, 8192, 8, 32, dtype=torch.float16))


def test_host_tensors_are_refused(F):
    c = cache_args()
    with pytest.raises(DiopiError, match="host memory"):
        F.quantized_copy_kv(*c.values(), as_device=False)


# ---- the call from Python ---------------------------------------------------------------------------
class ElsewhereTensor:
    """What a call looks at of a tensor, on the second device."""
    dtype, shape = torch.int32, (1,)

    def stride(self):
        return (1,)

    def data_ptr(self):
        return 4096

    def get_device(self):
        return 1


def test_tensors_of_another_device_are_refused(F):
    a, kw = table_args()
    with pytest.raises(ValueError, match="cuda:1"):
        F.build_block_table(ElsewhereTensor(), *list(a.values())[1:], **kw)


def test_what_a_call_takes(F, built_libs):
    """Handles made beforehand, None where a tensor may be missing, no other type; a dtype without a counterpart is an error."""
    from diopi_b200.runtime import Tensor
    c = cache_args()
    c["k_cache"] = Tensor(c["k_cache"], as_device=True)
    c["v_scale"] = Tensor(torch.zeros(6, 5), as_device=True)
    fails(ERROR_OCCURRED, F.quantized_copy_kv, *c.values(), match="'v_scale' must be")
    with pytest.raises(TypeError, match="complex"):
        F.quantized_copy_kv(*{**cache_args(), "k": torch.zeros(5, 4, 32, dtype=torch.complex64)}.values(), as_device=True)
    with pytest.raises(AttributeError):
        F.quantized_copy_kv(*{**cache_args(), "k": [1, 2]}.values(), as_device=True)
    fails(ERROR_OCCURRED, F.quantized_copy_kv, *{**cache_args(), "k": torch.zeros([1] * 9)}.values(), match="at most 8")


# ---- views that interleave ---------------------------------------------------------------------------
def test_views_that_alternate_do_not_share_memory(F):
    """Slices of one fused tensor whose byte ranges overlap but whose elements do not are no overlap: what is refused in these calls
    is a later argument. Slices that do share elements are refused as such."""
    c = cache_args()
    fused = torch.zeros(2, 3, 8, 32, dtype=torch.float16)
    cols = torch.zeros(2, 8, 64, dtype=torch.float16)

    def attend(q, out, match):
        fails(ERROR_OCCURRED, F.quantized_paged_attention, q, c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"], c["block_table"], c["cached_lens"], -1.0,
              match=match, out=out)

    attend(fused[:, 0], fused[:, 2], "softmax_scale")
    attend(fused[:, 1], fused[:, 0], "softmax_scale")
    attend(cols[..., :32], cols[..., 32:], "softmax_scale")
    attend(cols[..., :32], cols[..., 16:48], "not overlap")
    attend(fused[:, 0], fused.view(2, 24, 32)[:, 4:12], "not overlap")
    attend(fused.view(6, 8, 32)[:2], fused.view(6, 8, 32)[1:3], "not overlap")
    # the same with the head dim's rows apart: heads in front of the batch
    heads = torch.zeros(8, 2, 2, 32, dtype=torch.float16)
    attend(heads[:, 0].transpose(0, 1), heads[:, 1].transpose(0, 1), "softmax_scale")

    i32 = dict(dtype=torch.int32)
    both, five = torch.zeros(2, 2, **i32), torch.zeros(3, 5, **i32)

    def tables(match, **over):
        a, kw = table_args()
        a["block_size"] = 1 << 29      # refused after the views have been looked at
        for k, v in over.items():
            (a if k in a else kw)[k] = v
        fails(ERROR_OCCURRED, F.build_block_table, *a.values(), match=match, **kw)

    tables("2\\^31", cached_lens=both[:, 0], seq_lens=both[:, 1])
    tables("2\\^31", new_start=five[:, 0], seq_lens=five[:2, 2], new_lens=five[:2, 4], slot_map=five[:, 1])
    tables("share memory", cached_lens=both[:, 0], seq_lens=both[:, 0])
    tables("share memory", new_start=five[:, 0], seq_lens=five[:2, 0])
    tables("share memory", slot_map=both.view(-1), seq_lens=both[:, 1])
