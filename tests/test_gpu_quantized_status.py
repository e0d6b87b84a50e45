"""No kernel of the 8-bit cache operators reports anything (a block outside the cache, a wait given up) on inputs that are in order:
the other tests' calls again, with the status looked at after each."""
import pytest

import test_gpu_quantized_cache as Q
from test_gpu_quantized_cache import F, ctx  # noqa: F401

pytestmark = pytest.mark.gpu

CALLS = [
    *[(Q.test_attention_widths_and_types, (D, dt, e4m3)) for D, dt, e4m3 in ((64, "bf16", True), (128, "fp16", False), (256, "fp32", True), (80, "bf16", False), (40, "fp16", True))],
    *[(Q.test_attention_head_layouts, hg) for hg in ((1, 1), (1, 17), (1, 71), (5, 3), (7, 1), (8, 4), (1, 130), (2, 33))],
    *[(Q.test_attention_block_sizes, (bs, e4m3)) for bs, e4m3 in ((1, True), (17, False), (48, True), (272, False))],
    *[(Q.test_attention_ignores_the_next_block, (bs,)) for bs in (8, 24, 40)],
    *[(Q.test_attention_of_several_new_tokens, nd) for nd in ((2, 64, 2, 4), (5, 128, 1, 1), (16, 96, 3, 2))],
    *[(Q.test_attention_splits, bl) for bl in ((1, 5000), (3, 2100), (300, 20), (700, 3))],
    (Q.test_attention_large_logits_and_scales, ()),
    (Q.test_attention_hands_nan_on, ()),
    (Q.test_attention_keeps_nan_from_the_tokens_before_it, (128, 5, 4)),
    (Q.test_attention_strides, (True,)),
    (Q.test_attention_clamps_lengths_to_the_table, ()),
    (Q.test_attention_into_its_own_query, ()),
    (Q.test_attention_empty_calls, ()),
    (Q.test_attention_offsets_beyond_32_bits, ()),
    (Q.test_attention_gives_the_same_bits_again, ("bf16",)),
    (Q.test_plain_kernel_agrees, ()),
    *[(Q.test_attention_of_wide_groups, hd) for hd in ((1, 300, 64), (2, 129, 128), (1, 64, 256))],
    (Q.test_attention_of_thousands_of_requests, ()),
    (Q.test_the_next_operation_finds_the_output, ()),
    *[(Q.test_copy_block_sizes, (bs, e4m3)) for bs, e4m3 in ((1, True), (24, False), (64, True), (130, False), (256, True))],
    *[(Q.test_copy_of_a_decode_step, (B,)) for B in (1, 256, 700)],
    (Q.test_copy_ties_and_borders, ()),
    (Q.test_copy_magnitudes, (True, 3e4)),
    (Q.test_copy_zeros_infinities_and_nan, ("bf16", True, 64)),
    (Q.test_copy_strides, (False,)),
    (Q.test_copy_token_by_token_stays_near, (True,)),
    (Q.test_tables_of_an_empty_batch, ()),
]


@pytest.mark.parametrize("call,args", CALLS, ids=[f"{c.__name__[5:]}-{'-'.join(map(str, a))}" for c, a in CALLS])
def test_no_status(F, ctx, call, args):  # noqa: F811
    assert Q.take_status(F) is None
    given = (F, ctx) if "ctx" in call.__code__.co_varnames[:call.__code__.co_argcount] else (F,)
    names = call.__code__.co_varnames[len(given):call.__code__.co_argcount]
    assert len(names) == len(args)
    call(*given, *args)
    assert Q.take_status(F) is None
