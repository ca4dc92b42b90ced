"""The block-scaled KV cache at its edges, on a B200."""

import math

import pytest
import torch

from llmquant_b200 import native
from llmquant_b200.quantizers import BlockKVCache, BlockKVStore
from test_gpu_block_kv import EXTRA, attend64, check_attend, close_to, filled, rand

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------- half a unit
def leave_scales(dim, tokens, group, dtype, word):
    """A call of the same kernel that leaves `word` where it stages scales, in every CTA that an SM holds: one
    unit to a CTA, each the whole of its (sequence, head), so that no join runs over it."""
    heads = 8
    batch = 16 * torch.cuda.get_device_properties(0).multi_processor_count // heads
    store = BlockKVStore.allocate(batch, heads, dim, 32, 32, dtype)
    for scales in (store.k_scales, store.v_scales):
        scales.view(torch.int32).fill_(word)
    store.attend(rand((batch, tokens, heads * group, dim), 7, dtype).cuda(), 32 - tokens)


@pytest.mark.parametrize("word", [-2 ** 31, -2 ** 31 + 1, -2 ** 31 + 0x7fffff, 0, 0x7f800000, 0x7fc00000, -1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,tokens", [(64, 1), (64, 3), (128, 1), (128, 3)])  # 4 and 12 rows
def test_an_odd_number_of_short_blocks_whatever_shared_memory_held(dim, tokens, dtype, word):
    """Blocks of 16 are staged two to a unit: with three of them the last unit's second half is not there."""
    store, model = filled(8, 2, dim, 16, dtype, [48] * 8, 201)
    q = rand((8, tokens, 8, dim), 204, dtype, 2.0).cuda()
    leave_scales(dim, tokens, 4, dtype, word)
    check_attend(store, model, q, [48 - tokens] * 8, [tokens] * 8)
    # and behind a whole unit, with rows of the incomplete block after it
    store, model = filled(8, 2, dim, 16, dtype, [16 * 5 + 3] * 8, 205)
    leave_scales(dim, tokens, 4, dtype, word)
    check_attend(store, model, q, [83 - tokens] * 8, [tokens] * 8)


# ------------------------------------------------------------------------------- behind transformers' Cache
def test_stand_ins_of_a_fused_read_are_no_keys_and_values():
    """An attention function other than the library's must fail on them instead of computing with them."""
    cache = BlockKVCache(32, fused_read=True)
    rows = rand((2, 3, 40, 64), 211).cuda()
    k, v = cache.update(rows, rows, 0)
    assert k.shape == v.shape == (2, 3, 40, 64) and k.lq_layer is v.lq_layer is cache.layers[0]
    assert k.dtype == v.dtype == torch.int8
    q = rand((2, 3, 1, 64), 212).cuda()
    with pytest.raises(RuntimeError):
        torch.nn.functional.scaled_dot_product_attention(q, k, v)
    with pytest.raises(RuntimeError):
        q @ k.transpose(2, 3)


# ------------------------------------------------------------------------------- values that are not finite
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,tokens,group", [(64, 4, 2), (128, 6, 4), (64, 7, 9), (128, 70, 2)])  # 8, 24, 63, 140 rows
def test_a_value_that_is_not_finite_reaches_the_rows_that_see_it(dim, tokens, group, dtype, where, bad):
    """One value of one row: NaN for the rows that see a position of its block, or its own position while the
    block is incomplete; the definition's values, without it, for the rows before."""
    block, start = 32, 40
    total = start + tokens
    held = total - total % block
    store, model = filled(1, 2, dim, block, dtype, [total], 221)
    q = rand((1, tokens, 2 * group, dim), 224, dtype, 2.0).cuda()
    want = attend64(q[0], *(model.values(rows[0]) for rows in (model.k, model.v)), start, dim ** -0.5)
    largest = model.v[0].double().abs().max()
    for at in sorted({start, start + 1, held - 1, held, total - 2, total - 1} & set(range(start, total))):
        k, v = model.k[0].clone(), model.v[0].clone()
        (k if where == "k" else v)[0, at, dim - 3] = bad
        store.append(k[None].cuda(), v[None].cuda(), 0)
        got = store.attend(q, start)[0]
        first = max(0, (at if at >= held else at - at % block) - start)  # the first row that sees it
        assert got[first:, :group].isnan().all(), at
        if first:
            close_to(got[:first, :group], want[:first, :group], dtype, EXTRA, largest)
        close_to(got[:, group:], want[:, group:], dtype, EXTRA, largest)  # the other head
    assert native.library().lq_block_kv_device_error() == 0


# ------------------------------------------------------------------------------- long contexts
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,group", [(1, 2), (6, 2), (70, 2)])  # each of the kernels: 2, 12 and 140 rows
def test_many_small_weights_beside_a_large_one(tokens, group, dtype):
    """One token with nearly all of the weight and 131071 with 1.25 * 2^-24 of it each: together they count 1 %. So
    many sequences share the pages that a warp (CTA) has a context to itself."""
    heads, dim, block, length = 8, 64, 128, 131072
    batch = 16 * torch.cuda.get_device_properties(0).multi_processor_count // heads
    one = BlockKVStore.allocate(1, heads, dim, length, block, dtype)
    one.k_scales.fill_(1.0)
    one.v_scales.fill_(1.0 / 127.0)
    one.v_pages.fill_(127)
    one.v_pages[0, :, 0] = 0
    one.k_pages[0, :, 0, 0] = 1
    rings = [r.expand(batch, *r.shape[1:]).contiguous() for r in (one.k_ring, one.v_ring)]
    store = BlockKVStore(one.k_pages, one.v_pages, one.k_scales, one.v_scales, *rings, one.table.expand(batch, -1).contiguous())
    q = torch.zeros(batch, tokens, heads * group, dim, dtype=dtype, device="cuda")
    q[..., 0] = 16.0
    got = store.attend(q, length - tokens, scaling=math.log(2.0 ** 24 / 1.25) / 16)
    rest = torch.arange(length - tokens, length, dtype=torch.float64) * 1.25 * 2.0 ** -24
    want = (rest / (1 + rest))[None, :, None, None].expand(got.shape)
    # a weight is held as fp16 up to 2^7 above the point that it is counted from, so what lies below 2^-21 of the
    # largest is off by at most 2^-32 of it: 2^-15 in all. Exponents in fp32: 24 * 2^-24 of each weight.
    close_to(got, want, dtype, 2.0 ** -15 + 2.0 ** -17, torch.tensor(1.0))
    assert native.library().lq_block_kv_device_error() == 0
