"""The block-scaled KV cache and the norm + rotation of queries and keys, on a B200, against plain
implementations in 64 bits that are written here from the definitions.

Tolerances. A result rounded once to its type is off by at most half a step, eps / 2 relative to
itself (bf16 2^-8, fp16 2^-11, fp32 2^-24); what the kernels do before that rounding is fp32, whose own error is stated beside each bound. Codes and scales are
exact: the same IEEE division and rounding as the definition, on values that are exact in fp32."""

import math

import pytest
import torch

from llmquant_b200 import native
from llmquant_b200.cuda import qk_norm_rope
from llmquant_b200.quantizers import BlockKVStore

pytestmark = pytest.mark.gpu

HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}


def rand(shape, seed, dtype=torch.bfloat16, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype)


def tables(length, rot):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    angle = torch.arange(length, dtype=torch.float64)[:, None] * inv
    return angle.cos().float().cuda(), angle.sin().float().cuda()


# ------------------------------------------------------------------------------- the definitions
def norm_rope64(x, weight, cos, sin, interleaved, eps):
    """x [..., heads, D], cos / sin [..., rot / 2], in 64 bits on the CPU."""
    x, cos, sin = x.double().cpu(), cos.double().cpu()[..., None, :], sin.double().cpu()[..., None, :]
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double().cpu()
    half = cos.shape[-1]
    i = torch.arange(half)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y = x.clone()
    y[..., first] = x[..., first] * cos - x[..., second] * sin
    y[..., second] = x[..., second] * cos + x[..., first] * sin
    return y


class Model:
    """The cache by its definition: per sequence and head, the list of all rows that came."""

    def __init__(self, batch, heads, dim, block, dtype):
        self.k = [torch.zeros(heads, 0, dim, dtype=dtype) for _ in range(batch)]
        self.v = [torch.zeros(heads, 0, dim, dtype=dtype) for _ in range(batch)]
        self.block = block

    def put(self, b, k, v, start):
        self.k[b] = torch.cat((self.k[b][:, :start], k.cpu()), 1)
        self.v[b] = torch.cat((self.v[b][:, :start], v.cpu()), 1)

    def codes(self, rows):
        """Codes and scales of the complete blocks, by fp32 arithmetic (IEEE, as the definition's)."""
        whole = rows.shape[1] // self.block
        x = rows[:, : whole * self.block].float().unflatten(1, (whole, self.block))
        amax = x.abs().amax((2, 3)) if whole else x.new_zeros(x.shape[:2])
        scale = torch.clamp(amax / torch.tensor(127.0), min=1e-8)
        return torch.clamp(torch.round(x / scale[:, :, None, None]), -128, 127), scale

    def values(self, rows):
        """64-bit values of one sequence's rows [H, L, D] as the cache stands for them."""
        codes, scale = self.codes(rows)
        bad = ~torch.isfinite(scale)
        held = codes.double() * scale.double()[:, :, None, None]
        held[bad] = math.nan
        return torch.cat((held.flatten(1, 2), rows[:, codes.shape[1] * self.block:].double()), 1)


def attend64(q, k, v, start, scaling):
    """q [n, Hq, D]; k, v [H, start + n, D], 64 bits."""
    n, hq, _ = q.shape
    group = hq // k.shape[0]
    out = torch.empty(q.shape, dtype=torch.float64)
    for h in range(hq):
        s = q[:, h].double().cpu() @ k[h // group].T * scaling
        s[torch.arange(k.shape[1])[None] > start + torch.arange(n)[:, None]] = -math.inf
        out[:, h] = torch.softmax(s, -1) @ v[h // group]
    return out


def close_to(got, want, dtype, extra, scale=None):
    """|got - want| within half a step of the result plus `extra` of the scale (default: the largest value)."""
    got = got.double().cpu()
    scale = want.abs().max() if scale is None else scale
    bound = HALF_STEP[dtype] * want.abs() + extra * scale + torch.finfo(dtype).smallest_normal
    worst = ((got - want).abs() - bound).max().item()
    assert worst <= 0, f"off by {worst} beyond the bound"


def pool_store(batch, heads, dim, blocks, block, dtype, seed=0, spare=3):
    """A store whose pages lie scattered in a pool with spare pages, everything filled with rubbish."""
    g = torch.Generator().manual_seed(seed)
    pages = batch * blocks + spare
    table = torch.randperm(pages, generator=g)[: batch * blocks].reshape(batch, blocks).int().cuda()
    codes = [torch.randint(-128, 128, (pages, heads, block, dim), generator=g, dtype=torch.int8).cuda() for _ in range(2)]
    scales = [torch.full((pages, heads), math.nan).cuda() for _ in range(2)]
    rings = [torch.full((batch, heads, 2 * block, dim), math.nan, dtype=dtype).cuda() for _ in range(2)]
    return BlockKVStore(*codes, *scales, *rings, table)


def check_state(store, model, counts, ring_from=0):
    """Codes, scales and rings against the definition, bit for bit. `ring_from`: where the ring begins after
    tokens were taken back."""
    block = store.block
    for b, total in enumerate(counts):
        for rows, pages, scales, ring in ((model.k[b], store.k_pages, store.k_scales, store.k_ring),
                                          (model.v[b], store.v_pages, store.v_scales, store.v_ring)):
            assert rows.shape[1] == total
            codes, scale = model.codes(rows)
            whole = codes.shape[1]
            at = store.table[b, :whole].long()
            assert torch.equal(pages[at].cpu().transpose(0, 1).float(), codes)
            assert torch.equal(scales[at].cpu().T, scale)
            first = max(ring_from, (whole - 1) * block)
            slots = torch.arange(first, total) % (2 * block)
            assert torch.equal(ring[b].cpu()[:, slots], rows[:, first:])


# ------------------------------------------------------------------------------- norm + rotation
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("batch,tokens,hq,hk,dim,rot,interleaved,norm", [
    (1, 1, 1, 1, 64, 64, False, True), (1, 1, 32, 8, 128, 128, False, True), (2, 37, 7, 1, 128, 64, False, True),
    (3, 5, 6, 2, 96, 96, False, False), (2, 9, 4, 4, 256, 256, True, True), (1, 3, 3, 1, 16, 16, True, True),
    (1, 130, 5, 5, 80, 32, True, False), (2, 700, 8, 2, 128, 128, False, True), (1, 4, 2, 1, 24, 16, False, True),
    (4, 901, 10, 6, 64, 48, False, True),
])
def test_norm_rope(dtype, batch, tokens, hq, hk, dim, rot, interleaved, norm):
    qkv = rand((batch, tokens, hq + 2 * hk, dim), 1, dtype, 2.0).cuda()
    q, k = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
    cos, sin = tables(1500, rot)
    pos = torch.arange(tokens)[None] + torch.arange(batch)[:, None] * 100
    wq, wk = (rand((dim,), s, dtype).cuda() if norm else None for s in (2, 3))
    got = qk_norm_rope(q, k, cos, sin, pos.cuda(), q_weight=wq, k_weight=wk, eps=1e-5, interleaved=interleaved)
    for x, w, y in ((q, wq, got[0]), (k, wk, got[1])):
        want = norm_rope64(x, w, cos[pos.cuda()], sin[pos.cuda()], interleaved, 1e-5)
        # fp32 inside: the sum of squares (<= 9 roundings), division, sqrt reciprocal (2 ulp), two
        # products, two of the rotation: under 16 roundings of 2^-24 relative to |y|, and the rotation's
        # terms are each at most the pair's length
        pair = want.abs().amax(-1, keepdim=True) * math.sqrt(2)
        close_to(y, want, dtype, 16 * 2.0 ** -24, pair)
        assert y.dtype == dtype


def test_norm_rope_in_place_strided_and_unaligned():
    base = rand((2, 11, 9, 128), 5).cuda()
    cos, sin = tables(64, 128)
    pos = torch.arange(11).cuda()[None]
    w = rand((128,), 6).cuda()
    want = qk_norm_rope(base[:, :, :4], base[:, :, 4:6], cos, sin, pos, w, w)
    # rows that begin on odd elements
    odd = torch.empty(2 * 11 * 9 * 131 + 1, dtype=base.dtype, device="cuda")[1:].view(2, 11, 9, 131)[..., 1:129]
    odd.copy_(base)
    got = qk_norm_rope(odd[:, :, :4], odd[:, :, 4:6], cos, sin, pos, w, w)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # heads before tokens, head_dim not contiguous, and in place
    perm = base.transpose(1, 2).contiguous().transpose(1, 2)
    got = qk_norm_rope(perm[:, :, :4], perm[:, :, 4:6], cos, sin, pos, w, w)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    flip = base.transpose(2, 3).contiguous().transpose(2, 3)
    got = qk_norm_rope(flip[:, :, :4], flip[:, :, 4:6], cos, sin, pos, w, w)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    rest = base[:, :, 6:].clone()
    q, k = base[:, :, :4], base[:, :, 4:6]
    got = qk_norm_rope(q, k, cos, sin, pos, w, w, out=(q, k))
    assert got[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(base[:, :, 6:], rest)


def test_norm_rope_special_values_and_positions():
    x = rand((1, 4, 2, 64), 7, torch.float32).cuda()
    x[0, 0] = 0.0             # a zero head: eps keeps it finite
    x[0, 1, 0, 5] = math.nan  # stays in its own head
    x[0, 2, 1, 3] = math.inf
    cos, sin = tables(10, 64)
    w = torch.ones(64, device="cuda")
    native.library().lq_block_kv_device_error()
    q, k = qk_norm_rope(x, x[:, :, :1], cos, sin, torch.tensor([[0, 9, 3, 10]]).cuda(), w, w)
    assert (q[0, 0] == 0).all() and q[0, 1, 0].isnan().all() and q[0, 1, 1].isfinite().all()
    assert not q[0, 2, 1].isfinite().all() and q[0, 2, 0].isfinite().all()
    assert q[0, 3].isnan().all() and k[0, 3].isnan().all()  # position 10 has no angles
    assert native.library().lq_block_kv_device_error() == 3
    assert native.library().lq_block_kv_device_error() == 0


# ------------------------------------------------------------------------------- append and read
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_append_any_cut_gives_the_same_cache(dtype, dim, block):
    """Three sequences of different lengths, the same tokens in different cuts: one cache."""
    batch, heads = 3, 2
    lengths = [5 * block + 3, 2 * block, block - 1]
    rows = [rand((batch, heads, max(lengths), dim), s, dtype, 3.0).cuda() for s in (11, 12)]
    cuts = [[max(lengths)], [1, block - 1, 2 * block + 1, 3, block, block], [block + 5, 2 * block, 7, 3 * block]]
    states = []
    for cut in cuts:
        store = pool_store(batch, heads, dim, 6, block, dtype)
        start = torch.zeros(batch, dtype=torch.int64)
        at = 0
        for n in cut:
            n = min(n, max(lengths) - at)
            if n <= 0:
                break
            count = torch.tensor([max(0, min(n, length - at)) for length in lengths])
            k, v = (r[:, :, at:at + n] for r in rows)
            store.append(k, v, start.cuda(), count.cuda())
            start += count
            at += n
        while at < max(lengths):  # the rest one by one
            count = torch.tensor([int(at < length) for length in lengths])
            store.append(rows[0][:, :, at:at + 1], rows[1][:, :, at:at + 1], start.cuda(), count.cuda())
            start += count
            at += 1
        assert start.tolist() == lengths
        model = Model(batch, heads, dim, block, dtype)
        for b, length in enumerate(lengths):
            model.put(b, rows[0][b, :, :length], rows[1][b, :, :length], 0)
        check_state(store, model, lengths)
        length = max(lengths) + 5
        total = torch.tensor(lengths).cuda()
        k, v = store.read(length, total)
        for b, n in enumerate(lengths):
            for got, r in ((k, model.k[b]), (v, model.v[b])):
                # one product (exact operands) rounded to fp32, then to the type
                close_to(got[b, :, :n], model.values(r), dtype, 2.0 ** -24)
                assert (got[b, :, n:] == 0).all()
        states.append((k, v))
    assert all(torch.equal(states[0][0], s[0]) and torch.equal(states[0][1], s[1]) for s in states)
    assert native.library().lq_block_kv_device_error() == 0


def test_append_strides_host_start_and_taking_tokens_back():
    block, dim, heads = 32, 128, 3
    store = BlockKVStore.allocate(2, heads, dim, 200, block)
    assert store.capacity == 224 and store.max_blocks == 7
    model = Model(2, heads, dim, block, torch.bfloat16)
    wide = rand((2, 150, heads, dim + 8), 21).cuda()
    k, v = wide[..., 8:].transpose(1, 2), wide[..., 3:dim + 3].transpose(1, 2)  # v: rows on odd elements
    store.append(k[:, :, :70], v[:, :, :70], 0)
    store.append(k[:, :, 70:100], v[:, :, 70:100], 70)
    for b in range(2):
        model.put(b, k[b, :, :100], v[b, :, :100], 0)
    check_state(store, model, [100, 100])
    # 32 tokens back (over the border at 96), other tokens in their place: as if they had never been
    store.append(v[:, :, 100:150], k[:, :, 100:150], 68)
    for b in range(2):
        model.put(b, v[b, :, 100:150], k[b, :, 100:150], 68)
    check_state(store, model, [118, 118])
    got = store.read(118, 118)
    for b in range(2):
        close_to(got[0][b], model.values(model.k[b]), torch.bfloat16, 2.0 ** -24)
    before = [t.clone() for t in (store.k_pages, store.k_ring, store.v_ring)]  # (allocate() fills with zeros)
    store.append(k[:, :, :5], v[:, :, :5], 118, torch.zeros(2, dtype=torch.int64).cuda())  # nothing counts
    store.append(k[:, :, :0], v[:, :, :0], 118)
    assert all(torch.equal(a, c) for a, c in zip(before, (store.k_pages, store.k_ring, store.v_ring)))


def test_append_values_that_are_not_finite_and_zeros():
    block = 16
    store = pool_store(1, 2, 64, 3, block, torch.bfloat16)
    k, v = rand((1, 2, 40, 64), 31).cuda(), rand((1, 2, 40, 64), 32).cuda()
    k[0, 0, 3, 7] = math.inf
    v[0, 1, 17, 0] = math.nan
    v[0, 0, 16:32] = 0.0
    k[0, 1, 0, 0] = -3.0e38
    store.append(k, v, 0)
    got_k, got_v = store.read(40, 40)
    assert got_k[0, 0, :16].isnan().all() and got_k[0, 0, 16:].isfinite().all() and got_k[0, 1].isfinite().all()
    assert got_v[0, 1, 16:32].isnan().all() and got_v[0, 1, :16].isfinite().all() and got_v[0, 1, 32:].isfinite().all()
    assert (got_v[0, 0, 16:32] == 0).all()
    assert store.v_scales[store.table[0, 1].long(), 0].item() == torch.tensor(1e-8).item()


# ------------------------------------------------------------------------------- the joined form
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,hq,heads,dim,rot,norm,interleaved", [
    (1, 8, 2, 128, 128, True, False), (1, 3, 1, 64, 64, False, False), (37, 6, 2, 128, 64, True, True),
    (90, 5, 5, 64, 32, True, False),
])
def test_append_qkv_is_norm_rope_then_append(dtype, tokens, hq, heads, dim, rot, norm, interleaved):
    batch, block = 3, 32
    cos, sin = tables(200, rot)
    w = [rand((dim,), s, dtype).cuda() if norm else None for s in (41, 42)]
    one, two = (pool_store(batch, heads, dim, 6, block, dtype, seed=3) for _ in range(2))
    base = rand((batch, heads, 60, dim), 43, dtype).cuda()
    start, count = torch.tensor([30, 0, 60]).cuda(), torch.tensor([tokens, tokens, tokens // 2]).cuda()
    for store in (one, two):
        store.append(base, base, 0, start)
    qkv = rand((batch, tokens, hq + 2 * heads, dim), 44, dtype).cuda()
    pos = start[:, None] + torch.arange(tokens).cuda()
    q, k = qk_norm_rope(qkv[:, :, :hq], qkv[:, :, hq:hq + heads], cos, sin, pos, *w, interleaved=interleaved)
    one.append(k.transpose(1, 2), qkv[:, :, hq + heads:].transpose(1, 2), start, count)
    got = two.append_qkv(qkv, cos, sin, start, count, *w, interleaved=interleaved)
    live = (torch.arange(tokens).cuda()[None] < count[:, None])[..., None, None]
    assert torch.equal(got, torch.where(live, q, torch.zeros_like(q)))
    for name in ("k_pages", "v_pages", "k_scales", "v_scales", "k_ring", "v_ring"):
        a, b = getattr(one, name), getattr(two, name)
        assert torch.equal(a.nan_to_num(7.0) if a.is_floating_point() else a, b.nan_to_num(7.0) if b.is_floating_point() else b), name
    assert native.library().lq_block_kv_device_error() == 0


# ------------------------------------------------------------------------------- attention
def filled(batch, heads, dim, block, dtype, lengths, seed, kstd=1.0, vstd=1.0):
    """A store with `lengths` tokens in each sequence and the definition's values of them."""
    blocks = max(1, -(-(max(lengths)) // block))
    store = pool_store(batch, heads, dim, blocks, block, dtype, seed)
    model = Model(batch, heads, dim, block, dtype)
    n = max(max(lengths), 1)
    k, v = rand((batch, heads, n, dim), seed + 1, dtype, kstd).cuda(), rand((batch, heads, n, dim), seed + 2, dtype, vstd).cuda()
    store.append(k, v, 0, torch.tensor(lengths).cuda())
    for b, length in enumerate(lengths):
        model.put(b, k[b, :, :length], v[b, :, :length], 0)
    return store, model


# The kernel's arithmetic before the last rounding: the weights as fp16 (half a step 2^-11, of each
# weight); one group of bf16 queries as 15-bit integers (2^-14 of the row's largest value, so a score is
# off by at most 2^-14 max|q| sum|k| scaling, under 2^-14 here for all but the sharpest rows, and
# rms far less); scores in fp32. An output is a weighted mean of values, so all of it is within
# (2^-11 + 2^-13) of the largest value; query rows in fp16 and ring rows are exact after the lift.
EXTRA = 2.0 ** -11 + 2.0 ** -13


def check_attend(store, model, q, starts, counts, scaling=None, **kw):
    got = store.attend(q, torch.tensor(starts).cuda(), torch.tensor(counts).cuda(), scaling, **kw)
    scaling = store.head_dim ** -0.5 if scaling is None else scaling
    for b, (s, n) in enumerate(zip(starts, counts)):
        assert (got[b, n:] == 0).all()
        if n == 0:
            continue
        k, v = model.values(model.k[b]), model.values(model.v[b])
        want = attend64(q[b, :n], k, v, s, scaling)
        close_to(got[b, :n], want, store.dtype, EXTRA, v.abs().max())
    assert native.library().lq_block_kv_device_error() == 0
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,group", [(1, 1), (2, 4), (2, 8), (1, 3), (3, 5), (1, 16)])
def test_attend_one_token(dtype, dim, heads, group):
    block = 32
    lengths = [1, 16, 31, 32, 33, 500, 127, 64]
    store, model = filled(8, heads, dim, block, dtype, lengths, 51)
    q = rand((8, 1, heads * group, dim), 54, dtype, 2.0).cuda()
    check_attend(store, model, q, [n - 1 for n in lengths], [1] * 8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("tokens,group", [(2, 4), (3, 3), (4, 4), (5, 8), (17, 3), (64, 2), (150, 1), (80, 1), (81, 1),
                                          (43, 3), (129, 2)])
def test_attend_several_tokens(dtype, block, tokens, group):
    """Drafts and chunks: causal inside the call, counts that differ, sequences that begin empty."""
    dim, heads = (128, 2) if block != 16 else (64, 1)
    starts, counts = [0, 3 * block - 1, 70, 200], [tokens, tokens, max(1, tokens // 2), 0]
    lengths = [s + n for s, n in zip(starts, counts)]
    store, model = filled(4, heads, dim, block, dtype, lengths, 61)
    q = rand((4, tokens, heads * group, dim), 64, dtype, 2.0).cuda()
    check_attend(store, model, q, starts, counts)


def test_attend_long_context_and_single_run():
    store, model = filled(1, 2, 128, 128, torch.bfloat16, [20011], 71)
    q = rand((1, 1, 8, 128), 74, std=4.0).cuda()
    check_attend(store, model, q, [20010], [1])
    # many sequences: every CTA meets several of them
    lengths = [(37 * i) % 300 + 1 for i in range(200)]
    store, model = filled(200, 2, 64, 16, torch.float16, lengths, 75)
    q = rand((200, 1, 4, 64), 76, torch.float16, 2.0).cuda()
    check_attend(store, model, q, [n - 1 for n in lengths], [1] * 200)


@pytest.mark.parametrize("tokens", [1, 5, 60])  # each of the kernels: 2, 10 and 120 rows
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attend_blocks_of_very_different_scale(tokens, dtype):
    """Value scales far apart, blocks of zeros, keys that decide: the folded scale must cancel."""
    block = 16
    model = Model(1, 1, 64, block, dtype)
    store = pool_store(1, 1, 64, 8, block, dtype)
    k, v = rand((1, 1, 125, 64), 82, dtype).cuda(), rand((1, 1, 125, 64), 83, dtype).cuda()
    for i, s in enumerate((1e-6, 1e4, 0.0, 1.0, 3e-3, 100.0, 1e-2, 1.0)):
        v[:, :, i * 16:(i + 1) * 16] *= s
    model.put(0, k[0], v[0], 0)
    store.append(k, v, 0)
    for std in (0.1, 2.0, 12.0):
        q = rand((1, tokens, 2, 64), 84, dtype, std=std).cuda()
        check_attend(store, model, q, [125 - tokens], [tokens])
    v[:] = 0.0
    store.append(k, v, 0)
    assert (store.attend(q, 125 - tokens) == 0).all()


def test_attend_strides_scratch_out_and_scaling():
    store, model = filled(2, 2, 128, 64, torch.bfloat16, [130, 90], 91)
    q = rand((2, 8, 1, 128), 94).cuda().transpose(1, 2)  # [2, 1, 8, 128] from heads first
    got = check_attend(store, model, q, [129, 89], [1, 1], scaling=0.3)
    out = torch.empty_like(got)
    scratch = torch.empty(store.scratch_bytes(8, 1), dtype=torch.uint8, device="cuda").fill_(255)
    again = store.attend(q, torch.tensor([129, 89]).cuda(), scaling=0.3, out=out, scratch=scratch)
    assert again is out and torch.equal(out, got)
    for tokens in (1, 4, 30):  # rows on odd elements, each of the kernels
        q = rand((2, tokens, 8, 128), 95).cuda()
        wide = torch.zeros(2, tokens, 8, 256, dtype=q.dtype, device="cuda")[..., 1:129]
        wide.copy_(q)
        start = torch.tensor([130 - tokens, 90 - tokens]).cuda()
        assert torch.equal(store.attend(wide, start), store.attend(q, start))


@pytest.mark.parametrize("tokens", [1, 6, 50])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attend_values_that_are_not_finite(tokens, dtype):
    """What a sequence does not hold must not reach it: rubbish behind its length, other sequences."""
    block = 16
    lengths = [tokens + 39, tokens + 19]
    store, model = filled(2, 1, 64, block, dtype, [n + 33 for n in lengths], 101)
    q = rand((2, tokens, 2, 64), 104, dtype).cuda()
    start = torch.tensor([39, 19]).cuda()
    store.append(rand((2, 1, tokens, 64), 107, dtype).cuda(), rand((2, 1, tokens, 64), 108, dtype).cuda(), start)
    want = store.attend(q, start)
    assert want.isfinite().all()
    k = torch.full((2, 1, 4, 64), math.nan, dtype=dtype, device="cuda")
    store.append(k, k, torch.tensor(lengths).cuda())  # taken back by the next call's start
    assert torch.equal(store.attend(q, start), want)
    # one sequence with NaN in a complete block: its rows only
    k = rand((2, 1, 16, 64), 106, dtype).cuda()
    k[0, 0, 0, 0] = math.nan
    store.append(k, k, torch.tensor([16, 0]).cuda())
    got = store.attend(q, start)
    assert got[0].isnan().all() and got[1].isfinite().all()
    k = rand((2, 1, 16, 64), 109, dtype).cuda()
    store.append(k, k, torch.tensor([16, 0]).cuda())
    assert store.attend(q, start).isfinite().all()
    # a NaN in a row that is still in the ring: that sequence only
    k = rand((2, 1, 1, 64), 110, dtype).cuda()
    k[1] = math.inf
    store.append(k, k, torch.tensor([n - 1 for n in lengths]).cuda())
    got = store.attend(q, start)
    assert got[0].isfinite().all() and not got[1, -1].isfinite().any()
    # and a query that is not finite: its own row only
    q[0, tokens - 1, 1, 3] = math.nan
    got = store.attend(q, start)
    assert got[0, tokens - 1, 1].isnan().all() and got[0, tokens - 1, 0].isfinite().all()
    assert got[0, : tokens - 1].isfinite().all()


@pytest.mark.parametrize("tokens", [1, 6, 50])
def test_bad_pages_and_spans_are_skipped_and_reported(tokens):
    store, model = filled(2, 1, 64, 16, torch.bfloat16, [64, 64], 111)
    q = rand((2, tokens, 2, 64), 114).cuda()
    last = 64 - tokens
    want = store.attend(q, torch.tensor([last, last]).cuda())
    table = store.table.clone()
    for bad in (-1, store.k_pages.shape[0], 2 ** 31 - 1):
        store.table[0, 1] = bad
        got = store.attend(q, torch.tensor([last, last]).cuda())
        assert got[0, max(0, 16 - last):].isnan().all() and torch.equal(got[1], want[1])  # (the rows that see block 1)
        with pytest.raises(RuntimeError, match="page id outside the pool"):
            store.check_device_errors()
        k, _ = store.read(64, 64)
        assert k[0, :, 16:32].isnan().all() and k[0, :, :16].isfinite().all()
        pages = store.k_pages.clone()
        row = rand((2, 1, 32, 64), 115).cuda()
        store.append(row, row, 0, torch.tensor([32, 0]).cuda())
        keep = torch.ones(pages.shape[0], dtype=torch.bool)
        keep[table[0, 0].item()] = False
        assert torch.equal(store.k_pages[keep.cuda()], pages[keep.cuda()])
        with pytest.raises(RuntimeError, match="page id outside the pool"):
            store.check_device_errors()
        store.check_device_errors()
    store.table.copy_(table)
    ring = store.k_ring.view(torch.int16).clone()  # (by bits: there is rubbish NaN in it)
    for start in (-1, 64, 2 ** 40):  # the table ends at 64
        row = rand((2, 1, 1, 64), 116).cuda()
        store.append(row, row, torch.tensor([start, 64]).cuda(), torch.tensor([1, 0]).cuda())
        assert torch.equal(store.k_ring.view(torch.int16), ring)
        with pytest.raises(RuntimeError, match="outside the table"):
            store.check_device_errors()
        got = store.attend(q, torch.tensor([start, last]).cuda())
        assert (got[0] == 0).all() and torch.equal(got[1], want[1])
        with pytest.raises(RuntimeError, match="outside the table"):
            store.check_device_errors()


def test_counts_that_are_nothing_or_too_much():
    store, model = filled(3, 1, 64, 32, torch.bfloat16, [70, 70, 70], 151)
    for tokens in (1, 7, 100):
        q = rand((3, tokens, 2, 64), 152).cuda()
        none = torch.tensor([0, -5, -2 ** 40]).cuda()
        assert (store.attend(q, torch.tensor([0, 30, 69]).cuda(), none) == 0).all()
        before = store.k_ring.clone()
        row = rand((3, 1, tokens, 64), 153).cuda()
        store.append(row, row, torch.tensor([0, 30, 69]).cuda(), none)
        assert torch.equal(before.view(torch.int16), store.k_ring.view(torch.int16))
    q = rand((3, 4, 2, 64), 154).cuda()
    start = torch.tensor([66, 40, 33]).cuda()  # (the ring reaches back to 32)
    assert torch.equal(store.attend(q, start, torch.tensor([4, 2 ** 40, 99]).cuda()), store.attend(q, start))
    store.check_device_errors()


def test_a_pool_whose_offsets_pass_31_bits():
    """Pages behind 2^31 bytes of codes: append, read and both attentions."""
    heads, dim, block = 8, 128, 128
    pages = 2 ** 31 // (heads * dim * block) + 40
    codes = [torch.empty(pages, heads, block, dim, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.empty(pages, heads, device="cuda") for _ in range(2)]
    rings = [torch.empty(1, heads, 2 * block, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    table = torch.arange(pages - 1, pages - 9, -1, dtype=torch.int32, device="cuda")[None].contiguous()
    store = BlockKVStore(*codes, *scales, *rings, table)
    small = BlockKVStore.allocate(1, heads, dim, 8 * block, block)
    k, v = rand((1, heads, 1000, dim), 161).cuda(), rand((1, heads, 1000, dim), 162).cuda()
    for s in (store, small):
        s.append(k, v, 0)
    assert all(torch.equal(a, b) for a, b in zip(store.read(1000, 1000), small.read(1000, 1000)))
    for tokens in (1, 40):
        q = rand((1, tokens, 4 * heads, dim), 163).cuda()
        assert torch.equal(store.attend(q, 1000 - tokens), small.attend(q, 1000 - tokens))
    store.check_device_errors()


# ------------------------------------------------------------------------------- together
def test_decode_in_a_graph_and_on_another_stream():
    """Prompt, then decode steps: eager, replayed from a captured graph with the cursor on the device,
    and on a side stream; all the same bits."""
    batch, hq, heads, dim, block = 3, 8, 2, 128, 32
    cos, sin = tables(160, dim)
    w = rand((dim,), 121).cuda()
    prompt, steps = torch.tensor([20, 65, 1]), 70
    first = rand((batch, 65, hq + 2 * heads, dim), 122).cuda()
    rows = rand((steps, batch, 1, hq + 2 * heads, dim), 123).cuda()

    def fresh():
        store = pool_store(batch, heads, dim, 5, block, torch.bfloat16, seed=9)
        store.append_qkv(first, cos, sin, 0, prompt.cuda(), w, w)
        return store

    store, start, eager = fresh(), prompt.cuda(), []
    for i in range(steps):
        q = store.append_qkv(rows[i], cos, sin, start, None, w, w)
        eager.append(store.attend(q, start))
        start = start + 1

    graphed, start = fresh(), prompt.cuda()
    feed = rows[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q = graphed.append_qkv(feed, cos, sin, start, None, w, w)
        graphed.attend(q, start)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = graphed.append_qkv(feed, cos, sin, start, None, w, w)
        out = graphed.attend(q, start, pdl=True)
        start.add_(1)
    for i in range(steps):
        feed.copy_(rows[i])
        graph.replay()
        assert torch.equal(out, eager[i]), i

    other, start = fresh(), prompt.cuda()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for i in range(steps):
            q = other.append_qkv(rows[i], cos, sin, start, None, w, w, pdl=True)
            got = other.attend(q, start, pdl=True)
            start = start + 1
    side.synchronize()
    assert torch.equal(got, eager[-1])
    # and the definition at the last step
    model = Model(batch, heads, dim, block, torch.bfloat16)
    store.check_device_errors()
    k, v = store.read(160, prompt.cuda() + steps)
    for b in range(batch):
        n = int(prompt[b]) + steps
        q = norm_rope64(rows[-1][b, :, :hq], w, cos[n - 1:n], sin[n - 1:n], False, 1e-6).bfloat16()
        want = attend64(q, k[b, :, :n].double().cpu(), v[b, :, :n].double().cpu(), n - 1, dim ** -0.5)
        # (values read back are rounded to bf16 once more than the cache's: 2^-8 of keys and values,
        # the keys' error entering through scores |q| |k| 2^-9 <~ 2^-3 at these sizes)
        rel = (eager[-1][b].double().cpu() - want).norm() / want.norm()
        assert rel < 2.0 ** -6, rel
    assert model.block == block


@pytest.mark.parametrize("tokens", [1, 2, 24])
def test_two_stores_on_two_streams_at_once(tokens):
    stores = [filled(4, 2, 128, 64, torch.bfloat16, [900, tokens, 333, 64], 130 + i) for i in range(2)]
    q = rand((4, tokens, 16, 128), 139).cuda()
    start = torch.tensor([900 - tokens, 0, 333 - tokens, 64 - tokens]).cuda()
    want = [s.attend(q, start) for s, _ in stores]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, (s, _) in enumerate(stores):
            with torch.cuda.stream(streams[i]):
                got[i].append(s.attend(q, start))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_refusals():
    store = BlockKVStore.allocate(2, 2, 64, 100, 32)
    k = rand((2, 2, 3, 64), 141).cuda()
    with pytest.raises(RuntimeError, match="k must be torch.bfloat16"):
        store.append(k.half(), k.half(), 0)
    with pytest.raises(RuntimeError, match="v must be"):
        store.append(k, k[:, :1], 0)
    with pytest.raises(RuntimeError, match="do not fit"):
        store.append(k, k, 126)
    with pytest.raises(RuntimeError, match="start must be"):
        store.append(k, k, torch.zeros(3, dtype=torch.int64).cuda())
    with pytest.raises(RuntimeError, match="start must be"):
        store.append(k, k, torch.zeros(2, dtype=torch.int32).cuda())
    with pytest.raises(RuntimeError, match="count must be"):
        store.append(k, k, 0, torch.zeros(2).cuda())
    q = rand((2, 1, 4, 64), 142).cuda()
    with pytest.raises(RuntimeError, match="share 2 KV heads"):
        store.attend(q[:, :, :3], 0)
    with pytest.raises(RuntimeError, match="scratch must be"):
        store.attend(q, 0, scratch=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(RuntimeError, match="q must be"):
        store.attend(q[:1], 0)
    assert store.attend(q[:, :0], 0).shape == (2, 0, 4, 64)
    f32 = BlockKVStore.allocate(1, 1, 64, 32, 32, dtype=torch.float32)
    with pytest.raises(RuntimeError, match="float16 and bfloat16"):
        f32.attend(torch.zeros(1, 1, 1, 64, device="cuda"), 0)
    cos, sin = tables(10, 64)
    with pytest.raises(RuntimeError, match="no angles"):
        store.append_qkv(rand((2, 1, 8, 64), 143).cuda(), cos, sin, 10)
    with pytest.raises(RuntimeError, match="float32 tables"):
        qk_norm_rope(q, q, cos.half(), sin.half(), torch.zeros(2, 1, dtype=torch.int64).cuda())
    with pytest.raises(RuntimeError, match="both queries and keys"):
        qk_norm_rope(q, q, cos, sin, torch.zeros(2, 1, dtype=torch.int64).cuda(), q_weight=torch.ones(64).bfloat16().cuda())
    with pytest.raises(RuntimeError, match="contiguous on"):
        BlockKVStore(store.k_pages.transpose(0, 1), store.v_pages, store.k_scales, store.v_scales, store.k_ring,
                     store.v_ring, store.table)
    with pytest.raises(RuntimeError, match="one of"):
        BlockKVStore.allocate(1, 1, 64, 32, 48)


def test_errors_of_another_stream_are_reported():
    store, _ = filled(1, 1, 64, 16, torch.bfloat16, [64], 141)
    k = rand((1, 1, 1, 64), 142).cuda()
    late = torch.tensor([64], device="cuda")  # one token behind a cache of 64
    assert store.capacity == 64
    store.append(k, k, late - 1)
    store.check_device_errors()
    busy = torch.randn(4096, 4096, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(50):  # (the call is still waiting for these when the check is made)
            busy = busy @ busy
        store.append(k, k, late)
    with pytest.raises(RuntimeError, match="outside the table"):
        store.check_device_errors()
    store.check_device_errors()
