"""CPU-side checks of the block-scaled KV cache and the norm + rotation: what the C entry points and
the Python calls refuse before any launch, and the scratch arithmetic."""

import ctypes
import re

import pytest
import torch

from llmquant_b200 import native
from llmquant_b200.cuda import qk_norm_rope
from llmquant_b200.quantizers import BlockKVStore


def cache(**kw):
    fields = dict(k_pages=4096, v_pages=4096, k_scales=64, v_scales=64, k_ring=4096, v_ring=4096, table=64, num_pages=8,
                  max_blocks=4, batch=2, kv_heads=2, head_dim=128, block=64, dtype=native.LQ_BF16)
    return ctypes.byref(native.BlockKV(**dict(fields, **kw)))


def append(c, k=4096, tokens=1):
    strides = (ctypes.c_int64 * 3)(256, 128, 128)
    native.call("lq_block_kv_append", c, k, k, strides, strides, tokens, 0, 0, 0, 0, 0, 0)


def attend(c, q=4096, hq=8, tokens=1, scratch=4096, size=1 << 30, strides=(1024, 1024, 128), out=4096):
    native.call("lq_block_attn", c, q, (ctypes.c_int64 * 3)(*strides), out, scratch, size, hq, tokens, 0, 0, 0, 0, 0.1, 0, 0)


@pytest.mark.parametrize("fields,match", [
    (dict(head_dim=96), "head_dim 64 and 128"), (dict(block=48), "16, 32, 64 or 128"), (dict(batch=0), "bad cache shape"),
    (dict(num_pages=0), "bad cache shape"), (dict(max_blocks=1 << 26), "too many positions"), (dict(dtype=7), "dtype id 7"),
    (dict(table=0), "null cache pointer"), (dict(v_pages=4104), "16-byte aligned"), (dict(k_ring=4098), "16-byte aligned"),
])
def test_a_bad_cache_is_refused_everywhere(fields, match):
    bad = cache(**fields)
    for call in (append, attend,
                 lambda c: native.call("lq_block_kv_read", c, 4096, 4096, 10, 0, 0, 0, 0, 1, 0, 0),
                 lambda c: native.call("lq_block_kv_append_qkv", c, 4096, 1536, 1536, 4096, 8, 1, 0, 0, 1e-6, 64, 64, 10,
                                       128, 0, 0, 0, 0, 0, 0, 0)):
        with pytest.raises(RuntimeError, match=match):
            call(bad)


def test_bad_arguments_are_refused():
    with pytest.raises(RuntimeError, match="no cache given"):
        append(None)
    with pytest.raises(RuntimeError, match="null tensor pointer"):
        append(cache(), k=0)
    with pytest.raises(RuntimeError, match="no tokens"):
        append(cache(), tokens=0)
    with pytest.raises(RuntimeError, match="share 2 KV heads evenly"):
        attend(cache(), hq=7)
    with pytest.raises(RuntimeError, match="float16 and bfloat16"):
        attend(cache(dtype=native.LQ_F32))
    with pytest.raises(RuntimeError, match="bytes, .* are needed"):
        attend(cache(), size=64)
    with pytest.raises(RuntimeError, match="scratch must be 16-byte aligned"):
        attend(cache(), scratch=4100)
    with pytest.raises(RuntimeError, match="out must be 16-byte aligned"):
        attend(cache(), out=4098)
    with pytest.raises(RuntimeError, match="empty output"):
        native.call("lq_block_kv_read", cache(), 4096, 4096, 0, 0, 0, 0, 0, 1, 0, 0)
    qkv = [4096, 1536, 1536, 4096, 8, 1, 0, 0, 1e-6, 64, 64, 10, 128, 0, 0, 0, 0, 0, 0, 0]
    for at, value, match in ((4, 0, "no heads"), (6, 64, "both queries and keys"), (9, 0, "tables are missing"),
                             (9, 68, "tables must be 16-byte"), (12, 40, "multiple of 16"), (12, 144, "multiple of 16")):
        args = list(qkv)
        args[at] = value
        with pytest.raises(RuntimeError, match=match):
            native.call("lq_block_kv_append_qkv", cache(), *args)
    strides = (ctypes.c_int64 * 3)(1024, 1024, 128)
    rope = [4096, 4096, strides, strides, 4096, 4096, strides, strides, native.LQ_BF16, 1, 1, 8, 8, 128, 0, 0, 1e-6, 64, 64,
            10, 128, 0, 64, 0, 0, 0, 0]
    for at, value, match in ((8, 9, "dtype id 9"), (9, 0, "bad shape"), (13, 100, "multiple of 8"), (13, 264, "multiple of 8"),
                             (14, 64, "both queries and keys"), (20, 8, "multiple of 16"), (22, 0, "null tensor pointer"),
                             (0, 0, "null tensor pointer")):
        args = list(rope)
        args[at] = value
        with pytest.raises(RuntimeError, match=match):
            native.call("lq_qk_norm_rope", *args)


def test_scratch_covers_a_part_for_each_cta_and_head():
    lib = native.library()
    for batch, hkv, hq, tokens, dim in ((1, 8, 32, 1, 128), (64, 8, 32, 1, 64), (3, 2, 16, 5, 128), (1, 1, 1, 700, 64)):
        need = lib.lq_block_attn_scratch_bytes(cache(batch=batch, kv_heads=hkv, head_dim=dim), hq, tokens)
        rows = tokens * (hq // hkv)
        assert need % 4 == 0 and need >= batch * hkv * rows * (dim + 2) * 4
    assert lib.lq_block_attn_scratch_bytes(cache(), 7, 1) == -1


def test_cpu_tensors_are_refused():
    codes = torch.zeros(4, 2, 16, 64, dtype=torch.int8)
    scales, ring = torch.zeros(4, 2), torch.zeros(1, 2, 32, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        BlockKVStore(codes, codes, scales, scales, ring, ring, torch.zeros(1, 4, dtype=torch.int32))
    x = torch.zeros(1, 1, 2, 64)
    with pytest.raises(RuntimeError, match="must be CUDA tensors"):
        qk_norm_rope(x, x, torch.zeros(4, 32), torch.zeros(4, 32), torch.zeros(1, 1, dtype=torch.int64))


def test_block_kv_struct_matches_the_header():
    text = native.HEADER.read_text()
    body = text[text.index("typedef struct lq_block_kv {"):text.index("} lq_block_kv;")]
    body = re.sub(r"/\*.*?\*/", "", body.partition("{")[2], flags=re.S)
    names = [n for n in re.findall(r"\w+(?=\s*[;,])", body)]
    assert names == [n for n, _ in native.BlockKV._fields_]
    # seven pointers, one int64, six ints
    assert ctypes.sizeof(native.BlockKV) == 7 * 8 + 8 + 6 * 4
