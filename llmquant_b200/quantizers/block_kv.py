"""A paged KV cache in 8 bits with one scale for each block of tokens and KV head.

`BlockKVStore` is one layer's cache and the calls on it: `append` (quantize on write), `append_qkv`
(norms of q and k, rotation and append from the fused projection's rows, one launch), `attend` (any
number of new tokens, sequences of different lengths) and `read` (the values back). A block is
quantized once, when its last token arrives; the rows of the incomplete block and of the one
before it stay as they came in a ring, so the cache depends on the tokens and not on how they were
cut into calls, and a smaller `start` takes tokens back without loss as far as the ring reaches. The
layout is `lq_block_kv` of include/llmquant_b200.h.

`BlockKVCache` puts it behind transformers' `Cache`, as `KernelQuantCache` does with the cache that
has a scale per token; `make_cache_factory(8, block_tokens=64)` makes it. The reference has
neither pages nor sequences of different lengths (llmquant/quantizers/fake.py:39-62).
"""

import ctypes
import functools

import torch
from transformers.cache_utils import Cache, CacheLayerMixin

from llmquant_b200 import native
from llmquant_b200.cuda.ops import check_norm_weights, check_rope_tables

BLOCK_TOKENS = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)


class BlockKVStore:
    """One layer's block-scaled cache over tensors that the caller owns:

      k_pages, v_pages    int8 [pages, kv_heads, block, head_dim]
      k_scales, v_scales  float32 [pages, kv_heads]
      k_ring, v_ring      [batch, kv_heads, 2 * block, head_dim], the type of the rows that come and go
      table               int32 [batch, max_blocks], the page of each block of a sequence

    Every call names the tokens it is about: `start` cached tokens (an int for all sequences, or
    int64 [batch] / [1] on the device) and `count` new rows that count (None: all of them, or
    int64 [batch]). Nothing advances by itself. `start` and `count` tensors are read on the GPU: what
    is wrong in them (tokens beyond the table, page ids outside the pool) is skipped there and
    raised by `check_device_errors`. Calls run on torch's current stream of the cache's device and
    can be captured into CUDA graphs, once one call of the kind has run outside a capture. No gradients."""

    def __init__(self, k_pages, v_pages, k_scales, v_scales, k_ring, v_ring, table):
        tensors = dict(k_pages=k_pages, v_pages=v_pages, k_scales=k_scales, v_scales=v_scales, k_ring=k_ring,
                       v_ring=v_ring, table=table)
        for name, t in tensors.items():
            if not t.is_cuda:
                raise RuntimeError(f"{name} must be a CUDA tensor: there is no CPU fallback")
            if t.device != k_pages.device or not t.is_contiguous():
                raise RuntimeError(f"{name} must be contiguous on {k_pages.device}")
        if k_pages.dim() != 4 or k_pages.dtype != torch.int8:
            raise RuntimeError("k_pages must be int8 [pages, kv_heads, block, head_dim]")
        pages, heads, block, dim = k_pages.shape
        if block not in BLOCK_TOKENS:
            raise RuntimeError(f"a block must be one of {BLOCK_TOKENS} tokens, got {block}")
        if dim not in HEAD_DIMS:
            raise RuntimeError(f"head_dim must be one of {HEAD_DIMS}, got {dim}")
        if k_ring.dtype not in native.DTYPE_ID:
            raise RuntimeError(f"the rings must be float32, float16 or bfloat16, got {k_ring.dtype}")
        if table.dim() != 2 or table.dtype != torch.int32:
            raise RuntimeError("table must be int32 [batch, max_blocks]")
        batch, blocks = table.shape
        want = dict(v_pages=(k_pages.shape, torch.int8), k_scales=((pages, heads), torch.float32),
                    v_scales=((pages, heads), torch.float32), k_ring=((batch, heads, 2 * block, dim), k_ring.dtype),
                    v_ring=((batch, heads, 2 * block, dim), k_ring.dtype))
        for name, (shape, dtype) in want.items():
            if tuple(tensors[name].shape) != tuple(shape) or tensors[name].dtype != dtype:
                raise RuntimeError(f"{name} must be {dtype} {tuple(shape)}, got {tensors[name].dtype} "
                                   f"{tuple(tensors[name].shape)}")
        if min(pages, heads, batch, blocks) == 0:
            raise RuntimeError("the cache has no pages, heads, sequences or blocks")
        self.k_pages, self.v_pages, self.k_scales, self.v_scales = k_pages, v_pages, k_scales, v_scales
        self.k_ring, self.v_ring, self.table = k_ring, v_ring, table
        self.batch, self.max_blocks, self.heads, self.head_dim, self.block = batch, blocks, heads, dim, block
        self.capacity = blocks * block
        self.dtype, self.device = k_ring.dtype, k_ring.device
        desc = native.BlockKV(k_pages.data_ptr(), v_pages.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(),
                              k_ring.data_ptr(), v_ring.data_ptr(), table.data_ptr(), pages, blocks, batch, heads, dim,
                              block, native.DTYPE_ID[self.dtype])
        self._desc, self._ref = desc, ctypes.byref(desc)
        self._index, self._batch_shape = self.device.index, (batch,)
        self._scratch_bytes = {}

    @classmethod
    def allocate(cls, batch, kv_heads, head_dim, max_tokens, block_tokens=64, dtype=torch.bfloat16, device="cuda"):
        """An empty cache of `max_tokens` positions for each of `batch` sequences, with pages of its own."""
        if block_tokens not in BLOCK_TOKENS:
            raise RuntimeError(f"a block must be one of {BLOCK_TOKENS} tokens, got {block_tokens}")
        blocks = -(-max_tokens // block_tokens)
        pages = batch * blocks
        codes = [torch.zeros(pages, kv_heads, block_tokens, head_dim, dtype=torch.int8, device=device) for _ in range(2)]
        scales = [torch.zeros(pages, kv_heads, dtype=torch.float32, device=device) for _ in range(2)]
        rings = [torch.zeros(batch, kv_heads, 2 * block_tokens, head_dim, dtype=dtype, device=device) for _ in range(2)]
        table = torch.arange(pages, dtype=torch.int32, device=device).reshape(batch, blocks)
        return cls(*codes, *scales, *rings, table)

    def _span(self, start, count, tokens):
        """(start_dev, start_stride, start, count_dev) of the C calls."""
        if isinstance(start, torch.Tensor):
            shape = start.shape
            if start.dtype is not torch.int64 or start.device != self.device or (shape != self._batch_shape and shape != (1,)):
                raise RuntimeError(f"start must be an int or int64 [{self.batch}] (or [1]) on {self.device}")
            where, step, start = start.data_ptr(), start.stride(0) if shape == self._batch_shape else 0, 0
        else:
            if not 0 <= start <= self.capacity - (tokens if count is None else 0):
                raise RuntimeError(f"tokens {start} .. {start + tokens} do not fit a cache of {self.capacity}")
            where = step = 0
        if count is None:
            return where, step, start, 0
        if not isinstance(count, torch.Tensor) or count.dtype is not torch.int64 or count.device != self.device or \
                count.shape != self._batch_shape or not count.is_contiguous():
            raise RuntimeError(f"count must be None or a contiguous int64 [{self.batch}] on {self.device}")
        return where, step, start, count.data_ptr()

    def _rows(self, t, name, shape):
        if t.dtype is not self.dtype or t.device != self.device:
            raise RuntimeError(f"{name} must be {self.dtype} on {self.device}, got {t.dtype} on {t.device}")
        if t.shape != shape:
            raise RuntimeError(f"{name} must be {shape}, got {tuple(t.shape)}")

    def append(self, k, v, start, count=None, pdl=True):
        """Store new rows k, v [batch, kv_heads, tokens, head_dim] (any strides, head_dim contiguous)."""
        if k.dim() != 4:
            raise RuntimeError(f"k must be [batch, kv_heads, tokens, head_dim], got {tuple(k.shape)}")
        tokens = k.shape[2]
        shape = (self.batch, self.heads, tokens, self.head_dim)
        self._rows(k, "k", shape)
        self._rows(v, "v", shape)
        span = self._span(start, count, tokens)
        if tokens == 0:
            return
        ks, vs = k.stride(), v.stride()
        if ks[3] != 1:
            k = k.contiguous()
            ks = k.stride()
        if vs[3] != 1:
            v = v.contiguous()
            vs = v.stride()
        native.launch("lq_block_kv_append", self._index, self._ref, k.data_ptr(), v.data_ptr(), native.int64s(ks),
                      native.int64s(vs), tokens, *span, int(pdl))

    def append_qkv(self, qkv, cos, sin, start, count=None, q_weight=None, k_weight=None, eps=1e-6, interleaved=False,
                   q_out=None, pdl=True):
        """From the fused projection's rows qkv [batch, tokens, q heads + 2 kv heads, head_dim]: queries and
        keys normed (weights given) and turned by their positions' angles, keys and values stored,
        queries returned as [batch, tokens, q heads, head_dim] (`q_out`, which must not overlap qkv, or
        new). One launch; the same values as `qk_norm_rope` followed by `append`."""
        if qkv.dim() != 4 or qkv.shape[2] <= 2 * self.heads:
            raise RuntimeError(f"qkv must be [batch, tokens, q heads + {2 * self.heads}, head_dim], got {tuple(qkv.shape)}")
        _, tokens, heads, _ = qkv.shape
        self._rows(qkv, "qkv", (self.batch, tokens, heads, self.head_dim))
        heads -= 2 * self.heads
        table_len, rot = check_rope_tables(cos, sin, self.device, self.head_dim)
        wq, wk = check_norm_weights(q_weight, k_weight, self.dtype, self.device, self.head_dim)
        if isinstance(start, int) and count is None and start + tokens > table_len:
            raise RuntimeError(f"tokens {start} .. {start + tokens} have no angles in tables of {table_len} positions")
        span = self._span(start, count, tokens)
        strides = qkv.stride()
        if strides[3] != 1 or strides[2] != self.head_dim:
            qkv = qkv.contiguous()
            strides = qkv.stride()
        shape = (self.batch, tokens, heads, self.head_dim)
        if q_out is None:
            q_out = torch.empty(shape, dtype=self.dtype, device=self.device)
        else:
            self._rows(q_out, "q_out", shape)
            if not q_out.is_contiguous():
                raise RuntimeError("q_out must be contiguous")
        if tokens == 0:
            return q_out
        native.launch("lq_block_kv_append_qkv", self._index, self._ref, qkv.data_ptr(), strides[0], strides[1],
                      q_out.data_ptr(), heads, tokens, wq, wk, eps, cos.data_ptr(), sin.data_ptr(), table_len, rot,
                      int(interleaved), *span, int(pdl))
        return q_out

    def scratch_bytes(self, q_heads, tokens):
        """Bytes of scratch one `attend` call of this shape takes."""
        key = (q_heads, tokens)
        need = self._scratch_bytes.get(key)
        if need is None:
            with torch.cuda.device(self.device):  # (its SM count decides)
                need = native.library().lq_block_attn_scratch_bytes(self._ref, q_heads, tokens)
            if need < 0:
                raise RuntimeError(native.last_error())
            self._scratch_bytes[key] = need
        return need

    def attend(self, q, start, count=None, scaling=None, out=None, scratch=None, pdl=True):
        """Attention of the newest rows q [batch, tokens, q heads, head_dim] (head_dim contiguous) over the
        cache after their `append`: row t sees positions 0 .. start + t. Returns [batch, tokens,
        q heads, head_dim], zeros for rows behind `count`. float16 and bfloat16 caches. `scratch`
        (uint8, `scratch_bytes`) comes from torch's allocator unless given; two calls that may
        overlap must not share one."""
        if q.dim() != 4:
            raise RuntimeError(f"q must be [batch, tokens, q heads, head_dim], got {tuple(q.shape)}")
        _, tokens, heads, _ = q.shape
        shape = (self.batch, tokens, heads, self.head_dim)
        self._rows(q, "q", shape)
        if self.dtype is torch.float32:
            raise RuntimeError("attention over the block-scaled cache is built for float16 and bfloat16 rows")
        if heads == 0 or heads % self.heads:
            raise RuntimeError(f"{heads} query heads do not share {self.heads} KV heads evenly")
        span = self._span(start, count, tokens)
        if out is None:
            out = torch.empty(shape, dtype=self.dtype, device=self.device)
        else:
            self._rows(out, "out", shape)
            if not out.is_contiguous():
                raise RuntimeError("out must be contiguous")
        if tokens == 0:
            return out
        strides = q.stride()
        if strides[3] != 1:
            q = q.contiguous()
            strides = q.stride()
        need = self.scratch_bytes(heads, tokens)
        if scratch is None:
            scratch = torch.empty(need, dtype=torch.uint8, device=self.device)
        elif scratch.device != self.device or scratch.dtype is not torch.uint8 or scratch.numel() < need or \
                not scratch.is_contiguous():
            raise RuntimeError(f"scratch must be {need} contiguous uint8 on {self.device}")
        native.launch("lq_block_attn", self._index, self._ref, q.data_ptr(), native.int64s(strides), out.data_ptr(),
                      scratch.data_ptr(), need, heads, tokens, *span,
                      self.head_dim ** -0.5 if scaling is None else scaling, int(pdl))
        return out

    def read(self, length, start, count=None, tokens=0):
        """(K, V) [batch, kv_heads, length, head_dim]: the values the cache stands for with start + count
        tokens in it (count None: start + tokens), zeros behind each sequence."""
        if length < 0:
            raise RuntimeError(f"length must not be negative, got {length}")
        span = self._span(start, count, tokens)
        if count is not None:
            tokens = self.capacity  # count alone decides
        shape = (self.batch, self.heads, length, self.head_dim)
        k = torch.empty(shape, dtype=self.dtype, device=self.device)
        v = torch.empty(shape, dtype=self.dtype, device=self.device)
        if length:
            native.launch("lq_block_kv_read", self._index, self._ref, k.data_ptr(), v.data_ptr(), length, *span, tokens, 1)
        return k, v

    def check_device_errors(self):
        """Raise if a call since the last check met a bad `start`, `count`, page id or position (waits
        for the work of all streams)."""
        torch.cuda.synchronize(self.device)  # (the word is read on the default stream)
        with torch.cuda.device(self.device):
            word = native.library().lq_block_kv_device_error()
        if word:
            what = {1: "met a page id outside the pool and skipped it", 2: "met tokens outside the table and skipped them",
                    3: "met a position outside the angle tables", 4: "gave up a wait for the tensor cores",
                    }.get(word, f"left error word {word}")
            raise RuntimeError(f"block-scaled KV cache: a kernel {what}")


class BlockKVLayer(CacheLayerMixin):
    """One layer of `BlockKVCache`: a `BlockKVStore` that all sequences fill alike and that grows."""

    is_sliding = False
    is_compileable = False
    num_bits = 8

    def __init__(self, block_tokens: int = 64, max_cache_len=None, fused_read: bool = False):
        super().__init__()
        if block_tokens not in BLOCK_TOKENS:
            raise ValueError(f"a block must be one of {BLOCK_TOKENS} tokens, got {block_tokens}")
        self.block_tokens = block_tokens
        self.max_cache_len = max_cache_len
        self.fused_read = fused_read
        self.dequant_calls = self.fused_reads = 0  # how the cache has been read so far
        self._length = 0
        self._ring_from = 0  # the first position whose row as it came is still in the ring
        self.store = None

    @property
    def length(self):
        return self._length

    @length.setter
    def length(self, value):
        """More tokens were stored (here, or by a decoder that writes through `store`)."""
        self._length = value
        self._ring_from = max(self._ring_from, (value // self.block_tokens - 1) * self.block_tokens)

    def lazy_initialization(self, key_states, value_states):
        if not key_states.is_cuda:
            raise RuntimeError("the quantized KV cache needs CUDA tensors: there is no CPU fallback")
        native.library()
        self.dtype, self.device = key_states.dtype, key_states.device
        self.batch, self.heads, _, self.head_dim = key_states.shape
        self._allocate(self.max_cache_len or 256)
        self.is_initialized = True

    def _allocate(self, tokens):
        old = self.store
        self.store = BlockKVStore.allocate(self.batch, self.heads, self.head_dim, tokens, self.block_tokens, self.dtype,
                                           self.device)
        if old is not None:  # each sequence's pages are its own and in order
            for name in ("k_pages", "v_pages", "k_scales", "v_scales"):
                dst, src = getattr(self.store, name), getattr(old, name)
                dst.unflatten(0, (self.batch, -1))[:, : old.max_blocks] = src.unflatten(0, (self.batch, -1))
            self.store.k_ring, self.store.v_ring = old.k_ring, old.v_ring
            self.store = BlockKVStore(*(getattr(self.store, n) for n in (
                "k_pages", "v_pages", "k_scales", "v_scales", "k_ring", "v_ring", "table")))

    @property
    def capacity(self):
        return 0 if self.store is None else (self.max_cache_len or self.store.capacity)

    def append(self, key_states, value_states):
        """Store new tokens of every sequence; returns nothing."""
        if not self.is_initialized:
            self.lazy_initialization(key_states, value_states)
        need = self.length + key_states.shape[-2]
        if need > self.capacity:
            if self.max_cache_len is not None:
                raise RuntimeError(f"KV cache of {self.max_cache_len} tokens cannot take {need}")
            self._allocate(max(need, 2 * self.capacity))
        self.store.append(key_states, value_states, self.length)
        self.length = need

    def dequantized(self, length=None):
        """(K, V) in the model dtype, [B, H, length, D]."""
        self.dequant_calls += 1
        return self.store.read(self.length if length is None else length, self.length)

    def update(self, key_states, value_states, *args, **kwargs):
        self.append(key_states, value_states)
        if not self.fused_read:
            return self.dequantized()
        # Stand-ins of the right shape, tagged so that int_kv_attention knows what it was given. Codes, not rows
        # of the model's dtype: an attention function that takes them for keys and values fails on the type.
        shape = (self.batch, self.heads, self.length, self.head_dim)
        k, v = (p[:1, :, :1].expand(shape) for p in (self.store.k_pages, self.store.v_pages))
        k.lq_layer = v.lq_layer = self
        return k, v

    def attend(self, q, scaling):
        """Attention of the newest rows q [B, tokens, Hq, D] over the cache, [B, tokens, Hq, D]."""
        self.fused_reads += 1
        return self.store.attend(q, self.length - q.shape[1], scaling=scaling)

    def get_mask_sizes(self, query_length: int):
        return self.get_seq_length() + query_length, 0

    def get_seq_length(self) -> int:
        return self.length

    def get_max_cache_shape(self) -> int:
        return self.max_cache_len if self.max_cache_len is not None else -1

    def reset(self):
        self._length = self._ring_from = 0

    def crop(self, max_length: int):
        """Forget the tokens behind `max_length`. Within the ring (the incomplete block and the one before
        it) nothing is lost; further back the rows of the block that becomes the incomplete one are
        the values its codes stand for."""
        if max_length < 0:
            max_length = self.length - abs(max_length)
        length = min(self.length, max(max_length, 0))
        first = length - length % self.block_tokens
        if first < self._ring_from:
            if first < length:
                slots = torch.arange(first, length, device=self.device) % (2 * self.block_tokens)
                for ring, values in zip((self.store.k_ring, self.store.v_ring), self.store.read(length, self.length)):
                    ring[:, :, slots] = values[:, :, first:]
            self._ring_from = first
        self._length = length

    def offload(self):
        pass

    def prefetch(self):
        pass

    def reorder_cache(self, beam_idx):
        if self.length:
            idx = beam_idx.to(self.device)
            for name in ("k_pages", "v_pages", "k_scales", "v_scales"):
                t = getattr(self.store, name)
                t.copy_(t.unflatten(0, (self.batch, -1)).index_select(0, idx).flatten(0, 1))
            for t in (self.store.k_ring, self.store.v_ring):
                t.copy_(t.index_select(0, idx))


class BlockKVCache(Cache):
    """`Cache` whose layers hold 8-bit codes with one scale per block of tokens and KV head."""

    num_bits = 8

    def __init__(self, block_tokens: int = 64, max_cache_len=None, fused_read: bool = False):
        if block_tokens not in BLOCK_TOKENS:
            raise ValueError(f"a block must be one of {BLOCK_TOKENS} tokens, got {block_tokens}")
        super().__init__(layer_class_to_replicate=functools.partial(BlockKVLayer, block_tokens, max_cache_len, fused_read))
        self.block_tokens = block_tokens
        self.capacity_limit = max_cache_len
        self.fused_read = fused_read

    def crop(self, max_length: int):
        for layer in self.layers:
            layer.crop(max_length)


# Query tokens up to which `int_kv_attention` reads the codes; longer ones read the cache back once and take
# transformers' SDPA. With several tokens that can only be a prompt on an empty cache (chunks on top of
# cached tokens come with a mask, which the codes' kernels do not take). There a call takes 16 us by the
# codes and 36 read back, the host's part of both, for 2 to 16 tokens of 1 and 8 sequences, 32 query
# heads of 128 or 64 on 8, 16 on 2 and 8 on 8; the GPU itself needs 6 to 17 us by the codes and 4 to 6
# read back, and from 128 tokens of 8 sequences (512 of one) on the codes lose the call as well: 54 against 37 us.
ATTEND_TOKENS = 16


def attend_layer(layer, module, query, attention_mask, dropout, scaling, kwargs):
    """What `int_kv_attention` does with a `BlockKVLayer`: (output, None), or None where the kernel does
    not serve the call (a mask, dropout, a window, a long chunk, another dtype)."""
    heads, tokens = query.shape[1], query.shape[2]
    if attention_mask is not None or dropout or kwargs.get("sliding_window") is not None or tokens > ATTEND_TOKENS:
        return None
    if query.dtype != layer.dtype or layer.dtype == torch.float32 or heads % layer.heads:
        return None
    if tokens > 1 and not kwargs.get("is_causal", getattr(module, "is_causal", True)):
        return None
    return layer.attend(query.transpose(1, 2), layer.head_dim ** -0.5 if scaling is None else scaling), None
