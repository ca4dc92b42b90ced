"""The block-scaled cache where models meet it: behind transformers' `Cache`, in `generate`, in the
fused decoder (graphed and eager), and the norms of queries and keys in a model that has them."""

import pytest
import torch

from gpu_util import rel_l2, seeded
from llmquant_b200.core import QuantConfig, oneshot
from llmquant_b200.quantizers import BlockKVCache, BlockKVStore, make_cache_factory
from test_gpu_block_kv import Model, check_state, close_to

pytestmark = pytest.mark.gpu


def _tiny(normed=False, **kw):
    """A tiny kernel-mode Llama; `normed`: its attention normalises queries and keys for each head."""
    from oracle.real_mode import tiny_llama

    model = tiny_llama(seed=0, **kw)
    if normed:
        from transformers.models.llama import modeling_llama as llama

        class NormedAttention(llama.LlamaAttention):
            def __init__(self, config, layer_idx):
                super().__init__(config, layer_idx)
                self.q_norm = llama.LlamaRMSNorm(self.head_dim, eps=config.rms_norm_eps)
                self.k_norm = llama.LlamaRMSNorm(self.head_dim, eps=config.rms_norm_eps)

            def forward(self, hidden_states, position_embeddings, attention_mask, past_key_values=None, **kwargs):
                shape = (*hidden_states.shape[:-1], -1, self.head_dim)
                q = self.q_norm(self.q_proj(hidden_states).view(shape)).transpose(1, 2)
                k = self.k_norm(self.k_proj(hidden_states).view(shape)).transpose(1, 2)
                v = self.v_proj(hidden_states).view(shape).transpose(1, 2)
                q, k = llama.apply_rotary_pos_emb(q, k, *position_embeddings)
                if past_key_values is not None:
                    k, v = past_key_values.update(k, v, self.layer_idx)
                attend = llama.ALL_ATTENTION_FUNCTIONS.get_interface(self.config._attn_implementation,
                                                                     llama.eager_attention_forward)
                out, weights = attend(self, q, k, v, attention_mask, dropout=0.0, scaling=self.scaling, **kwargs)
                return self.o_proj(out.reshape(*hidden_states.shape[:-1], -1).contiguous()), weights

        g = torch.Generator().manual_seed(5)
        for i, layer in enumerate(model.model.layers):
            attn = NormedAttention(model.config, i).to(torch.bfloat16)
            attn.load_state_dict(layer.self_attn.state_dict(), strict=False)
            for norm in (attn.q_norm, attn.k_norm):
                # small heads would leave softmax nearly flat without the norms: weights of 1 .. 3 sharpen it
                norm.weight.data = (torch.rand(norm.weight.shape, generator=g) * 2 + 1).to(torch.bfloat16)
            layer.self_attn = attn
    cfg = QuantConfig(attn_weight="int8", mlp_weight="int4", head_weight="int8", kv_cache="int8")
    return oneshot(model.cuda(), cfg.to_modifier(mode="kernel"))


@pytest.mark.parametrize("block", [16, 64])
def test_cache_class_grows_crops_and_reorders(block):
    cache = make_cache_factory(8, block_tokens=block)()
    assert isinstance(cache, BlockKVCache) and cache.num_bits == 8 and cache.block_tokens == block
    chunks = [seeded((2, 3, n, 64), n).bfloat16().cuda() for n in (200, 1, 99, 300)]
    model = Model(2, 3, 64, block, torch.bfloat16)
    at = 0
    for c in chunks:
        k, v = cache.update(c, -c, 0)
        for b in range(2):
            model.put(b, c[b], -c[b], at)
        at += c.shape[2]
        assert cache.get_seq_length() == at and k.shape == (2, 3, at, 64)
    layer = cache.layers[0]
    check_state(layer.store, model, [at, at])
    for b in range(2):
        close_to(k[b], model.values(model.k[b]), torch.bfloat16, 2.0 ** -24)
        close_to(v[b], model.values(model.v[b]), torch.bfloat16, 2.0 ** -24)
    # within the ring: nothing lost
    cache.crop(at - block)
    for b in range(2):
        model.put(b, chunks[0][b, :, :5], chunks[0][b, :, 5:10], at - block)
    cache.update(chunks[0][:, :, :5], chunks[0][:, :, 5:10], 0)
    check_state(layer.store, model, [at - block + 5] * 2, (at // block - 1) * block)
    # far back, then further by one token at a time over a block's border: the rows are the codes' values
    keep = 3 * block + 7 if block == 16 else 2 * block + 7
    k, v = layer.dequantized()
    cache.crop(keep)
    for n in (keep, keep - 7, keep - 8):
        cache.crop(n)
        got = layer.dequantized()
        assert torch.equal(got[0], k[:, :, :n]) and torch.equal(got[1], v[:, :, :n])
    cache.crop(-1)
    assert cache.get_seq_length() == keep - 9
    cache.layers[0].reorder_cache(torch.tensor([1, 1]))
    got = layer.dequantized()
    assert torch.equal(got[0], k[[1, 1], :, :keep - 9]) and torch.equal(got[1], v[[1, 1], :, :keep - 9])
    layer.reset()
    assert cache.get_seq_length() == 0
    k, _ = cache.update(chunks[1], chunks[1], 0)
    assert torch.equal(k, chunks[1])
    fixed = BlockKVCache(32, max_cache_len=40)
    fixed.update(chunks[0][:, :, :30], chunks[0][:, :, :30], 0)
    with pytest.raises(RuntimeError, match="cannot take"):
        fixed.update(chunks[0][:, :, :11], chunks[0][:, :, :11], 0)


def test_factory_refusals():
    with pytest.raises(ValueError, match="holds 8 bits"):
        make_cache_factory(4, block_tokens=64)
    with pytest.raises(ValueError, match="one of"):
        make_cache_factory(8, block_tokens=48)
    with pytest.raises(ValueError, match="one of"):
        BlockKVCache(8)
    assert make_cache_factory(None, block_tokens=64) is None


@pytest.mark.parametrize("batch", [1, 3])
@pytest.mark.parametrize("kw", [dict(head_dim=64), dict(head_dim=128, hidden=512, inter=1024)])
def test_generate_reads_the_codes(kw, batch):
    """transformers' `generate`: the prompt reads the cache back once, decode steps and short chunks read
    the codes, and the logits agree with the route that reads the cache back every time."""
    model = _tiny(**kw)
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(0, 512, (batch, 90), generator=g).cuda()
    factory = make_cache_factory(8, model=model, block_tokens=32)
    cache, new = factory(), 10
    assert cache.fused_read
    out = model.generate(ids, attention_mask=torch.ones_like(ids), max_new_tokens=new, do_sample=False, pad_token_id=0,
                         past_key_values=cache)
    assert out.shape == (batch, 90 + new)
    layers = len(model.model.layers)
    assert [x.dequant_calls for x in cache.layers] == [1] * layers
    assert [x.fused_reads for x in cache.layers] == [new - 1] * layers
    a, b = factory(), make_cache_factory(8, block_tokens=32)()
    with torch.no_grad():
        for lo, hi in ((0, 90), *((i, i + 1) for i in range(90, 99))):
            la = model(out[:, lo:hi], past_key_values=a, use_cache=True).logits[:, -1]
            lb = model(out[:, lo:hi], past_key_values=b, use_cache=True).logits[:, -1]
            assert rel_l2(la.float().cpu().numpy(), lb.float().cpu().numpy()) <= 1e-2, lo
    assert b.layers[0].fused_reads == 0
    assert torch.equal(a.layers[0].dequantized()[0], b.layers[0].dequantized()[0])


def test_padded_batch_takes_the_masked_route():
    """Left padding needs a mask, which the kernel does not take: the cache is read back, and a padded
    sequence gives what it gives alone."""
    model = _tiny(head_dim=64)
    g = torch.Generator().manual_seed(6)
    ids = torch.randint(1, 512, (2, 40), generator=g).cuda()
    mask = torch.ones_like(ids)
    mask[0, :13] = 0
    cache = make_cache_factory(8, model=model, block_tokens=64)()
    with torch.no_grad():
        both = model(ids, attention_mask=mask, past_key_values=cache, use_cache=True,
                     position_ids=(mask.cumsum(1) - 1).clamp_min(0)).logits[0, -1]
        step = model(ids[:, :1], attention_mask=torch.cat((mask, mask[:, -1:]), 1), past_key_values=cache, use_cache=True,
                     position_ids=mask.sum(1, keepdim=True)).logits[0, -1]
        alone_cache = make_cache_factory(8, model=model, block_tokens=64)()
        alone = model(ids[:1, 13:], past_key_values=alone_cache, use_cache=True).logits[0, -1]
        alone_step = model(ids[:1, :1], past_key_values=alone_cache, use_cache=True).logits[0, -1]
    assert cache.layers[0].fused_reads == 0
    # 40 tokens: one incomplete block, so both hold the same rows as they came
    assert rel_l2(both.float().cpu().numpy(), alone.float().cpu().numpy()) <= 2e-2
    assert rel_l2(step.float().cpu().numpy(), alone_step.float().cpu().numpy()) <= 2e-2


@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("batch", [1, 3, 9])
@pytest.mark.parametrize("kw", [dict(head_dim=64), dict(head_dim=128, hidden=512, inter=1024)])
def test_fused_decoder_on_the_block_cache(kw, batch, normed):
    """Teacher-forced against the module path with the same cache class; graphed and eager alike; the
    stored state is what the modules stored."""
    from llmquant_b200.runtime.decoder import FusedLlamaDecoder, supports

    model = _tiny(normed, **kw)
    assert supports(model)
    g = torch.Generator().manual_seed(7)
    ids = torch.randint(0, 512, (batch, 75), generator=g).cuda()
    prompt = 50
    # 2e-2 is what the routes of the linears differ by (their own tests' bound). With the norms the modules
    # round a query or key to bf16 after the norm, after its weight, twice in the rotation and once at
    # its end, and take bf16 angles: six roundings of 2^-8 / sqrt(3) * 0.72 = 1.6e-3 rms, where the
    # kernel rounds once: sqrt(2 * (6 + 1)) * 1.6e-3 = 6.1e-3 of each product q_i k_i. The weights (1 .. 3, mean
    # square 4.3) make the products 4.3 rms and a score's error 6.1e-3 * 4.3 * sqrt(D) / sqrt(D) = 0.026,
    # which is the relative error of a softmax weight and so, rms, of an attention output; two
    # layers of it, uncorrelated: 0.037.
    bound = 2e-2 + (0.037 if normed else 0.0)
    kv_block = None if normed else 32  # (a model with the norms takes the block cache by itself)
    dec = FusedLlamaDecoder(model, batch, 128, use_graph=False, kv_block=kv_block)
    assert dec.kv_block == (64 if normed else 32)
    cache = make_cache_factory(8, block_tokens=dec.kv_block)()
    with torch.no_grad():
        model(ids[:, :prompt], past_key_values=cache, use_cache=True)
        dec.prefill(ids[:, :prompt])
        for i in range(prompt, 75):
            dec.tokens.copy_(ids[:, i])
            dec.step()
            want = model(ids[:, i:i + 1], past_key_values=cache, use_cache=True).logits[:, -1]
            err = rel_l2(dec.logits.float().cpu().numpy(), want.float().cpu().numpy())
            assert err <= bound, (i, err)
    dec.check_device_errors()
    for layer, ref in zip(dec.cache.layers, cache.layers):
        layer.length = 75
        for a, b in zip(layer.dequantized(), ref.dequantized()):
            assert rel_l2(a.float().cpu().numpy(), b.float().cpu().numpy()) <= bound
    streams = []
    for use_graph in (False, True):
        dec = FusedLlamaDecoder(model, batch, 128, use_graph=use_graph, kv_block=kv_block)
        streams.append(dec.generate(ids[:, :prompt], 40))
    assert torch.equal(*streams)


def test_entry_points_choose_the_block_cache():
    from llmquant_b200.runtime import can_graph, graphed_generate
    from llmquant_b200.runtime.decoder import FusedLlamaDecoder, supports

    model = _tiny(head_dim=64)
    ids = torch.randint(0, 512, (2, 20), generator=torch.Generator().manual_seed(8)).cuda()
    want = FusedLlamaDecoder(model, 2, 20 + 12 + 1, kv_block=16).generate(ids, 12)
    assert torch.equal(graphed_generate(model, ids, 12, kv_cache_bits=8, kv_block_tokens=16), want)
    assert can_graph(model, make_cache_factory(8, block_tokens=16))
    assert torch.equal(graphed_generate(model, ids, 12), want)
    assert can_graph(model, make_cache_factory(8))  # the cache with a scale per token again
    assert torch.equal(graphed_generate(model, ids, 12), FusedLlamaDecoder(model, 2, 33).generate(ids, 12))
    normed = _tiny(True, head_dim=64)
    assert torch.equal(graphed_generate(normed, ids, 12, kv_cache_bits=8),
                       FusedLlamaDecoder(normed, 2, 33, kv_block=64).generate(ids, 12))
    with pytest.raises(ValueError, match="holds 8 bits"):
        FusedLlamaDecoder(normed, 2, 33, kv_bits=4)
    assert can_graph(normed, make_cache_factory(8)) and not can_graph(normed, make_cache_factory(4))
    normed.model.layers[0].self_attn.q_norm = torch.nn.Identity()
    assert not supports(normed)  # norms of another kind: not served rather than left out
    assert isinstance(BlockKVStore.allocate(1, 1, 64, 1), BlockKVStore)
