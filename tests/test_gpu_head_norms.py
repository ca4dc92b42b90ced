"""Models whose attention normalises queries and keys for each head, in the fused decoder: on the cache that
the caller names, and not at all when the norms are of another kind."""

import pytest
import torch

from gpu_util import rel_l2
from llmquant_b200.quantizers import BlockKVCache, KernelQuantCache, make_cache_factory
from llmquant_b200.runtime import can_graph, graphed_generate
from llmquant_b200.runtime.decoder import FusedLlamaDecoder, supports
from test_gpu_block_kv_model import _tiny

pytestmark = pytest.mark.gpu


def ids_of(batch, tokens, seed=7):
    return torch.randint(0, 512, (batch, tokens), generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.fixture
def caches(monkeypatch):
    """The caches of the decoders that generated."""
    seen, generate = [], FusedLlamaDecoder.generate

    def spy(self, *args):
        seen.append(self.cache)
        return generate(self, *args)

    monkeypatch.setattr(FusedLlamaDecoder, "generate", spy)
    return seen


@pytest.mark.parametrize("normed", [True, False])
@pytest.mark.parametrize("block", [None, 16])
def test_the_cache_that_was_named_is_the_one_decoded_on(caches, normed, block):
    model, ids = _tiny(normed, head_dim=64), ids_of(2, 70)
    want = FusedLlamaDecoder(model, 2, 111, kv_block=block or 0).generate(ids, 40)
    factory = make_cache_factory(8, block_tokens=block)
    assert can_graph(model, factory)
    assert torch.equal(graphed_generate(model, ids, 40), want)
    assert torch.equal(graphed_generate(model, ids, 40, kv_cache_bits=8, kv_block_tokens=block), want)
    kind = KernelQuantCache if block is None else BlockKVCache
    assert [type(c) for c in caches] == [kind] * 3 and all(getattr(c, "block_tokens", None) == block for c in caches)
    assert type(factory()) is kind


@pytest.mark.parametrize("batch", [1, 3, 9])
@pytest.mark.parametrize("kw", [dict(head_dim=64), dict(head_dim=128, hidden=512, inter=1024)])
def test_head_norms_on_the_cache_with_a_scale_per_token(kw, batch):
    """Teacher-forced against the module path with the same cache class; graphed and eager alike."""
    model, ids, prompt = _tiny(True, **kw), ids_of(batch, 75), 50
    # As on the block-scaled cache the routes of the linears differ by 2e-2, and a query or key by seven roundings
    # of bf16, sqrt(7) * 1.6e-3 = 4.3e-3 rms of its size (3.4e-3 on average). But here every key is a code at once
    # (there the newest rows stay as they came): keys that differ by delta get codes one step apart with
    # probability |delta| / step, so what is read differs by sqrt(E|delta| * step) rms. A step is the largest of 64
    # or 128 values over 127; with weights of 1 .. 3 that is 3.3 times their rms, a step 0.026 of it and the
    # difference sqrt(3.4e-3 * 0.026) = 9.4e-3. Products q_i k_i then differ by sqrt(4.3^2 + 9.4^2) * 1e-3 = 1.03e-2
    # instead of 6.1e-3, a softmax weight by 1.03e-2 * 4.3 = 0.044, two layers uncorrelated by 0.063.
    bound = 2e-2 + 0.063
    dec = FusedLlamaDecoder(model, batch, 128, use_graph=False, kv_block=0)
    assert dec.kv_block is None and isinstance(dec.cache, KernelQuantCache)
    cache = make_cache_factory(8)()
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
    streams = [FusedLlamaDecoder(model, batch, 128, use_graph=g, kv_block=0).generate(ids[:, :prompt], 40) for g in (False, True)]
    assert torch.equal(*streams)


def test_other_bits_are_refused():
    model = _tiny(True, head_dim=64)
    for block in (None, 0, 64):
        with pytest.raises(ValueError, match="holds 8 bits"):
            FusedLlamaDecoder(model, 1, 33, kv_bits=4, kv_block=block)
    assert not can_graph(model, make_cache_factory(4))


def test_norms_of_another_kind_and_strange_parts_are_not_served():
    model = _tiny(True, head_dim=64)
    assert supports(model)
    attn = model.model.layers[0].self_attn
    good = attn.q_norm
    attn.q_norm = torch.nn.LayerNorm(64, eps=good.variance_epsilon).to("cuda", torch.bfloat16)
    assert not supports(model) and not can_graph(model, make_cache_factory(8))
    attn.q_norm = good
    assert supports(model)
    attn.query_layernorm = torch.nn.LayerNorm(64).to("cuda", torch.bfloat16)
    assert not supports(model)


@pytest.mark.parametrize("block", [0, 64])
def test_a_position_without_angles_is_reported(block):
    """A decoder stepped behind its last position: heads without angles, said by the check after the step."""
    model = _tiny(True, head_dim=64)
    dec = FusedLlamaDecoder(model, 1, 64, use_graph=False, kv_block=block)
    dec.start_empty(ids_of(1, 1)[:, 0])
    dec.step()
    dec.check_device_errors()
    dec.cos_half, dec.sin_half = dec.cos_half[:1].contiguous(), dec.sin_half[:1].contiguous()
    dec.step()  # position 1
    with pytest.raises(RuntimeError, match="head norms"):
        dec.check_device_errors()
    dec.check_device_errors()
