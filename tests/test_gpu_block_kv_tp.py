"""The block-scaled cache under tensor parallelism, all ranks on one GPU: launches in lock step on one stream,
so that no kernel waits for one that has not been launched (as in the tests of the folded step)."""

import pytest
import torch

from gpu_util import rel_l2
from llmquant_b200.core import QuantConfig, oneshot
from llmquant_b200.runtime import tp
from llmquant_b200.runtime.decoder import FusedLlamaDecoder
from llmquant_b200.runtime.tp import PeerExchange
from test_gpu_tp_folded import _lockstep

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("normed,block", [(False, 16), (False, 64), (True, 16), (True, 0)])
@pytest.mark.parametrize("world", [2, 4])
def test_folded_decode_on_the_block_cache(world, normed, block):
    """A seeded tiny Llama split over the ranks, from an empty cache over four blocks, against the one-GPU
    decoder on the same cache: every rank holds its heads' share of the same blocks."""
    from oracle.real_mode import tiny_llama
    from transformers.models.llama.modeling_llama import LlamaRMSNorm

    kw = dict(head_dim=128, hidden=512, inter=1024, heads=4, kv_heads=4)
    quant = QuantConfig(attn_weight="int8", mlp_weight="int4", head_weight="int8", kv_cache="int8")

    def model(ctx=None):
        m = tiny_llama(seed=0, **kw)
        if normed:  # (the decoder takes them from the attention; its module is not run here)
            for i, layer in enumerate(m.model.layers):
                for j, name in enumerate(("q_norm", "k_norm")):
                    norm = LlamaRMSNorm(128, eps=1e-5).to(torch.bfloat16)
                    norm.weight.data = (torch.rand(128, generator=torch.Generator().manual_seed(2 * i + j)) + 1).bfloat16()
                    setattr(layer.self_attn, name, norm)
        if ctx is not None:
            m = tp.shard_linears_(m, ctx)
        m = m.cuda()
        oneshot(m, quant.to_modifier(mode="kernel"))
        return m

    batch, total = 2, 66
    ids = torch.randint(0, 512, (batch, total), generator=torch.Generator().manual_seed(3)).cuda()
    single = FusedLlamaDecoder(model(), batch, total + 2, use_graph=False, kv_block=block)
    exs = PeerExchange.on_one_device(world, batch, kw["hidden"], torch.device("cuda"))
    decs = []
    for r in range(world):
        ctx = tp.TPContext(r, world)
        decs.append(FusedLlamaDecoder(model(ctx), batch, total + 2, use_graph=False, tp=ctx, exchange=exs[r], kv_block=block))
        assert decs[-1].launches_per_step == single.launches_per_step and decs[-1].kv_block == (block or None)
    for d in [single] + decs:
        d.start_empty(ids[:, 0])
    for s in range(total - 1):
        for d in [single] + decs:
            d.tokens.copy_(ids[:, s])
        single.step()
        logits = _lockstep(decs)
        # the bound of the folded step's own comparison with one GPU (the order of the split sums)
        assert rel_l2(logits.float().cpu().numpy(), single.logits.float().cpu().numpy()) <= 1e-2, s
    heads = kw["kv_heads"] // world
    for i, whole in enumerate(single.cache.layers):
        whole.length = total - 1
        for r, d in enumerate(decs):
            mine = d.cache.layers[i]
            mine.length = total - 1
            assert mine.heads == heads
            for a, b in zip(mine.dequantized(), whole.dequantized()):
                want = b[:, r * heads:(r + 1) * heads]
                # rows that differ by delta (rms up to 1e-2 of their size, as the logits; 0.8e-2 on average) get codes
                # one step apart with probability |delta| / step: sqrt(0.8e-2 * step) rms. A step is the largest of
                # up to 8192 values over 127, about 5 times their rms: 0.04, and so 1.8e-2.
                assert rel_l2(a.float().cpu().numpy(), want.float().cpu().numpy()) <= 1.8e-2
    single.check_device_errors()
