"""Which attentions the fused decoder takes: norms of queries and keys are recognised by what they compute,
and an attention with parts that the decoder does not know is left to its own module."""

import pytest
import torch
from transformers.models.llama.configuration_llama import LlamaConfig
from transformers.models.llama.modeling_llama import LlamaAttention, LlamaRMSNorm

from llmquant_b200.runtime import decoder

DIM = 64


class PlusOne(torch.nn.Module):
    """x * rsqrt(mean(x^2) + eps) * (1 + weight)"""

    def __init__(self, dim, eps=1e-6):
        super().__init__()
        self.eps = eps
        self.weight = torch.nn.Parameter(torch.zeros(dim))

    def forward(self, x):
        y = x.float()
        return (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + self.eps) * (1.0 + self.weight.float())).to(x.dtype)


class Clamped(LlamaRMSNorm):
    """eps as a lower bound of the root, not under it"""

    def forward(self, x):
        y = x.float()
        return (y / y.square().mean(-1, keepdim=True).sqrt().clamp_min(self.variance_epsilon)).to(x.dtype) * self.weight


class Late(LlamaRMSNorm):
    def forward(self, x):
        raise RuntimeError("takes something else")


def attention(q_norm, k_norm, dtype=torch.bfloat16):
    attn = LlamaAttention(LlamaConfig(hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=DIM), 0)
    attn.q_norm, attn.k_norm = q_norm, k_norm
    return attn.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("eps", [1e-6, 1e-5, 1e-3])
def test_rms_norms_are_taken(dtype, eps):
    norms = [LlamaRMSNorm(DIM, eps=eps) for _ in range(2)]
    for i, norm in enumerate(norms):
        norm.weight.data = torch.randn(DIM, generator=torch.Generator().manual_seed(i)) * 2
    attn = attention(*norms, dtype)
    q, k, got = decoder._head_norms(attn, DIM)
    assert got == eps and torch.equal(q, norms[0].weight.data.bfloat16()) and torch.equal(k, norms[1].weight.data.bfloat16())
    assert decoder._plain_attention(attn)
    torch_norms = [torch.nn.RMSNorm(DIM, eps=eps) for _ in range(2)]
    assert decoder._head_norms(attention(*torch_norms, dtype), DIM)[2] == eps


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("make", [torch.nn.LayerNorm, PlusOne, Clamped, Late], ids=lambda c: c.__name__)
def test_norms_of_another_kind_are_not(make, dtype):
    rms = LlamaRMSNorm(DIM)
    for pair in ((make(DIM), make(DIM)), (rms, make(DIM)), (make(DIM), rms)):
        for norm in pair:
            if hasattr(norm, "variance_epsilon"):
                norm.variance_epsilon = 1e-6
            elif hasattr(norm, "eps"):
                norm.eps = 1e-6
        with pytest.raises(ValueError, match="RMS norms|do not compute"):
            decoder._head_norms(attention(*pair, dtype), DIM)


def test_none_missing_and_different_norms():
    attn = attention(None, None)
    assert decoder._head_norms(attn, DIM) is None and decoder._plain_attention(attn)
    for pair in ((LlamaRMSNorm(DIM), None), (LlamaRMSNorm(2 * DIM), LlamaRMSNorm(2 * DIM)),
                 (LlamaRMSNorm(DIM, eps=1e-5), LlamaRMSNorm(DIM, eps=1e-6)), (torch.nn.Identity(), torch.nn.Identity())):
        with pytest.raises(ValueError):
            decoder._head_norms(attention(*pair), DIM)


def test_an_attention_with_other_parts_is_not_plain():
    """Norms behind the rotation under names of their own, parameters (sinks), gates."""
    attn = attention(None, None)
    attn.query_layernorm, attn.key_layernorm = LlamaRMSNorm(DIM), LlamaRMSNorm(DIM)
    assert not decoder._plain_attention(attn)
    attn = attention(None, None)
    attn.sinks = torch.nn.Parameter(torch.zeros(4))
    assert not decoder._plain_attention(attn)
    attn = attention(None, None)
    attn.register_buffer("gate", torch.zeros(4))
    assert not decoder._plain_attention(attn)
    attn = attention(None, None)
    attn.dropout, attn.rotary_emb = torch.nn.Dropout(0.1), torch.nn.Identity()
    assert decoder._plain_attention(attn)
