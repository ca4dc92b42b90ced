"""What `graphed_generate` refuses before it touches a device."""

import pytest
import torch

from llmquant_b200.runtime import graphed_generate


def test_block_tokens_without_the_integer_cache():
    """They choose among the 8-bit caches: without one they would be left out."""
    model, ids = torch.nn.Linear(2, 2), torch.zeros(1, 3, dtype=torch.long)
    with pytest.raises(ValueError, match="give kv_cache_bits=8"):
        graphed_generate(model, ids, 4, kv_block_tokens=64)
    model.__dict__["_graph_kv_cache_bits"] = 4  # what can_graph was asked about last
    with pytest.raises(ValueError, match="holds 8 bits"):
        graphed_generate(model, ids, 4, kv_block_tokens=64)
    with pytest.raises(ValueError, match="one of"):
        graphed_generate(model, ids, 4, kv_cache_bits=8, kv_block_tokens=48)
