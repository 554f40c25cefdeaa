"""What a model over 4-bit pages refuses, and that it does before anything runs."""
import pytest
import torch

from src.config import KVEviction, ModelConfig
from src.inference.generate_with_cache import generate_with_cache
from src.model.transformer import TinyTransformerLM
from src.serving.continuous_generate import StepExecutor

EVICTION = KVEviction(limit=30, keep=20, window=8)


def _model(d_model=128, heads=2, **kw):
    return TinyTransformerLM(vocab_size=50, d_model=d_model, num_heads=heads, num_layers=1, d_ff=64, max_seq_len=96,
                             attention_backend="paged_reference", kv_pool_initial_blocks=2, **kw).eval()


@pytest.mark.parametrize("d_model, heads", [(64, 2), (160, 2), (512, 2)])
def test_head_dims_without_4_bit_pages(d_model, heads):
    with pytest.raises(ValueError, match="head_dim 64 or 128"):
        _model(d_model, heads, kv_cache_dtype="int4")
    _model(d_model, heads)  # (other pools hold any)


def test_block_sizes_without_4_bit_pages():
    with pytest.raises(ValueError, match="16 tokens"):
        _model(kv_cache_dtype="int4", kv_block_size=32)
    for d_model, heads in ((128, 2), (128, 1)):
        _model(d_model, heads, kv_cache_dtype="int4", kv_block_size=16)


def test_the_defaults_take_4_bit_pages():
    c = ModelConfig()
    assert c.d_model // c.num_heads in (64, 128) and c.kv_block_size == 16


@pytest.mark.parametrize("kind", [{}, {"kv_cache_dtype": "int4"}])
def test_eviction_needs_weights_from_the_start(kind):
    """A model that keeps no attention weights refuses a run with eviction before it takes a block."""
    model = _model(**kind)
    with pytest.raises(ValueError, match="track_attention_weights"):
        generate_with_cache(model, torch.zeros(2, 40, dtype=torch.long), [4, 4], eviction=EVICTION)
    assert model.paged_memory_stats()["allocated_kv_block_bytes"] == 0
    with pytest.raises(ValueError, match="track_attention_weights"):
        StepExecutor(model, "cpu", eviction=EVICTION)
    StepExecutor(model, "cpu")
