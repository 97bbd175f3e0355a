"""Bytes of a cached token as the native configuration counts them: those of the cache that the runtime builds."""
import json

import pytest

from tensorrt_edge_llm_b200.checkpoint.artifacts import runtime_config_dict
from tensorrt_edge_llm_b200.config import QuantConfig, tiny_llama_config
from tensorrt_edge_llm_b200.runtime import native as rt
from tensorrt_edge_llm_b200.runtime.kv_cache import KVCacheManager


@pytest.mark.parametrize("head,page,shared,four", [(64, 64, 0, True), (128, 16, 0, True), (32, 64, 0, False), (64, 48, 0, False), (64, 8, 0, False), (128, 64, 1, False)])
def test_four_bit_pages_that_give_way_count_as_the_compute_type(head, page, shared, four):
    """A checkpoint names four-bit pages; heads, pages and stacks that cannot have them keep 16 bits."""
    cfg = tiny_llama_config(num_hidden_layers=3, vocab_size=256, dtype="bfloat16", head_dim=head, num_attention_heads=4, num_key_value_heads=2, hidden_size=128,
                            quant=QuantConfig(kv_cache_quant="nvfp4"))
    if shared:
        cfg.num_kv_shared_layers = shared
    c = rt.LLMEngineConfig.from_runtime_config(json.dumps(runtime_config_dict(cfg, 4, 64, 128, 1), default=str))
    c.kv_page_size = page
    kv = KVCacheManager(cfg, num_pages=2, page_size=page, max_seats=1, max_pages_per_seq=2)
    assert kv.kv_fp4 == four and c.kv_bytes_per_token() == (3 - shared) * 2 * 2 * (head * 9 // 16 if four else 2 * head)
    if not shared:              # the pool of a stack with shared layers keeps their rows too
        assert c.kv_bytes_per_token() == kv.bytes_per_token
