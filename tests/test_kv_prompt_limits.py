"""Lengths that the prompt calls of the kv_* family take, without a GPU."""
import pytest

from raftinfer_b200 import kernels as K


def test_a_chunk_that_no_launch_holds_is_refused_before_anything_is_enqueued():
    """A context may have 2^23 tokens, a launch 65535 tiles of 128: the sizes and the calls agree."""
    most = 65535 * 128
    shape = lambda tokens, past=0: K.Qwen35AttentionShape(tokens, 16, 4, 256, 2 ** 23, past)
    row = 2 * 4 * 256 * 2
    assert K.kv_prefill_workspace_bytes(shape(most), 0, 0, K.KV_E4M3) == most * row
    assert K.kv_prefill_workspace_bytes(shape(most, 128), 0, 0, K.KV_E4M3) == 2 ** 23 * row
    common = dict(query=16, key=16, value=16, gate=16, output=16, workspace=16, workspace_bytes=1 << 50, window_tokens=0,
                  sink_tokens=0, activation_dtype=K.DTYPE_BF16, stream=16)
    for tokens in (most + 1, 2 ** 23):
        for kind in (K.KV_BF16, K.KV_E4M3):
            for call in (lambda: K.kv_prefill_workspace_bytes(shape(tokens), 0, 0, kind),
                         lambda: K.kv_attention_prefill(**common, kv_cache=16, kv_cache_bytes=1 << 50, shape=shape(tokens),
                                                        cache_dtype=kind),
                         lambda: K.kv_paged_prefill(**common, page_pool=16, pool_pages=9, block_table=16, max_blocks=2 ** 15,
                                                    shape=shape(tokens), cache_dtype=kind)):
                with pytest.raises(K.Qwen35PrimitiveError, match="65535") as refusal:
                    call()
                assert refusal.value.code == K.UNSUPPORTED
