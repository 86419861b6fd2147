"""The scratch sizes that nanovllm.kernels.paged_attention states."""
import pytest

from nanovllm import _native

SIZES = [(1, 1), (37, 1), (300, 300), (16384, 4), (131072, 16), (1 << 22, 64), (1 << 22, 65535)]


@pytest.mark.parametrize("hq,hkv", [(1, 1), (5, 1), (16, 1), (32, 8), (48, 3)])
@pytest.mark.parametrize("tokens,batch", SIZES)
def test_prefill_scratch(tokens, batch, hq, hkv):
    """A block has as many whole tokens as make at most 128 rows of a KV head."""
    blocks = tokens // (128 // (hq // hkv)) + batch
    n = _native.paged_prefill_attention_workspace_bytes(tokens, batch, hq, hkv)
    assert 40 * blocks < n <= 43e6 + 40 * blocks


@pytest.mark.parametrize("hq,hkv", [(1, 1), (5, 1), (16, 1), (32, 8), (48, 3)])
@pytest.mark.parametrize("batch,groups", [(1, 0), (4, 1), (32, 32), (1024, 7), (65535, 65535)])
def test_decode_scratch(batch, groups, hq, hkv):
    n = _native.shared_prefix_attention_workspace_bytes(batch, groups, hq, hkv)
    assert 4160 * batch * hq < n <= 43e6 + 4160 * batch * hq + 100 * (batch + groups)
