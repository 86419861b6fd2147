"""append_kv with so many rows that a half warp takes four of a token: every way in which
these straddle q, k and v, against the 64-bit reference."""
import pytest
import torch

import paged_reference as ref
from nanovllm import _native
from nanovllm.kernels.paged_attention import append_kv
from test_paged_attention_gpu import D, PAGE, caches, rand, rotary, views

pytestmark = pytest.mark.gpu

EPS = 1e-6


def inputs(hq, hkv, layout, dim, device, without_q=False):
    """At least 16,385 rows; a seventh of the slots negative, the others scattered."""
    tokens = 16384 // ((0 if without_q else hq) + 2 * hkv) + 40
    q, k, v = views(layout, tokens, hq, hkv, device)
    g = torch.Generator().manual_seed(hq + dim)
    pages = -(-tokens // PAGE) + 1
    slots = torch.randperm(pages * PAGE, generator=g)[:tokens].int()
    slots[::7] = -1 - torch.arange(len(slots[::7])).int()
    positions = torch.randint(0, 5000, (tokens,), generator=g).to(device)
    return q, k, v, rotary(5000, dim, device), positions, slots.to(device), *caches(pages, hkv, device)


@pytest.mark.parametrize("hq,hkv", [(5, 1), (6, 2), (1, 1), (7, 3), (32, 8), (9, 1)])
@pytest.mark.parametrize("layout,dim,norm,how", [
    ("fused", 128, "both", "new"), ("strided", 16, "k", "new"), ("strided", 112, "q", "new"),
    ("separate", 64, "none", "in place"), ("separate", 16, "both", "in place"), ("strided", 112, "k", "without q"),
    ("fused", 32, "none", "without q")])
def test_append_of_many_rows(cuda_device, hq, hkv, layout, dim, norm, how):
    dev = cuda_device
    q, k, v, cos_sin, positions, slots, k_cache, v_cache = inputs(hq, hkv, layout, dim, dev, how == "without q")
    qw = (1 + rand(D, dev, 7, 0.3)) if norm in ("both", "q") else None
    kw = (1 + rand(D, dev, 8, 0.3)) if norm in ("both", "k") else None
    q_in, want_k, want_v = q.clone(), k_cache.clone(), v_cache.clone()
    out = append_kv(None if how == "without q" else q, k, v, cos_sin, positions, slots, k_cache, v_cache, q_weight=qw,
                    k_weight=kw, eps=EPS, q_out=q if how == "in place" else None)
    stored, at = slots >= 0, slots[slots >= 0].long()
    keys, size = ref.norm_rope(k, kw, cos_sin, positions, EPS)
    got = k_cache.flatten(0, 1)[at]
    ref.assert_rows_close(got, keys[stored], size[stored])
    want_k.flatten(0, 1)[at] = got
    want_v.flatten(0, 1)[at] = v[stored]
    assert torch.equal(k_cache, want_k) and torch.equal(v_cache, want_v)  # no other row was written
    if how == "without q":
        assert out is None and torch.equal(q, q_in)
    else:
        assert (out is q) == (how == "in place")
        ref.assert_rows_close(out, *ref.norm_rope(q_in, qw, cos_sin, positions, EPS))
    assert _native.device_error() == 0


@pytest.mark.parametrize("hq,hkv", [(5, 1), (6, 2), (1, 1)])
def test_append_of_many_rows_bad_indices(cuda_device, hq, hkv):
    dev = cuda_device
    q, k, v, cos_sin, positions, slots, k_cache, v_cache = inputs(hq, hkv, "fused", 64, dev)
    beyond = k_cache.shape[0] * PAGE
    slots[3], slots[-1], slots[100] = beyond, (1 << 31) - 1, -(1 << 31)
    before = k_cache.clone()
    out = append_kv(q, k, v, cos_sin, positions, slots, k_cache, v_cache)
    assert _native.device_error() == 7 and torch.isfinite(out).all()
    rest = torch.ones(beyond, dtype=torch.bool, device=dev)
    rest[slots[(slots >= 0) & (slots < beyond)].long()] = False
    assert torch.equal(k_cache.flatten(0, 1)[rest], before.flatten(0, 1)[rest])
    slots[3] = slots[-1] = slots[100] = -1
    bad = torch.tensor([1, 500, len(slots) - 2], device=dev)
    positions[bad] = torch.tensor([5000, -1, 1 << 40], device=dev)
    slots[bad] = rest.nonzero()[:3, 0].int()
    out = append_kv(q, k, v, cos_sin, positions, slots, k_cache, v_cache)
    assert _native.device_error() == 8
    good = torch.ones(len(slots), dtype=torch.bool, device=dev)
    good[bad] = False
    assert torch.isnan(out[bad]).all() and torch.isfinite(out[good]).all()
    stored = good & (slots >= 0)
    assert torch.isnan(k_cache.flatten(0, 1)[slots[bad].long()]).all()
    assert torch.isfinite(k_cache.flatten(0, 1)[slots[stored].long()]).all()
    assert torch.equal(v_cache.flatten(0, 1)[slots[bad].long()], v[bad])
