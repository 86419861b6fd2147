"""Refusals of the entry points for requests that share cached tokens, made before any
device work (no GPU)."""
import ctypes

import pytest
import torch

from nanovllm import _native
from nanovllm.kernels.paged_attention import append_kv, paged_prefill_attention, shared_prefix_attention

V = ctypes.c_void_p
INVALID, UNSUPPORTED, ALIGNMENT = _native.ERR_INVALID_ARGUMENT, _native.ERR_UNSUPPORTED, _native.ERR_ALIGNMENT


def at(i):
    return V((i + 1) << 40)  # far apart: no argument over another


def append(ptrs=(), **over):
    a = dict(t=3, hq=8, hkv=2, d=128, qs=1024, ks=256, vs=256, rot=128, page=256, pages=10, pos=64, eps=1e-6) | over
    p = [at(i) for i in range(11)]
    for i, x in dict(ptrs).items():
        p[i] = x
    return _native.load().nv4_append_kv(*p, *(a[n] for n in ("t", "hq", "hkv", "d", "qs", "ks", "vs", "rot", "page",
                                                             "pages", "pos", "eps")), None)


@pytest.mark.parametrize("over,status", [
    (dict(t=0), INVALID), (dict(t=(1 << 30) + 1), INVALID), (dict(hq=0), INVALID), (dict(hkv=0), INVALID),
    (dict(pages=0), INVALID), (dict(pages=1 << 23), INVALID), (dict(pos=0), INVALID), (dict(eps=-1.0), INVALID),
    (dict(eps=float("nan")), INVALID), (dict(eps=1.0), INVALID), (dict(qs=1016), INVALID), (dict(ks=248), INVALID),
    (dict(vs=128), INVALID), (dict(ks=(1 << 32) + 8), INVALID), (dict(d=64), UNSUPPORTED),
    (dict(page=128), UNSUPPORTED), (dict(rot=0), UNSUPPORTED), (dict(rot=24), UNSUPPORTED),
    (dict(rot=144), UNSUPPORTED), (dict(qs=1028), ALIGNMENT),
    (dict(ks=260), ALIGNMENT), (dict(vs=257), ALIGNMENT)])
def test_append_refusals(over, status):
    assert append(**over) == status


@pytest.mark.parametrize("i", range(11))
def test_append_pointers(i):
    if i not in (3, 4):  # the weights are optional
        assert append(ptrs={i: None}) == INVALID
    assert append(ptrs={i: V(at(i).value + 2)}) == ALIGNMENT


@pytest.mark.parametrize("i,j", [(8, 1), (8, 2), (8, 5), (9, 0), (9, 1), (9, 2), (9, 7), (10, 9), (10, 3), (8, 9)])
def test_append_overlaps(i, j):
    assert append(ptrs={i: at(j)}) == INVALID


def test_append_q_in_place_needs_contiguous_rows():
    assert append(ptrs={8: at(0)}, qs=2048) == INVALID


def attention(name, count, ptrs=(), **over):
    a = dict(ws=1 << 40, rows=6, batch=2, groups=1, hq=8, hkv=2, d=128, page=256, pages=10, max_pages=4,
             scale=0.1) | over
    p = [at(i) for i in range(count)]
    for i, x in dict(ptrs).items():
        p[i] = x
    sizes = ("ws", "rows", "batch") if name == "prefill" else ("ws", "batch", "groups")
    lib = _native.load()
    call = lib.nv4_paged_prefill_attention if name == "prefill" else lib.nv4_shared_prefix_attention
    return call(*p, *(a[n] for n in sizes + ("hq", "hkv", "d", "page", "pages", "max_pages", "scale")), None)


BOTH = [("prefill", 8), ("shared", 9)]


@pytest.mark.parametrize("name,count", BOTH)
@pytest.mark.parametrize("over,status", [
    (dict(batch=0), INVALID), (dict(batch=65536), INVALID), (dict(hkv=0), INVALID), (dict(hq=9), INVALID),
    (dict(hq=1), INVALID), (dict(hq=65536, hkv=1024), INVALID), (dict(hq=1025, hkv=1025), INVALID),
    (dict(pages=0), INVALID), (dict(pages=1 << 23), INVALID),
    (dict(max_pages=0), INVALID), (dict(max_pages=1 << 16), INVALID), (dict(scale=0.0), INVALID),
    (dict(scale=-1.0), INVALID), (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID),
    (dict(ws=8), INVALID), (dict(d=64), UNSUPPORTED), (dict(page=128), UNSUPPORTED), (dict(hq=34), UNSUPPORTED)])
def test_attention_refusals(name, count, over, status):
    assert attention(name, count, **over) == status


@pytest.mark.parametrize("name,count", BOTH)
def test_attention_refuses_more_tiles_than_a_worker_can_count(name, count):
    rows = dict(rows=65535) if name == "prefill" else {}
    assert attention(name, count, batch=65535, max_pages=65535, hkv=8, hq=64, ws=1 << 62, **rows) == UNSUPPORTED


def test_attention_counts():
    assert attention("prefill", 8, rows=0) == INVALID
    assert attention("prefill", 8, rows=(1 << 22) + 1) == INVALID
    assert attention("shared", 9, groups=-1) == INVALID
    assert attention("shared", 9, groups=65536) == INVALID
    lib = _native.load()
    for sizes in ((0, 1, 8, 2), (1, 0, 8, 2), (1, 1, 8, 3), (1, 1, 34, 2), (1 << 23, 1, 8, 2)):
        assert lib.nv4_paged_prefill_attention_workspace_bytes(*sizes) == 0
    for sizes in ((0, 1, 8, 2), (1, -1, 8, 2), (1, 1, 8, 3), (1, 1, 34, 2), (65536, 1, 8, 2)):
        assert lib.nv4_shared_prefix_attention_workspace_bytes(*sizes) == 0


@pytest.mark.parametrize("name,count", BOTH)
def test_workspaces_grow_with_every_size(name, count):
    """One made for the largest call serves the smaller ones."""
    of = getattr(_native, f"{'paged_prefill' if name == 'prefill' else 'shared_prefix'}_attention_workspace_bytes")
    for heads in ((1, 1), (8, 2), (5, 1), (32, 8), (48, 3)):
        last = 0
        for a, b in ((1, 1), (2, 1), (2, 2), (7, 3), (100, 3), (129, 64), (1000, 64), (60000, 600)):
            n = of(a, b, *heads)
            assert n >= last > -1 and n > 0
            last = n


@pytest.mark.parametrize("name,count", BOTH)
def test_attention_pointers(name, count):
    for i in range(count):
        assert attention(name, count, ptrs={i: None}) == INVALID, i
        assert attention(name, count, ptrs={i: V(at(i).value + 2)}) == ALIGNMENT, i
    out = count - 2
    assert attention(name, count, ptrs={out: V(at(out).value + 16)}) == ALIGNMENT  # stored 32 bytes at a time
    for over in range(out):  # the inputs
        assert attention(name, count, ptrs={out: at(over)}) == INVALID, over
        assert attention(name, count, ptrs={count - 1: at(over)}) == INVALID, over
    assert attention(name, count, ptrs={out: at(count - 1)}) == INVALID


# ------------------------------------------------------------------ through Python
def cpu(shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


def append_args(**over):
    a = dict(q=cpu((3, 8, 128)), k=cpu((3, 2, 128)), v=cpu((3, 2, 128)), cos_sin=cpu((64, 128), torch.float32),
             positions=cpu(3, torch.int64), slot_mapping=cpu(3, torch.int32), k_cache=cpu((4, 256, 2, 128)),
             v_cache=cpu((4, 256, 2, 128))) | over
    return a


@pytest.mark.parametrize("over,text", [
    (dict(), "CUDA device"), (dict(q=cpu((2, 8, 128))), "q"), (dict(q=cpu((3, 8, 64))), "q"),
    (dict(q=cpu((3, 8, 128), torch.float32)), "q"), (dict(k=cpu((3, 4, 128))), "KV heads"),
    (dict(v=cpu((3, 1, 128))), "KV heads"), (dict(k=cpu((3, 2, 128), torch.float16)), "BF16 k"),
    (dict(cos_sin=cpu((64, 24), torch.float32)), "rotary_dim"),
    (dict(cos_sin=cpu((64, 256), torch.float32)), "rotary_dim"),
    (dict(cos_sin=cpu((64, 128), torch.float64)), "cos_sin"), (dict(positions=cpu(3, torch.int32)), "positions"),
    (dict(slot_mapping=cpu(3, torch.int64)), "slot_mapping"), (dict(k_cache=cpu((4, 128, 2, 128))), "k_cache"),
    (dict(v_cache=cpu((5, 256, 2, 128))), "v_cache"), (dict(q_weight=cpu(64)), "q_weight"),
    (dict(k_weight=cpu(128, torch.float32)), "k_weight"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(q_out=cpu((3, 4, 128))), "q_out"), (dict(q=None, q_out=cpu((3, 8, 128))), "q_out")])
def test_append_kv_refusals(over, text):
    with pytest.raises(ValueError, match=text):
        append_kv(**append_args(**over))
    with pytest.raises(TypeError):
        append_kv(**append_args(k=3))


def attention_args(**over):
    return dict(q=cpu((3, 8, 128)), k_cache=cpu((4, 256, 2, 128)), v_cache=cpu((4, 256, 2, 128)),
                block_tables=cpu((3, 2), torch.int32), context_lens=cpu(3, torch.int32), scale=0.1) | over


COMMON = [
    (dict(), "CUDA device"), (dict(q=cpu((3, 7, 128))), "query heads"), (dict(q=cpu((3, 1, 128))), "query heads"),
    (dict(q=cpu((3, 34, 128))), "query heads"), (dict(q=cpu((3, 8, 64))), "q"),
    (dict(q=cpu((3, 8, 128), torch.float16)), "q"),
    (dict(k_cache=cpu((4, 256, 2, 64))), "k_cache"), (dict(v_cache=cpu((4, 256, 1, 128))), "v_cache"),
    (dict(block_tables=cpu((3, 2), torch.int64)), "block_tables"),
    (dict(block_tables=cpu((3, 0), torch.int32)), "block_tables"),
    (dict(context_lens=cpu(2, torch.int32)), "context_lens"), (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(out=cpu((3, 8, 64))), "out")]


@pytest.mark.parametrize("over,text", COMMON + [(dict(query_starts=cpu(3, torch.int32)), "query_starts"),
                                                (dict(query_starts=cpu(4, torch.int64)), "query_starts")])
def test_prefill_refusals(over, text):
    with pytest.raises(ValueError, match=text):
        paged_prefill_attention(**attention_args(**dict(query_starts=cpu(4, torch.int32)) | over))


@pytest.mark.parametrize("over,text", COMMON + [(dict(group_starts=cpu(3, torch.int32)), "group_starts"),
                                                (dict(prefix_lens=cpu(1, torch.int64)), "prefix_lens"),
                                                (dict(q=cpu((2, 8, 128))), "one query token")])
def test_shared_refusals(over, text):
    with pytest.raises(ValueError, match=text):
        shared_prefix_attention(**attention_args(**dict(group_starts=cpu(2, torch.int32),
                                                        prefix_lens=cpu(1, torch.int32)) | over))
