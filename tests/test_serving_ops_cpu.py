"""Refusals of the 4-bit cache, step table and log-probability entry points, made
before any device work (no GPU), and the reference of their tests against
itself."""
import ctypes

import pytest
import torch

import kv4_reference as ref
from nanovllm import _native
from nanovllm.kernels.kv4_cache import (Kv4Cache, alloc_kv4_cache, kv4_attention_workspace, page_bytes,
                                        paged_decode_attention_kv4, qk_norm_rope_store_kv4)
from nanovllm.kernels.step_tables import alloc_step_tables, build_step_tables
from nanovllm.kernels.token_logprobs import token_logprobs

V = ctypes.c_void_p
P = V(256)
INVALID, UNSUPPORTED, ALIGNMENT = _native.ERR_INVALID_ARGUMENT, _native.ERR_UNSUPPORTED, _native.ERR_ALIGNMENT


def attention(ptrs=(), **over):
    a = dict(ws=1 << 40, batch=2, hq=8, hkv=2, d=128, page=256, pages=10, max_pages=4, scale=0.1) | over
    p = [P] * 9
    for i, x in dict(ptrs).items():
        p[i] = x
    return _native.load().nv4_paged_decode_attention_kv4(*p, a["ws"], a["batch"], a["hq"], a["hkv"], a["d"], a["page"],
                                                         a["pages"], a["max_pages"], a["scale"], None)


@pytest.mark.parametrize("over,status", [
    (dict(batch=0), INVALID), (dict(batch=65536), INVALID), (dict(hkv=0), INVALID), (dict(hq=9), INVALID),
    (dict(hq=1), INVALID), (dict(pages=0), INVALID), (dict(pages=1 << 23), INVALID), (dict(max_pages=0), INVALID),
    (dict(max_pages=1 << 16), INVALID), (dict(scale=0.0), INVALID), (dict(scale=float("nan")), INVALID),
    (dict(scale=float("inf")), INVALID), (dict(ws=16), INVALID), (dict(d=64), UNSUPPORTED), (dict(page=128), UNSUPPORTED),
    (dict(hq=18), UNSUPPORTED),
    (dict(batch=65535, hq=65535, hkv=65535, ws=1 << 62), INVALID)])
def test_attention_refusals(over, status):
    assert attention(**over) == status


@pytest.mark.parametrize("i", range(9))
def test_attention_pointers(i):
    assert attention(ptrs={i: None}) == INVALID
    assert attention(ptrs={i: V(256 + 2)}) == ALIGNMENT


def store(ptrs=(), **over):
    a = dict(t=3, hq=8, hkv=2, d=128, page=256, pages=10, pos=64, eps=1e-6) | over
    p = [P] * 13
    for i, x in dict(ptrs).items():
        p[i] = x
    return _native.load().nv4_qk_norm_rope_store_kv4(*p, a["t"], a["hq"], a["hkv"], a["d"], a["page"], a["pages"],
                                                     a["pos"], a["eps"], None)


@pytest.mark.parametrize("over,status", [
    (dict(t=0), INVALID), (dict(t=1 << 31), INVALID), (dict(hq=0), INVALID), (dict(hkv=0), INVALID),
    (dict(pages=0), INVALID), (dict(pages=1 << 23), INVALID), (dict(pos=0), INVALID), (dict(eps=-1.0), INVALID),
    (dict(eps=float("nan")), INVALID), (dict(d=64), UNSUPPORTED), (dict(page=64), UNSUPPORTED)])
def test_store_refusals(over, status):
    assert store(**over) == status


@pytest.mark.parametrize("i", range(13))
def test_store_pointers(i):
    assert store(ptrs={i: None}) == INVALID  # slot_mapping and the cache, k_out and v_out, only together
    assert store(ptrs={i: V(256 + 2)}) == ALIGNMENT


def tables(ptrs=(), **over):
    a = dict(batch=3, rows=4, listed=10, tokens=9, max_pages=4, page=256) | over
    p = [P] * 8
    for i, x in dict(ptrs).items():
        p[i] = x
    return _native.load().nv4_step_tables(*p, a["batch"], a["rows"], a["listed"], a["tokens"], a["max_pages"], a["page"],
                                          None)


@pytest.mark.parametrize("over,status", [
    (dict(batch=0), INVALID), (dict(rows=2), INVALID), (dict(listed=-1), INVALID), (dict(tokens=-1), INVALID),
    (dict(max_pages=0), INVALID), (dict(page=0), INVALID), (dict(batch=28673, rows=28673), UNSUPPORTED)])
def test_step_tables_refusals(over, status):
    assert tables(**over) == status


@pytest.mark.parametrize("i", range(8))
def test_step_tables_pointers(i):
    assert tables(ptrs={i: None}) == INVALID
    assert tables(ptrs={i: V(256 + 2)}) == ALIGNMENT


def logprobs(ptrs=(), **over):
    a = dict(fp32=1, rows=3, vocab=100000, stride=100000, k=2, ws=1 << 30) | over
    p = [P] * 8
    for i, x in dict(ptrs).items():
        p[i] = x
    return _native.load().nv4_token_logprobs(p[0], a["fp32"], *p[1:], a["ws"], a["rows"], a["vocab"], a["stride"],
                                             a["k"], None)


@pytest.mark.parametrize("over,status", [
    (dict(fp32=2), INVALID), (dict(rows=0), INVALID), (dict(vocab=0), INVALID), (dict(stride=99999), INVALID),
    (dict(k=-1), INVALID), (dict(ws=100), INVALID), (dict(k=33), UNSUPPORTED), (dict(vocab=(1 << 24) + 1, stride=1 << 25), UNSUPPORTED)])
def test_logprob_refusals(over, status):
    assert logprobs(**over) == status


@pytest.mark.parametrize("i", range(8))
def test_logprob_pointers(i):
    assert logprobs(ptrs={i: None}) == INVALID
    assert logprobs(ptrs={i: V(256 + 1)}) == ALIGNMENT


def test_python_refusals():
    """Shapes, types and devices refused by the Python entry points."""
    cache = alloc_kv4_cache(2, 2, "cpu")
    assert sum(x.numel() * x.element_size() for x in cache) == 2 * page_bytes(2)
    q = torch.zeros(3, 8, 128, dtype=torch.bfloat16)
    tab, lens = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        paged_decode_attention_kv4(q, cache, tab, lens, scale=0.1)
    with pytest.raises(ValueError, match="q"):
        paged_decode_attention_kv4(q.float(), cache, tab, lens, scale=0.1)
    with pytest.raises(ValueError, match="128"):
        paged_decode_attention_kv4(q[..., :64], cache, tab, lens, scale=0.1)
    with pytest.raises(ValueError, match="at least one"):
        alloc_kv4_cache(0, 2, "cpu")
    assert kv4_attention_workspace(3, 8, 2, "cpu").numel() > 0
    t, hq, hkv = 3, 4, 2
    qkv, w = torch.zeros(t, 8 * 128, dtype=torch.bfloat16), torch.ones(128, dtype=torch.bfloat16)
    cs, pos, slots = torch.zeros(16, 128), torch.zeros(t, dtype=torch.int64), torch.zeros(t, dtype=torch.int32)
    kw = dict(num_heads=hq, num_kv_heads=hkv, eps=1e-6)
    for bad, match in (((qkv[:, :-1], w, w, cs, pos, slots, cache), "qkv"), ((qkv, w[:64], w, cs, pos, slots, cache), "weight"),
                       ((qkv, w, w, cs.double(), pos, slots, cache), "cos_sin"), ((qkv, w, w, cs, pos.int(), slots, cache), "positions"),
                       ((qkv, w, w, cs, pos, slots.long(), cache), "slot"), ((qkv, w, w, cs, pos, None, cache), "together"),
                       ((qkv, w, w, cs, pos, slots, cache._replace(k_scales=None)), "together"),
                       ((qkv, w, w, cs, pos, None, cache._replace(k_codes=None)), "together"),
                       ((qkv, w, w, cs, pos, slots, cache), "CUDA")):
        with pytest.raises(ValueError, match=match):
            qk_norm_rope_store_kv4(*bad, **kw)
    with pytest.raises(RuntimeError, match="ambiguous"):
        qk_norm_rope_store_kv4(qkv, w, w, cs, pos, slots, cache, return_values=torch.ones(2), **kw)
    with pytest.raises(TypeError, match="tensor"):
        paged_decode_attention_kv4(q, cache._replace(v_codes=None), tab, lens, scale=0.1)
    one = torch.ones(2, dtype=torch.int32)
    for bad, over, match in (((one.long(), one, one), {}, "cached"), ((one, one[:1], one), {}, "cached"), ((one, one, one[None]), {}, "pages"),
                             ((one, one, one), dict(num_tokens=-1), "num_tokens"), ((one, one, one), dict(max_pages=0), "max_pages"),
                             ((one, one, one), {}, "CUDA"), ((torch.ones(28673, dtype=torch.int32),) * 2 + (one,), {}, "28672")):
        with pytest.raises(ValueError, match=match):
            build_step_tables(*bad, **(dict(num_tokens=2, max_pages=1) | over))
    assert alloc_step_tables(2, 3, 4, "cpu").positions.shape == (3,)
    x, t = torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64)
    for bad, over, match in (((x.half(), t), {}, "logits"), ((x[0], t), {}, "logits"), ((x, t.int()), {}, "targets"), ((x, t[:1]), {}, "targets"),
                             ((x, t), dict(top_k=33), "top_k"), ((x, t), dict(top_k=-1), "top_k"), ((x, t), {}, "CUDA")):
        with pytest.raises(ValueError, match=match):
            token_logprobs(*bad, **over)


def test_cache_checks():
    check = _native.serving().check_cache
    c = alloc_kv4_cache(2, 3, "cpu")
    assert check(*c) == 3
    for bad, err in ((c._replace(k_codes=c.k_codes[:, :, :128]), ValueError), (c._replace(v_codes=c.v_codes[:1]), ValueError),
                     (c._replace(k_scales=c.k_scales[..., :2]), ValueError), (c._replace(v_scales=c.v_scales.half()), TypeError),
                     (c._replace(k_codes=c.k_codes.to(torch.int8)), TypeError)):
        with pytest.raises(err):
            check(*bad)


def test_reference_packing_round_trip():
    """The tests' own packer and reader agree, and every nibble of a page is used once."""
    g = torch.Generator().manual_seed(0)
    codes = torch.randint(-7, 8, (2, 3, 256, 128), generator=g)
    scales = torch.ones(2, 3, 256, 4, dtype=torch.bfloat16)
    k, v = ref.pack(codes, scales, "cpu")
    cache = Kv4Cache(k, scales, v, scales)
    assert torch.equal(ref.read_k(cache), codes.double()) and torch.equal(ref.read_v(cache), codes.double())
    for byte in (ref.K_BYTE, ref.V_BYTE):
        assert torch.equal((byte * 2 + ref.SHIFT // 4).flatten().sort().values, torch.arange(256 * 128))


def test_logprob_workspace():
    """None once the rows alone fill the GPU; a part for every CTA of a row else."""
    size = _native.load().nv4_token_logprobs_workspace_bytes
    assert size(1024, 151936, 20) == 0 and size(1, 100, 5) == 0
    assert size(1, 151936, 0) > 0 and size(1, 151936, 20) - size(1, 151936, 0) == 37 * 20 * 8  # 297 chunks, 8 a part
    assert size(1024, 1 << 24, 0) > 0 and size(0, 100, 5) == 0 and size(1, 100, 33) == 0


def test_engine_parameters(tmp_path):
    from nanovllm.config import Config
    from nanovllm.engine.sequence import Sequence
    from nanovllm.sampling_params import SamplingParams
    from nanovllm.utils import synthetic
    model = synthetic.write_qwen3_config(str(tmp_path), num_hidden_layers=1)
    assert Config(model).kv_cache_dtype == "bf16" and Config(model, kv_cache_dtype="int4").kv_cache_dtype == "int4"
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        Config(model, kv_cache_dtype="fp8")
    for bad in (dict(logprobs=-1), dict(logprobs=33), dict(prompt_logprobs=33)):
        with pytest.raises(ValueError, match="logprobs"):
            SamplingParams(**bad)
    s = Sequence([1, 2], SamplingParams(logprobs=0, prompt_logprobs=4))
    assert s.top_logprobs == 0 and s.top_prompt_logprobs == 4 and s.logprobs == [] and s.prompt_logprobs is None
    assert Sequence([1]).top_logprobs is None


@pytest.mark.parametrize("bad", [2.5, 1.0, "3", float("nan"), [1], -1, 33])
def test_logprob_counts_are_whole_numbers(bad):
    """A step would refuse the rest, with its requests already scheduled."""
    from nanovllm.sampling_params import SamplingParams
    for name in ("logprobs", "prompt_logprobs"):
        with pytest.raises(ValueError, match="logprobs"):
            SamplingParams(**{name: bad})
        assert getattr(SamplingParams(**{name: torch.tensor(3)}), name) == 3


def spread_pointers():
    """Addresses of the step tables' arguments, far from one another."""
    return {i: V(4096 * (i + 1)) for i in range(8)}


def test_step_tables_refuse_outputs_over_inputs_or_one_another():
    """Every CTA reads the lengths and pages while others write."""
    far = spread_pointers()
    without_gpu = _native.ERR_DEVICE if not torch.cuda.is_available() else None
    if without_gpu is not None:  # the arguments pass, the device does not
        assert tables(ptrs=far) == without_gpu
        # side by side: 3 lengths, 10 pages; 4 x 4 table, 4 lengths, 5 starts, 9 slots, 9 positions
        assert tables(ptrs={0: V(256), 1: V(268), 2: V(280), 3: V(320), 4: V(384), 5: V(400), 6: V(420), 7: V(456)}) == without_gpu
    for out in range(3, 8):
        for other in range(8):
            if other != out:
                assert tables(ptrs=far | {out: far[other]}) == INVALID
    assert tables(ptrs=far | {3: V(far[0].value - 4 * 4 * 4 + 4)}) == INVALID   # the table's last element
    assert tables(ptrs=far | {7: V(far[2].value + 9 * 4 + 4 - 8)}) == INVALID   # the last page


def test_the_4_bit_cache_needs_its_head_dim(tmp_path):
    """Said before a model is built."""
    from nanovllm.config import Config
    from nanovllm.utils import synthetic
    model = synthetic.write_qwen3_config(str(tmp_path), num_hidden_layers=1, head_dim=64)
    with pytest.raises(ValueError, match="head_dim 128"):
        Config(model, kv_cache_dtype="int4")
    assert Config(model).kv_cache_dtype == "bf16"
