"""The 4-bit KV cache on the GPU against its definition in 64 bits: the store's
codes, scales and values exactly, q and the attention within the roundings of
their 16-bit operands."""
import pytest
import torch

import kv4_reference as ref
from gpu_helpers import Guarded
from nanovllm import _native
from nanovllm.kernels.kv4_cache import (Kv4Cache, alloc_kv4_cache, kv4_attention_workspace,
                                        paged_decode_attention_kv4, qk_norm_rope_store_kv4)
from nanovllm.layers.common import rotary_cos_sin

pytestmark = pytest.mark.gpu
D, PAGE = 128, 256


def random_cache(pages, heads, device, seed=0):
    """A cache with codes over the whole range and uneven scales, and its values in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    halves = []
    for _ in range(2):
        codes = torch.randint(-7, 8, (pages, heads, PAGE, D), generator=g)
        scales = (torch.rand(pages, heads, PAGE, 4, generator=g) + 0.1).bfloat16()
        halves.append((codes, scales))
    k_codes = ref.pack(halves[0][0], None, device)[0]
    v_codes = ref.pack(halves[1][0], None, device)[1]
    cache = Kv4Cache(k_codes, halves[0][1].to(device), v_codes, halves[1][1].to(device))
    k, v = (c.double() * s.double().repeat_interleave(32, -1) for c, s in halves)
    return cache, k, v


def spread_tables(lens, pages, max_pages, seed=0, device="cpu"):
    """Block tables over shuffled pages (pages may be shared once they run out)."""
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    tables, at = torch.zeros(len(lens), max_pages, dtype=torch.int32), 0
    for i, n in enumerate(lens):
        for j in range(-(-max(n, 0) // PAGE)):
            tables[i, j] = order[at % pages]
            at += 1
    return tables.to(device)


def poison(cache, tables, lens):
    """NaN scales in the rows behind each sequence's end and in pages that no sequence owns."""
    used = torch.zeros(cache.k_codes.shape[0], PAGE, dtype=torch.bool)
    for i, n in enumerate(lens):
        for j in range(-(-max(n, 0) // PAGE)):
            used[tables[i, j], :min(PAGE, n - j * PAGE)] = True
    gone = ~used.to(cache.k_scales.device)
    cache.k_scales.transpose(1, 2)[gone] = float("nan")
    cache.v_scales.transpose(1, 2)[gone] = float("nan")


LENS = [1, 2, 0, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 700, 1536, 4352]


@pytest.mark.parametrize("hq,hkv", [(32, 8), (5, 1), (16, 2), (4, 4), (1, 1), (21, 3)])
def test_attention(cuda_device, hq, hkv):
    pages, max_pages = 40, 18
    cache, k, v = random_cache(pages, hkv, cuda_device, seed=hq)
    tables = spread_tables(LENS, pages, max_pages, seed=1)
    poison(cache, tables, LENS)
    g = torch.Generator().manual_seed(hq * 10 + hkv)
    q = torch.randn(len(LENS), hq, D, generator=g).bfloat16()
    out = Guarded((len(LENS), hq, D), torch.bfloat16, cuda_device, canary=3.0, fill=float("nan"))
    ws = Guarded((kv4_attention_workspace(len(LENS), hq, max_pages, "cpu").numel() // 4,), torch.float32, cuda_device,
                 canary=7.0, fill=float("nan"))
    lens = torch.tensor(LENS, dtype=torch.int32, device=cuda_device)
    paged_decode_attention_kv4(q.to(cuda_device), cache, tables.to(cuda_device), lens, scale=0.1, out=out.view,
                               workspace=ws.view)
    want, size = ref.attention(q, k, v, tables, LENS, 0.1)
    ref.assert_attention_close(out.view, want, size)
    assert (out.view[LENS.index(0)] == 0).all()
    assert out.intact() and ws.intact()
    assert torch.equal(lens.cpu(), torch.tensor(LENS, dtype=torch.int32))
    again = paged_decode_attention_kv4(q.to(cuda_device), cache, tables.to(cuda_device), lens, scale=0.1)
    assert torch.equal(again, out.view)  # sums in a fixed order
    assert _native.device_error() == 0


@pytest.mark.parametrize("lens", [[40000], [33000, 5, 20000], [9] * 300, [1], [0], [0, 0, 0, 77]])
def test_attention_lengths(cuda_device, lens):
    """Few long sequences, many short ones, nothing at all."""
    hq, hkv, pages = 8, 2, 64
    cache, k, v = random_cache(pages, hkv, cuda_device, seed=5)
    max_pages = max(1, -(-max(lens) // PAGE))
    tables = spread_tables(lens, pages, max_pages, seed=2)
    q = torch.randn(len(lens), hq, D, generator=torch.Generator().manual_seed(3)).bfloat16()
    out = paged_decode_attention_kv4(q.to(cuda_device), cache, tables.to(cuda_device),
                                     torch.tensor(lens, dtype=torch.int32, device=cuda_device), scale=D ** -0.5)
    want, size = ref.attention(q, k, v, tables, lens, D ** -0.5)
    ref.assert_attention_close(out, want, size)


def test_attention_large_scores_and_small_queries(cuda_device):
    """Scores of some hundreds (one token takes all) beside queries near BF16's smallest."""
    lens = [300, 300, 300, 300]
    cache, k, v = random_cache(8, 1, cuda_device, seed=6)
    tables = spread_tables(lens, 8, 2, seed=4)
    q = torch.randn(4, 4, D, generator=torch.Generator().manual_seed(8)).bfloat16()
    q[0] *= 30
    q[1] *= 1e-30
    q[2, 0] = 0
    q[3, :, ::7] *= 200
    out = paged_decode_attention_kv4(q.to(cuda_device), cache, tables.to(cuda_device),
                                     torch.tensor(lens, dtype=torch.int32, device=cuda_device), scale=0.5)
    want, size = ref.attention(q, k, v, tables, lens, 0.5)
    # the scores here reach 1e4: their FP32 error moves a probability by up to 2^-24 * 1e4 * a few
    got = out.double().cpu()
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -6) * size + 1e-30
    assert ((got - want).abs() <= bound).all()


def test_attention_nan_groups_and_values(cuda_device):
    """A NaN scale in K makes the head's output NaN, one in V only its 32 channels."""
    cache, _, _ = random_cache(4, 2, cuda_device, seed=7)
    tables = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=cuda_device)
    lens = torch.tensor([300, 300], dtype=torch.int32, device=cuda_device)
    cache.k_scales[0, 0, 17, 2] = float("nan")
    cache.v_scales[3, 1, 10, 1] = float("nan")
    q = torch.randn(2, 8, D, device=cuda_device).bfloat16()
    out = paged_decode_attention_kv4(q, cache, tables, lens, scale=0.1)
    assert out[0, :4].isnan().all() and not out[0, 4:].isnan().any()
    assert not out[1, :4].isnan().any()
    assert out[1, 4:, 32:64].isnan().all()
    assert not out[1, 4:, :32].isnan().any() and not out[1, 4:, 64:].isnan().any()


def test_attention_bad_pages_count_as_absent(cuda_device):
    cache, k, v = random_cache(6, 2, cuda_device, seed=8)
    q = torch.randn(3, 4, D, generator=torch.Generator().manual_seed(1)).bfloat16()
    lens = torch.tensor([600, 300, 256], dtype=torch.int32, device=cuda_device)
    tables = torch.tensor([[0, 6, 1], [2, -1, 0], [2 ** 30, 0, 0]], dtype=torch.int32, device=cuda_device)
    assert _native.device_error() == 0
    out = paged_decode_attention_kv4(q.to(cuda_device), cache, tables, lens, scale=0.1)
    assert _native.device_error() == 6
    # the same tokens without the bad pages: 256 + 88, 256, none
    good = torch.tensor([[0, 1], [2, 0], [0, 0]], dtype=torch.int32)
    want, size = ref.attention(q, k, v, good, [256 + 88, 256, 0], 0.1)
    ref.assert_attention_close(out, want, size)


def test_attention_scores_far_below_zero(cuda_device):
    """All scores equal and about -1e33: the mean of the values."""
    cache, _, _ = random_cache(4, 1, cuda_device, seed=22)
    cache.k_codes.copy_(cache.k_codes[0, 0, 0].clone().expand_as(cache.k_codes))
    cache.k_scales.copy_(cache.k_scales[0, 0, 0].clone().expand_as(cache.k_scales))
    k, v = ref.read_k(cache), ref.read_v(cache)
    q = (-1e32 * k[0, 0, 0].sign()).bfloat16().view(1, 1, D).expand(3, 4, D).contiguous()
    tables = torch.tensor([[2, 0], [1, 3], [0, 1]], dtype=torch.int32)
    lens = [300, 17, 512]
    out = paged_decode_attention_kv4(q.to(cuda_device), cache, tables.to(cuda_device),
                                     torch.tensor(lens, dtype=torch.int32, device=cuda_device), scale=0.1)
    want, size = ref.attention(torch.zeros_like(q), k, v, tables, lens, 0.1)  # equal scores
    ref.assert_attention_close(out, want, size)


def test_bad_indices_leave_the_rest_and_later_calls_alone(cuda_device):
    """One sequence's pages are all bad; the other sequences' outputs, and a later call's before the error is
    read, are those of a batch without it."""
    cache, _, _ = random_cache(64, 4, cuda_device, seed=20)
    gen = torch.Generator().manual_seed(21)
    lens = torch.randint(4000, 16384, (24,), generator=gen, dtype=torch.int32).to(cuda_device)
    tables = torch.randint(0, 64, (24, 64), generator=gen, dtype=torch.int32).to(cuda_device)
    q = torch.randn(24, 16, D, generator=gen).bfloat16().to(cuda_device)
    want = paged_decode_attention_kv4(q, cache, tables, lens, scale=0.1)
    assert _native.device_error() == 0
    bad = tables.clone()
    bad[0] = 64
    for _ in range(5):
        out = paged_decode_attention_kv4(q, cache, bad, lens, scale=0.1)
        assert torch.equal(out[1:], want[1:]) and not out[0].any()
        assert torch.equal(paged_decode_attention_kv4(q, cache, tables, lens, scale=0.1), want)
    assert _native.device_error() == 6
    assert _native.device_error() == 0


def test_attention_lengths_beyond_the_table_and_below_zero(cuda_device):
    cache, k, v = random_cache(4, 2, cuda_device, seed=9)
    q = torch.randn(2, 4, D, generator=torch.Generator().manual_seed(2)).bfloat16()
    tables = torch.tensor([[3, 1], [2, 0]], dtype=torch.int32, device=cuda_device)
    lens = torch.tensor([10 ** 9, -5], dtype=torch.int32, device=cuda_device)
    out = paged_decode_attention_kv4(q.to(cuda_device), cache, tables, lens, scale=0.1)
    want, size = ref.attention(q, k, v, tables, [512, 0], 0.1)
    ref.assert_attention_close(out, want, size)


def test_attention_beyond_32_bit_offsets(cuda_device):
    """Pages whose bytes lie beyond 4 GB of the codes tensor."""
    pages, hkv = 33000, 8
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    cache = alloc_kv4_cache(pages, hkv, cuda_device)
    small, k, v = random_cache(3, hkv, cuda_device, seed=10)
    where = [pages - 1, 16500, 32900]
    for s, big in zip(small, cache):
        for i, p in enumerate(where):
            big[p] = s[i]
    q = torch.randn(1, 32, D, generator=torch.Generator().manual_seed(4)).bfloat16()
    lens = torch.tensor([700], dtype=torch.int32, device=cuda_device)
    out = paged_decode_attention_kv4(q.to(cuda_device), cache,
                                     torch.tensor([where], dtype=torch.int32, device=cuda_device), lens, scale=0.1)
    want, size = ref.attention(q, k, v, torch.tensor([[0, 1, 2]]), [700], 0.1)
    ref.assert_attention_close(out, want, size)
    # a store to the last slots of that cache
    t, slots = 2, torch.tensor([pages * PAGE - 1, (pages - 1) * PAGE + 3], dtype=torch.int32, device=cuda_device)
    qkv = torch.randn(t, (2 + 2 * hkv) * D, generator=torch.Generator().manual_seed(5)).bfloat16().to(cuda_device)
    ones = torch.ones(D, dtype=torch.bfloat16, device=cuda_device)
    cos_sin = rotary_cos_sin(D, 16, 1e6).to(cuda_device)
    pos = torch.tensor([0, 7], device=cuda_device)
    _, kv, vv = qk_norm_rope_store_kv4(qkv, ones, ones, cos_sin, pos, slots, cache, num_heads=2, num_kv_heads=hkv,
                                       eps=1e-6, return_values=True)
    last = Kv4Cache(*(x[pages - 1:] for x in cache))
    assert torch.equal(ref.read_k(last)[0, :, [255, 3]].transpose(0, 1).bfloat16(), kv.cpu())
    assert torch.equal(ref.read_v(last)[0, :, [255, 3]].transpose(0, 1).bfloat16(), vv.cpu())
    assert _native.device_error() == 0


def test_attention_in_graphs_with_one_workspace(cuda_device):
    """Two captured graphs (two batch sizes) share a workspace and are replayed in turn with new lengths."""
    cache, k, v = random_cache(16, 2, cuda_device, seed=11)
    max_pages = 4
    tables = torch.arange(4 * max_pages, dtype=torch.int32, device=cuda_device).view(4, max_pages)
    lens = torch.tensor([3, 300, 600, 900], dtype=torch.int32, device=cuda_device)
    q = torch.randn(4, 8, D, device=cuda_device).bfloat16()
    out = torch.empty_like(q)
    ws = kv4_attention_workspace(4, 8, max_pages, cuda_device)
    graphs = {}
    for n in (4, 2):
        paged_decode_attention_kv4(q[:n], cache, tables[:n], lens[:n], scale=0.1, out=out[:n], workspace=ws)
        graphs[n] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[n]):
            paged_decode_attention_kv4(q[:n], cache, tables[:n], lens[:n], scale=0.1, out=out[:n], workspace=ws)
    for n, new in ((4, [1000, 1, 0, 512]), (2, [257, 1024, 5, 5]), (4, [0, 0, 64, 1024])):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        q.copy_(torch.randn(4, 8, D, device=cuda_device).bfloat16())
        out.fill_(float("nan"))
        graphs[n].replay()
        want, size = ref.attention(q, k, v, tables, new, 0.1)
        ref.assert_attention_close(out[:n], want[:n], size[:n])
        assert out[n:].isnan().all()


def test_attention_on_two_streams(cuda_device):
    """Calls that overlap on two streams, each with the workspace that it is given or takes."""
    cache, k, v = random_cache(32, 2, cuda_device, seed=12)
    lens_list = [4096, 1000, 31, 2222]
    tables = spread_tables(lens_list, 32, 16, seed=6)
    lens = torch.tensor(lens_list, dtype=torch.int32, device=cuda_device)
    q = torch.randn(2, 4, 8, D, generator=torch.Generator().manual_seed(6)).bfloat16()
    qd, td = q.to(cuda_device), tables.to(cuda_device)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(paged_decode_attention_kv4(qd[i], cache, td, lens, scale=0.1))
    torch.cuda.synchronize()
    for i in range(2):
        want, size = ref.attention(q[i], k, v, tables, lens_list, 0.1)
        ref.assert_attention_close(outs[i][0], want, size)
        assert all(torch.equal(o, outs[i][0]) for o in outs[i])


# ------------------------------------------------------------------ store
def store_inputs(t, hq, hkv, device, seed=0, pages=9):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(t, hq + 2 * hkv, D, generator=g) * (0.2 + 3 * torch.rand(t, 1, 1, generator=g))
    w = (1 + 0.3 * torch.randn(2, D, generator=g)).bfloat16()
    cos_sin = rotary_cos_sin(D, 4096, 1e6)
    pos = torch.randint(0, 4096, (t,), generator=g)
    slots = torch.randperm(pages * PAGE, generator=g)[:t].int()
    cache = Kv4Cache(*(torch.full(s, v, dtype=d, device=device) for s, v, d in (
        ((pages, hkv, PAGE, 64), 0x3C, torch.uint8), ((pages, hkv, PAGE, 4), 5.0, torch.bfloat16)) * 2))
    return qkv.bfloat16(), w, cos_sin, pos, slots, cache


def check_store(qkv, w, cos_sin, pos, slots, cache, hq, hkv, device, eps=1e-6, values=True):
    t = qkv.shape[0]
    before = Kv4Cache(*(x.clone() for x in cache))
    args = [x.to(device) for x in (qkv.reshape(t, -1), w[0], w[1], cos_sin, pos, slots)]
    q_out = Guarded((t, hq, D), torch.bfloat16, device, canary=3.0, fill=float("nan"))
    got = qk_norm_rope_store_kv4(*args, cache, num_heads=hq, num_kv_heads=hkv, eps=eps, q_out=q_out.view,
                                 return_values=values)
    assert q_out.intact()
    q, k, v = qkv.split([hq, hkv, hkv], 1)
    want_q = ref.norm_rope(q, w[0], cos_sin, pos, eps)
    # one rounding to BF16; 2^-20 of the pair's size for the FP32 arithmetic before it
    size = want_q.abs() + want_q.roll(64, -1).abs()
    assert ((q_out.view.double().cpu() - want_q).abs() <= 2.0 ** -8 * want_q.abs() + 2.0 ** -20 * size).all()
    k_codes, k_scales = ref.quantise(ref.norm_rope(k, w[1], cos_sin, pos, eps).float())
    v_codes, v_scales = ref.quantise(v.float())
    for name, codes, scales, read in (("k", k_codes, k_scales, ref.read_k), ("v", v_codes, v_scales, ref.read_v)):
        held = codes * scales.repeat_interleave(32, -1)
        if values:
            assert torch.equal(got[1 if name == "k" else 2].cpu(), held.bfloat16()), name
        stored = read(cache).transpose(1, 2).reshape(-1, hkv, D)
        old = read(before).transpose(1, 2).reshape(-1, hkv, D)
        keep = slots >= 0
        assert torch.equal(stored[slots[keep].long()], held[keep]), name
        rest = torch.ones(stored.shape[0], dtype=torch.bool)
        rest[slots[keep].long()] = False
        assert torch.equal(stored[rest], old[rest]), name
    return got


@pytest.mark.parametrize("t,hq,hkv", [(1, 32, 8), (37, 5, 1), (300, 6, 3), (64, 4, 4), (2000, 8, 2)])
def test_store(cuda_device, t, hq, hkv):
    qkv, w, cos_sin, pos, slots, cache = store_inputs(t, hq, hkv, cuda_device, seed=t + hq)
    slots[::5] = -1
    check_store(qkv, w, cos_sin, pos, slots, cache, hq, hkv, cuda_device)
    assert _native.device_error() == 0


def test_store_borders_zeros_and_tiny_values(cuda_device):
    """V on exact ties of the quantiser, all-zero groups, and values down to BF16's smallest."""
    t, hq, hkv = 64, 1, 2
    qkv, w, cos_sin, pos, slots, cache = store_inputs(t, hq, hkv, cuda_device, seed=1)
    v = qkv[:, hq + hkv:]
    # absmax 7 * 2^e: the scale is 2^e exactly, and (n + 1/2) 2^e are ties
    for i in range(16):
        ties = (torch.arange(32) % 14 - 6.5) * 2.0 ** (i - 8)
        ties[0] = 7 * 2.0 ** (i - 8)
        v[i] = ties.repeat(4).bfloat16()
    v[16, 0, :64] = 0
    qkv[17] = 0                                         # a zero row: q and k are 0 as well
    for i in range(18, 40):
        v[i] = (torch.randn(hkv, D, generator=torch.Generator().manual_seed(i)) * 2.0 ** (-120 - (i - 18))).bfloat16()
    v[40] = torch.tensor(3.3e38).bfloat16()
    check_store(qkv, w, cos_sin, pos, slots, cache, hq, hkv, cuda_device)


def test_store_not_finite(cuda_device):
    """A group with an infinity or a NaN reads back as NaN; the others are as they were."""
    t, hq, hkv = 8, 2, 1
    qkv, w, cos_sin, pos, slots, cache = store_inputs(t, hq, hkv, cuda_device, seed=2)
    v = qkv[:, hq + hkv:]
    v[0, 0, 40] = float("inf")
    v[1, 0, 127] = float("nan")
    v[2, 0, 0] = -float("inf")
    qkv[3, hq, 5] = float("nan")                        # K: the norm spreads it over the head
    clean = qkv.nan_to_num(0.5, 0.5, 0.5)
    _, k, vv = qk_norm_rope_store_kv4(qkv.view(t, -1).to(cuda_device), *(x.to(cuda_device) for x in (w[0], w[1], cos_sin, pos, slots)),
                                      cache, num_heads=hq, num_kv_heads=hkv, eps=1e-6, return_values=True)
    bad = torch.zeros(t, 1, D, dtype=torch.bool)
    bad[0, 0, 32:64] = bad[1, 0, 96:] = bad[2, 0, :32] = True
    assert torch.equal(vv.cpu().isnan(), bad)
    assert k[3].isnan().all() and not k[[0, 1, 2, 4, 5, 6, 7]].isnan().any()
    held = ref.read_v(cache).transpose(1, 2).reshape(-1, 1, D)[slots.long()]
    assert torch.equal(held.isnan(), bad)
    codes, scales = ref.quantise(clean[:, hq + hkv:].float())
    want = codes * scales.repeat_interleave(32, -1)
    assert torch.equal(held[~bad], want[~bad])


def test_store_without_cache_and_bad_indices(cuda_device):
    t, hq, hkv = 6, 2, 2
    qkv, w, cos_sin, pos, slots, cache = store_inputs(t, hq, hkv, cuda_device, seed=3, pages=2)
    dev = [x.to(cuda_device) for x in (qkv.view(t, -1), w[0], w[1], cos_sin, pos)]
    kw = dict(num_heads=hq, num_kv_heads=hkv, eps=1e-6, return_values=True)
    first = qk_norm_rope_store_kv4(*dev, slots.to(cuda_device), cache, **kw)
    second = qk_norm_rope_store_kv4(*dev, None, None, **kw)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    assert _native.device_error() == 0
    before = [x.clone() for x in cache]
    beyond = torch.tensor([2 * PAGE, -1, 2 ** 31 - 1, -7, 2 * PAGE + 5, -2 ** 31], dtype=torch.int32, device=cuda_device)
    third = qk_norm_rope_store_kv4(*dev, beyond, cache, **kw)
    assert _native.device_error() == 7
    assert all(torch.equal(a, b) for a, b in zip(cache, before))
    assert all(torch.equal(a, b) for a, b in zip(first, third))
    pos_bad = pos.clone()
    pos_bad[1], pos_bad[4] = 4096, -1
    dev[4] = pos_bad.to(cuda_device)
    q, k, v = qk_norm_rope_store_kv4(*dev, None, None, **kw)
    assert _native.device_error() == 8
    rows = torch.tensor([False, True, False, False, True, False])
    assert q[rows].isnan().all() and k[rows].isnan().all() and not v.isnan().any()
    assert torch.equal(q[~rows], first[0][~rows]) and torch.equal(v, first[2])


def test_store_then_attend_in_a_graph(cuda_device):
    """A decode step captured once: store the token's K and V, attend over the cache that now holds them."""
    b, hq, hkv, pages, eps = 3, 8, 2, 6, 1e-6
    cache = alloc_kv4_cache(pages, hkv, cuda_device)
    for x in cache:
        x.zero_()
    tables = torch.tensor([[4, 0], [1, 5], [3, 2]], dtype=torch.int32, device=cuda_device)
    w = torch.ones(D, dtype=torch.bfloat16, device=cuda_device)
    cos_sin = rotary_cos_sin(D, 1024, 1e6).to(cuda_device)
    qkv = torch.zeros(b, (hq + 2 * hkv) * D, dtype=torch.bfloat16, device=cuda_device)
    pos = torch.zeros(b, dtype=torch.int64, device=cuda_device)
    slots = torch.full((b,), -1, dtype=torch.int32, device=cuda_device)
    lens = torch.zeros(b, dtype=torch.int32, device=cuda_device)
    ws = kv4_attention_workspace(b, hq, 2, cuda_device)
    out = torch.empty(b, hq, D, dtype=torch.bfloat16, device=cuda_device)

    def step():
        q = qk_norm_rope_store_kv4(qkv, w, w, cos_sin, pos, slots, cache, num_heads=hq, num_kv_heads=hkv, eps=eps)
        paged_decode_attention_kv4(q, cache, tables, lens, scale=D ** -0.5, out=out, workspace=ws)
        return q
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = step()
    start = [0, 250, 40]
    g = torch.Generator().manual_seed(0)
    for i in range(12):
        at = [s + i for s in start]
        qkv.copy_(torch.randn(qkv.shape, generator=g).bfloat16())
        pos.copy_(torch.tensor(at))
        lens.copy_(torch.tensor([a + 1 for a in at], dtype=torch.int32))
        slots.copy_(torch.tensor([int(tables[r, a // PAGE]) * PAGE + a % PAGE for r, a in enumerate(at)],
                                 dtype=torch.int32))
        graph.replay()
        want, size = ref.attention(q, ref.read_k(cache), ref.read_v(cache), tables, [a + 1 for a in at], D ** -0.5)
        ref.assert_attention_close(out, want, size)
    assert _native.device_error() == 0


@pytest.mark.parametrize("hq,hkv", [(8, 2), (32, 8), (5, 1)])
def test_attention_rounds_its_result_once(cuda_device, hq, hkv):
    """The output's rounding to BF16 is the only one that shows, in a batch of any size, and a sequence's
    output does not depend on the sequences beside it."""
    lens = [2, 3, 4, 5, 7, 19, 33, 128] * 8
    scale = 0.1
    cache, k, v = random_cache(16, hkv, cuda_device, seed=30)
    tables = spread_tables(lens, 16, 1, seed=31)
    q = (0.02 * torch.randn(len(lens), hq, D, generator=torch.Generator().manual_seed(32))).bfloat16()
    td, ld = tables.to(cuda_device), torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    out = paged_decode_attention_kv4(q.to(cuda_device), cache, td, ld, scale=scale)
    want, size = ref.attention(q, k, v, tables, lens, scale)
    # Scores: a group's 32 products with 128 + u <= 143 and their excess 136 sum(q) are summed in FP32, in at most
    # four roundings (or truncations: 2^-23) of a partial sum of at most 143 sum |q|; group scales are below 1.1.
    # A probability moves by twice a score's error, and is held in two BF16 terms (2^-16) and FP32 (2^-18 for the
    # exponential and the sums).
    moved = 2 * 4 * 2.0 ** -23 * 143 * 1.1 * scale * q.double().abs().sum(-1, keepdim=True)
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -16 + 2.0 ** -18 + moved) * size
    assert moved.max() < 2.0 ** -11  # well below a BF16 rounding
    assert ((out.double().cpu() - want).abs() <= bound).all()
    for i in (0, 5, 63):
        alone = paged_decode_attention_kv4(q[i:i + 1].to(cuda_device), cache, td[i:i + 1], ld[i:i + 1], scale=scale)
        assert torch.equal(alone[0], out[i])
