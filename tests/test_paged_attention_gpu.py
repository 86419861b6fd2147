"""Operators of requests that share cached tokens (csrc/paged_attention.cu) against
64-bit references: append_kv, paged_prefill_attention, shared_prefix_attention."""
import pytest
import torch

import paged_reference as ref
from nanovllm import _native
from nanovllm.kernels.paged_attention import (append_kv, paged_prefill_attention, prefill_attention_workspace,
                                              shared_prefix_attention, shared_prefix_workspace)
from nanovllm.kernels.step_tables import build_step_tables

pytestmark = pytest.mark.gpu
D, PAGE = 128, 256
SCALE = D ** -0.5


def rand(shape, device, seed, scale=1.0):
    g = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(shape, device=device, generator=g) * scale).bfloat16()


def rotary(length, dim, device):
    inverse = 1.0 / (1e4 ** (torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim))
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * inverse
    return torch.cat((angle.cos(), angle.sin()), -1).float()


def caches(pages, hkv, device, seed=0):
    k, v = rand((pages, PAGE, hkv, D), device, seed + 100), rand((pages, PAGE, hkv, D), device, seed + 200)
    k *= 1 + 4 * (torch.arange(D, device=device) % 23 == 3)
    return k, v


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def page_lists(counts, seed):
    order = torch.randperm(sum(counts), generator=torch.Generator().manual_seed(seed)).tolist()
    out, at = [], 0
    for n in counts:
        out.append(order[at:at + n])
        at += n
    return out


def padded(lists, width=None):
    width = width or max(1, max(len(x) for x in lists))
    return [x + [0] * (width - len(x)) for x in lists]


# ------------------------------------------------------------------ append
def views(layout, t, hq, hkv, device, seed=0):
    if layout == "fused":
        return rand((t, hq + 2 * hkv, D), device, seed).split([hq, hkv, hkv], 1)
    if layout == "strided":  # tokens 24 channels further apart than their heads
        return [rand((t, h * D + 24), device, seed + i)[:, :h * D].unflatten(1, (h, D))
                for i, h in enumerate((hq, hkv, hkv))]
    return [rand((t, h, D), device, seed + i) for i, h in enumerate((hq, hkv, hkv))]


def check_append(q, k, v, cos_sin, positions, slots, hkv, qw, kw, device, **kw_args):
    pages = 4
    k_cache, v_cache = caches(pages, hkv, device)
    want_k, want_v = k_cache.clone(), v_cache.clone()
    q_in, eps = (None if q is None else q.clone()), 1e-6
    out = append_kv(q, k, v, cos_sin, positions, slots, k_cache, v_cache, q_weight=qw, k_weight=kw, eps=eps, **kw_args)
    at = slots.long()
    stored = (at >= 0) & (at < pages * PAGE)
    wk, sk = ref.norm_rope(k, kw, cos_sin, positions, eps)
    got = k_cache.flatten(0, 1)[at[stored]]
    ref.assert_rows_close(got, wk[stored], sk[stored])
    want_k.flatten(0, 1)[at[stored]] = got
    want_v.flatten(0, 1)[at[stored]] = v[stored]
    assert torch.equal(k_cache, want_k) and torch.equal(v_cache, want_v)  # nothing else was written
    if q is None:
        assert out is None
    else:
        ref.assert_rows_close(out, *ref.norm_rope(q_in, qw, cos_sin, positions, eps))
    assert _native.device_error() == 0
    return out


@pytest.mark.parametrize("t,hq,hkv", [(1, 8, 2), (3, 5, 1), (33, 32, 8), (301, 40, 8), (7, 1, 1), (5, 48, 3),
                                      (2, 128, 8)])
@pytest.mark.parametrize("layout,dim,norm", [("fused", 128, "both"), ("separate", 64, "none"), ("strided", 16, "k"),
                                             ("strided", 112, "q")])
def test_append(cuda_device, t, hq, hkv, layout, dim, norm):
    dev = cuda_device
    q, k, v = views(layout, t, hq, hkv, dev)
    g = torch.Generator().manual_seed(t)
    slots = torch.randperm(4 * PAGE, generator=g)[:t].int().to(dev)
    slots[t // 2] = -1 if t > 1 else slots[0]
    positions = torch.randint(0, 5000, (t,), generator=g).to(dev)
    positions[0], positions[-1] = 0, 4999
    qw = (1 + rand(D, dev, 7, 0.3)) if norm in ("both", "q") else None
    kw = (1 + rand(D, dev, 8, 0.3)) if norm in ("both", "k") else None
    check_append(q, k, v, rotary(5000, dim, dev), positions, slots, hkv, qw, kw, dev)


def test_append_without_q_in_place_and_empty(cuda_device):
    dev = cuda_device
    q, k, v = views("separate", 9, 6, 2, dev)
    cos_sin, positions, slots = rotary(64, 128, dev), torch.arange(9, device=dev), i32(list(range(250, 259)), dev)
    check_append(None, k, v, cos_sin, positions, slots, 2, None, None, dev)
    assert check_append(q, k, v, cos_sin, positions, slots, 2, None, None, dev, q_out=q) is q
    k_cache, v_cache = caches(1, 2, dev)
    out = append_kv(q[:0], k[:0], v[:0], cos_sin, positions[:0], slots[:0], k_cache, v_cache)
    assert out.shape == (0, 6, D)


def test_append_many_tokens(cuda_device):
    dev, t = cuda_device, 4999
    q, k, v = views("fused", t, 8, 4, dev)
    k_cache, v_cache = caches(20, 4, dev)
    slots = torch.arange(t, device=dev).int().flip(0).contiguous()
    cos_sin, positions = rotary(t, 128, dev), torch.arange(t, device=dev)
    out = append_kv(q, k, v, cos_sin, positions, slots, k_cache, v_cache, k_weight=torch.ones(D, device=dev).bfloat16())
    ref.assert_rows_close(out, *ref.norm_rope(q, None, cos_sin, positions, 0))
    ref.assert_rows_close(k_cache.flatten(0, 1)[:t].flip(0), *ref.norm_rope(k, torch.ones(D, device=dev), cos_sin,
                                                                            positions, 1e-6))
    assert torch.equal(v_cache.flatten(0, 1)[:t].flip(0), v)


def test_append_bad_indices(cuda_device):
    dev = cuda_device
    q, k, v = views("separate", 4, 2, 1, dev)
    k_cache, v_cache = caches(2, 1, dev)
    before = k_cache.clone(), v_cache.clone()
    cos_sin = rotary(10, 128, dev)
    slots = i32([512, -1, -(1 << 31), (1 << 31) - 1], dev)
    out = append_kv(q, k, v, cos_sin, torch.arange(4, device=dev), slots, k_cache, v_cache)
    assert _native.device_error() == 7
    assert torch.equal(k_cache, before[0]) and torch.equal(v_cache, before[1]) and torch.isfinite(out).all()
    positions = torch.tensor([10, -1, 9, 1 << 40], device=dev)
    out = append_kv(q, k, v, cos_sin, positions, i32([0, 1, 2, 3], dev), k_cache, v_cache)
    assert _native.device_error() == 8
    for rows in (out, k_cache.flatten(0, 1)):
        assert torch.isnan(rows[[0, 1, 3]]).all() and torch.isfinite(rows[2]).all()
    assert torch.equal(v_cache.flatten(0, 1)[:4], v)


def test_append_extreme_rows(cuda_device):
    dev = cuda_device
    q, k, v = views("separate", 4, 2, 1, dev)
    k[0] = 0
    k[1] *= 2.0 ** 100  # the square overflows without the norm only
    k[2] *= 2.0 ** -100
    k[3, 0, 5] = float("inf")
    cos_sin, positions, slots = rotary(8, 128, dev), torch.arange(4, device=dev), i32([0, 1, 2, 3], dev)
    k_cache, v_cache = caches(1, 1, dev)
    append_kv(q, k, v, cos_sin, positions, slots, k_cache, v_cache)
    want, size = ref.norm_rope(k[:3], None, cos_sin, positions[:3], 0)
    ref.assert_rows_close(k_cache.flatten(0, 1)[:3], want, size)
    assert not torch.isfinite(k_cache[0, 3]).all()


# ------------------------------------------------------------------ prefill
def prefill_case(lens, hq, hkv, device, seed=0, extra_rows=0, spare_pages=2):
    """lens: (cached, new) per request; returns the call's inputs and host lists."""
    lists = page_lists([-(-(c + n) // PAGE) for c, n in lens] + [spare_pages], seed)[:-1]
    tables, context, starts = padded(lists), [c + n for c, n in lens], [0]
    for _, n in lens:
        starts.append(starts[-1] + n)
    k_cache, v_cache = caches(sum(len(x) for x in lists) + spare_pages, hkv, device, seed)
    q = rand((starts[-1] + extra_rows, hq, D), device, seed)
    return q, k_cache, v_cache, tables, context, starts


def close_prompt(got, want, size):
    ref.assert_attention_close(got, want, size, terms=1)


def run_prefill(q, k_cache, v_cache, tables, context, starts, **kw):
    dev = q.device
    return paged_prefill_attention(q, k_cache, v_cache, i32(tables, dev), i32(context, dev), i32(starts, dev),
                                   scale=kw.pop("scale", SCALE), **kw)


LENS = [
    [(0, 1)], [(0, 2)], [(300, 1)], [(255, 2)], [(0, 257)], [(256, 128)], [(127, 129)],
    [(0, 5), (511, 1), (700, 130), (0, 0), (128, 129), (1, 255)],
    [(1000, 3), (2000, 64), (0, 600)],
]


@pytest.mark.parametrize("hq,hkv", [(8, 2), (5, 1), (16, 1), (3, 3), (1, 1)])
@pytest.mark.parametrize("lens", LENS, ids=lambda x: "-".join(f"{c}+{n}" for c, n in x))
def test_prefill(cuda_device, lens, hq, hkv):
    case = prefill_case(lens, hq, hkv, cuda_device, seed=len(lens))
    out = run_prefill(*case)
    want, size, rows = ref.prefill(*case, SCALE)
    assert rows.all()
    close_prompt(out, want, size)
    assert _native.device_error() == 0


@pytest.mark.parametrize("lens,hq,hkv", [([(1500, 1100)], 32, 8), ([(0, 2500)], 12, 2), ([(4000, 37)], 32, 8),
                                         ([(100 * i, 37 * i % 90) for i in range(70)], 8, 1)])
def test_prefill_larger(cuda_device, lens, hq, hkv):
    case = prefill_case(lens, hq, hkv, cuda_device)
    close_prompt(run_prefill(*case), *ref.prefill(*case, SCALE)[:2])


@pytest.mark.parametrize("hq,hkv", [(32, 8), (5, 1), (16, 1), (9, 3), (2, 2)])
@pytest.mark.parametrize("new,cached", [(1, 0), (3, 700), (6, 250), (8, 3000)])
def test_prefill_many_requests_with_few_new_tokens(cuda_device, new, cached, hq, hkv):
    """Up to one block of rows each, ragged, with requests that have none, and NaN behind the last ones."""
    lens = [(max(0, cached - 37 * i) + 128 * (i % 3), (new + i) % (new + 2)) for i in range(21)]
    q, k_cache, v_cache, tables, context, starts = prefill_case(lens, hq, hkv, cuda_device, seed=new)
    live = torch.zeros(k_cache.shape[:2], dtype=torch.bool, device=cuda_device)
    for t, n in zip(tables, context):
        for i in range(-(-n // PAGE)):
            live[t[i], :min(PAGE, n - i * PAGE)] = True
    want, size, _ = ref.prefill(q, k_cache, v_cache, tables, context, starts, SCALE)
    k_cache[~live] = v_cache[~live] = float("nan")
    close_prompt(run_prefill(q, k_cache, v_cache, tables, context, starts), want, size)
    assert _native.device_error() == 0


def test_prefill_ignores_what_lies_behind_the_last_token(cuda_device):
    """NaN and infinities behind the context (in its last page, in pages of no request)."""
    lens, dev = [(130, 7), (0, 300), (255, 1), (256, 9)], cuda_device
    q, k_cache, v_cache, tables, context, starts = prefill_case(lens, 8, 2, dev)
    want, size, _ = ref.prefill(q, k_cache, v_cache, tables, context, starts, SCALE)
    live = torch.zeros(k_cache.shape[:2], dtype=torch.bool, device=dev)
    for t, n in zip(tables, context):
        for i in range(-(-n // PAGE)):
            live[t[i], :min(PAGE, n - i * PAGE)] = True
    for fill in (float("nan"), float("inf"), -float("inf")):
        k_cache[~live] = fill
        v_cache[~live] = fill
        close_prompt(run_prefill(q, k_cache, v_cache, tables, context, starts), want, size)


def test_prefill_later_tokens_do_not_matter(cuda_device):
    dev = cuda_device
    q, k_cache, v_cache, tables, context, starts = prefill_case([(200, 300)], 4, 1, dev)
    first = run_prefill(q, k_cache, v_cache, tables, context, starts)
    slot = [tables[0][t // PAGE] * PAGE + t % PAGE for t in range(350, 500)]
    k_cache.flatten(0, 1)[slot] *= -3
    v_cache.flatten(0, 1)[slot] += 100
    second = run_prefill(q, k_cache, v_cache, tables, context, starts)
    assert torch.equal(first[:150], second[:150]) and not torch.equal(first[150:], second[150:])


def test_prefill_rows_of_no_request_and_rows_that_see_nothing(cuda_device):
    dev = cuda_device
    lens = [(100, 20), (0, 10), (50, 30)]
    q, k_cache, v_cache, tables, context, starts = prefill_case(lens, 6, 2, dev, extra_rows=9)
    starts = [s + 4 for s in starts]   # rows before the first request and behind the last
    context[1] = 3                     # of its ten tokens the first seven come before the context
    context[2] = -5
    out = torch.full_like(q, 7.0)
    assert run_prefill(q, k_cache, v_cache, tables, context, starts, out=out) is out
    want, size, rows = ref.prefill(q, k_cache, v_cache, tables, context, starts, SCALE)
    close_prompt(out[rows], want[rows], size[rows])
    assert (out[~rows] == 7).all() and (~rows).sum() == 9
    assert (out[starts[1]:starts[1] + 7] == 0).all() and (out[starts[2]:starts[3]] == 0).all()


def test_prefill_starts_that_fall_or_pass_the_end(cuda_device):
    """Starts count as the running maximum of themselves, cut at the number of rows."""
    dev = cuda_device
    q, k_cache, v_cache, tables, context, starts = prefill_case([(10, 20), (30, 20), (5, 20)], 4, 2, dev)
    out = run_prefill(q, k_cache, v_cache, tables, context, [-3, 20, 10, 1 << 30])
    want, size, rows = ref.prefill(q, k_cache, v_cache, tables, context, [0, 20, 20, 60], SCALE)
    close_prompt(out, want, size)


def test_prefill_bad_pages_and_narrow_tables(cuda_device):
    dev = cuda_device
    q, k_cache, v_cache, tables, context, starts = prefill_case([(600, 40), (300, 8)], 8, 2, dev)
    pages = k_cache.shape[0]
    tables[0][1], tables[1][0] = pages, -1
    out = run_prefill(q, k_cache, v_cache, tables, context, starts)
    assert _native.device_error() == 6
    close_prompt(out, *ref.prefill(q, k_cache, v_cache, tables, context, starts, SCALE)[:2])
    tables = [[1 << 30] * 3, [pages + 7] * 3]
    assert (run_prefill(q, k_cache, v_cache, tables, context, starts) == 0).all()
    assert _native.device_error() == 6
    # a context longer than its table: only what the table names is read
    q, k_cache, v_cache, tables, context, starts = prefill_case([(600, 40)], 4, 1, dev)
    narrow = [tables[0][:1]]
    out = run_prefill(q, k_cache, v_cache, narrow, context, starts)
    close_prompt(out, *ref.prefill(q, k_cache, v_cache, narrow, context, starts, SCALE)[:2])
    _native.device_error()


@pytest.mark.parametrize("factor", [2.0 ** 40, 2.0 ** -40, -1000.0])
def test_prefill_extreme_scores(cuda_device, factor):
    """Scores around 1e13 and more: one token takes all; tiny ones: all take the same."""
    q, k_cache, v_cache, tables, context, starts = prefill_case([(150, 200)], 4, 1, cuda_device)
    # powers of two and whole numbers, so that every score is exact and ties are ties
    q.copy_(torch.sign(q.float()) * 2)
    k_cache.copy_(torch.round(k_cache.float()).clamp(-3, 3) * factor)
    out = run_prefill(q, k_cache, v_cache, tables, context, starts)
    close_prompt(out, *ref.prefill(q, k_cache, v_cache, tables, context, starts, SCALE)[:2])


def test_prefill_scores_that_rise_along_the_context(cuda_device):
    """The maximum moves with every tile, by far: what was summed before becomes nothing."""
    q, k_cache, v_cache, tables, context, starts = prefill_case([(900, 140)], 4, 1, cuda_device)
    q.fill_(1.0)
    for t in range(context[0]):
        k_cache[tables[0][t // PAGE], t % PAGE] = (t // 4) / 8  # exact in BF16
    for scale in (SCALE, 0.001):
        out = run_prefill(q, k_cache, v_cache, tables, context, starts, scale=scale)
        close_prompt(out, *ref.prefill(q, k_cache, v_cache, tables, context, starts, scale)[:2])


def test_prefill_error_is_two_roundings(cuda_device):
    """Each probability's rounding is as large, relative to its share, as the output's own
    and independent of it: together sqrt(2) = 1.414 of the latter, 1.45 with what is left of chance."""
    case = prefill_case([(300, 500)], 8, 2, cuda_device)
    want = ref.prefill(*case, SCALE)[0]
    rounded = (want.bfloat16().double() - want).norm()
    assert (run_prefill(*case).double() - want).norm() <= 1.45 * rounded


def test_prefill_same_whatever_is_beside_it(cuda_device):
    """A request's rows do not depend on the requests beside it beyond the order of sums."""
    q, k_cache, v_cache, tables, context, starts = prefill_case([(777, 60), (0, 400), (5, 5)], 8, 2, cuda_device)
    together = run_prefill(q, k_cache, v_cache, tables, context, starts)
    for b in range(3):
        lo, hi = starts[b], starts[b + 1]
        alone = run_prefill(q[lo:hi].contiguous(), k_cache, v_cache, [tables[b]], [context[b]], [0, hi - lo])
        seen = range(context[b] - (hi - lo) + 1, context[b] + 1)
        want, size = ref.attend(q[lo:hi], k_cache, v_cache, tables[b], seen, SCALE)
        close_prompt(alone, want, size)
        assert (alone.double() - together[lo:hi].double()).norm() <= 2.0 ** -8 * want.norm()


def test_prefill_is_reproducible_and_workspaces_may_be_reused(cuda_device):
    dev = cuda_device
    case = prefill_case([(1500, 60), (3, 90)], 8, 2, dev)
    other = prefill_case([(10, 20)], 8, 2, dev, seed=5)
    ws = prefill_attention_workspace(150, 4, 8, 2, dev)
    ws.fill_(255)
    first = run_prefill(*case, workspace=ws)
    run_prefill(*other, workspace=ws)
    assert torch.equal(first, run_prefill(*case, workspace=ws)) and torch.equal(first, run_prefill(*case))


# ------------------------------------------------------------------ shared prefix
def shared_case(groups, hq, hkv, device, seed=0, before=0, after=0):
    """groups: (prefix, own lengths) each; ``before`` / ``after`` requests of no group around them."""
    counts, context = [], []
    loose = [(0, [40 + 300 * i]) for i in range(before)], [(0, [17 + 260 * i]) for i in range(after)]
    for prefix, own in loose[0] + groups + loose[1]:
        counts += [prefix // PAGE] + [-(-(prefix + n) // PAGE) - prefix // PAGE for n in own]
        context += [prefix + n for n in own]
    lists = page_lists(counts, seed)
    tables, starts, at = [], [before], 0
    for i, (prefix, own) in enumerate(loose[0] + groups + loose[1]):
        tables += [lists[at] + lists[at + 1 + j] for j in range(len(own))]
        at += 1 + len(own)
        if before <= i < before + len(groups):
            starts.append(starts[-1] + len(own))
    k_cache, v_cache = caches(max(1, sum(counts)), hkv, device, seed)
    q = rand((len(tables), hq, D), device, seed)
    return q, k_cache, v_cache, padded(tables), context, starts, [p for p, _ in groups]


def run_shared(q, k_cache, v_cache, tables, context, starts, prefix, **kw):
    dev = q.device
    return shared_prefix_attention(q, k_cache, v_cache, i32(tables, dev), i32(context, dev), i32(starts, dev),
                                   i32(prefix, dev), scale=kw.pop("scale", SCALE), **kw)


def check_shared(case, **kw):
    out = run_shared(*case, **kw)
    ref.assert_attention_close(out, *ref.decode(*case[:5], SCALE))
    return out


GROUPS = [
    [(0, [1])], [(256, [1])], [(256, [1, 2])], [(255, [1, 1, 3])], [(257, [1, 256, 300])], [(512, [0, 4, 0])],
    [(1000, [5] * 9)], [(300, [1, 2]), (0, [3]), (1024, [700, 1, 129, 64]), (100, [1] * 5)],
    [(2048, list(range(1, 34)))], [(768, [1 + 50 * (i % 7) for i in range(70)])],
]


@pytest.mark.parametrize("hq,hkv", [(8, 2), (5, 1), (16, 1), (3, 3), (1, 1)])
@pytest.mark.parametrize("groups", GROUPS, ids=lambda g: "-".join(f"{p}x{len(o)}" for p, o in g))
def test_shared(cuda_device, groups, hq, hkv):
    check_shared(shared_case(groups, hq, hkv, cuda_device, seed=len(groups)))
    assert _native.device_error() == 0


@pytest.mark.parametrize("groups,hq,hkv,around", [([(4096, [100, 7, 256, 30] * 4)], 32, 8, 0),
                                                  ([(3000, [10, 600]), (1500, [256] * 20)], 40, 8, 3)])
def test_shared_larger(cuda_device, groups, hq, hkv, around):
    check_shared(shared_case(groups, hq, hkv, cuda_device, before=around, after=around))


def test_shared_requests_of_no_group_and_padding(cuda_device):
    dev = cuda_device
    q, k_cache, v_cache, tables, context, starts, prefix = shared_case([(600, [3, 4]), (0, []), (256, [5])], 8, 2, dev,
                                                                       before=2, after=3)
    context[-1], context[0] = 0, -4
    out = check_shared((q, k_cache, v_cache, tables, context, starts, prefix))
    assert (out[-1] == 0).all() and (out[0] == 0).all()
    # no groups at all
    check_shared((q, k_cache, v_cache, tables, context, [0], []))
    # every request empty
    assert (run_shared(q, k_cache, v_cache, tables, [0] * len(context), starts, prefix) == 0).all()


def test_shared_prefix_longer_than_some_requests(cuda_device):
    """A request that ends within the prefix, and padding rows inside a group."""
    dev = cuda_device
    q, k_cache, v_cache, tables, context, starts, prefix = shared_case([(1024, [5, 6, 7, 8])], 8, 2, dev)
    context[1], context[2] = 300, 0
    check_shared((q, k_cache, v_cache, tables, context, starts, prefix))
    context[0] = 1
    check_shared((q, k_cache, v_cache, tables, context, starts, [1 << 30]))
    check_shared((q, k_cache, v_cache, tables, context, starts, [-7]))


def test_shared_ignores_what_lies_behind_the_last_token(cuda_device):
    dev = cuda_device
    case = shared_case([(600, [3, 130, 200]), (256, [1, 2])], 8, 2, dev, after=1)
    q, k_cache, v_cache, tables, context, starts, prefix = case
    want, size = ref.decode(*case[:5], SCALE)
    live = torch.zeros(k_cache.shape[:2], dtype=torch.bool, device=dev)
    for t, n in zip(tables, context):
        for i in range(-(-n // PAGE)):
            live[t[i], :min(PAGE, n - i * PAGE)] = True
    for fill in (float("nan"), float("inf")):
        k_cache[~live] = fill
        v_cache[~live] = fill
        ref.assert_attention_close(run_shared(*case), want, size)


def test_shared_bad_pages_and_starts(cuda_device):
    dev = cuda_device
    q, k_cache, v_cache, tables, context, starts, prefix = shared_case([(600, [3, 130, 200]), (256, [1, 2])], 8, 2, dev)
    bad = [list(t) for t in tables]
    for row in bad[:3]:
        row[0] = k_cache.shape[0]  # in the shared part
    bad[4][1] = -1
    out = run_shared(q, k_cache, v_cache, bad, context, starts, prefix)
    assert _native.device_error() == 6
    ref.assert_attention_close(out, *ref.decode(q, k_cache, v_cache, bad, context, SCALE))
    # starts that fall count as their running maximum, cut at the number of requests
    check_shared((q, k_cache, v_cache, tables, context, [-2, 3, 1], [600, 256]))
    check_shared((q, k_cache, v_cache, tables, context, [0, 3, 1 << 30], [600, 256]))
    _native.device_error()


def test_shared_error_is_the_outputs_rounding(cuda_device):
    case = shared_case([(1024, [100 + 3 * i for i in range(32)])], 32, 8, cuda_device)
    want = ref.decode(*case[:5], SCALE)[0]
    rounded = (want.bfloat16().double() - want).norm()
    assert (run_shared(*case).double() - want).norm() <= 1.02 * rounded


def test_shared_agrees_with_the_decode_attention(cuda_device):
    q, k_cache, v_cache, tables, context, starts, prefix = shared_case([(700, [3, 90, 260])], 16, 2, cuda_device)
    out = run_shared(q, k_cache, v_cache, tables, context, starts, prefix)
    other = torch.empty_like(q)
    ws = torch.empty(_native.paged_attention_workspace_bytes(3, 16, len(tables[0])), dtype=torch.uint8, device=q.device)
    _native.paged_decode_attention(q, k_cache, v_cache, i32(tables, q.device), i32(context, q.device), other, ws, SCALE)
    assert (out.double() - other.double()).norm() <= 2.0 ** -7 * other.double().norm()


# ------------------------------------------------------------------ together, streams, graphs
def test_conversation_over_a_shared_prefix(cuda_device):
    """A prompt is appended and attended to; requests take its pages, append what differs,
    attend over both, then decode together: every output against the plain causal attention."""
    dev, hq, hkv = cuda_device, 8, 2
    k_cache, v_cache = caches(24, hkv, dev)
    kw, qw, cos_sin = (1 + rand(D, dev, 1, 0.2)), (1 + rand(D, dev, 2, 0.2)), rotary(4096, 128, dev)

    def step(cached, new, page_lists_, groups=None):
        t = sum(new)
        pages = [p for x in page_lists_ for p in x]
        tab = build_step_tables(i32(cached, dev), i32(new, dev), i32(pages, dev), num_tokens=t, max_pages=8)
        fused = rand((t, hq + 2 * hkv, D), dev, t + sum(cached))
        q, k, v = fused.split([hq, hkv, hkv], 1)
        q = append_kv(q, k, v, cos_sin, tab.positions, tab.slot_mapping, k_cache, v_cache, q_weight=qw, k_weight=kw)
        lists = padded(page_lists_, 8)
        if groups is None:
            out = paged_prefill_attention(q, k_cache, v_cache, tab.block_tables, tab.context_lens, tab.query_starts,
                                          scale=SCALE)
            want = ref.prefill(q, k_cache, v_cache, lists, [c + n for c, n in zip(cached, new)],
                               tab.query_starts.tolist(), SCALE)
        else:
            out = shared_prefix_attention(q, k_cache, v_cache, tab.block_tables, tab.context_lens, i32(groups[0], dev),
                                          i32(groups[1], dev), scale=SCALE)
            want = ref.decode(q, k_cache, v_cache, lists, [c + 1 for c in cached], SCALE)
        ref.assert_attention_close(out, want[0], want[1], terms=1 if groups is None else 2)
        expected, size = ref.norm_rope(k, kw, cos_sin, tab.positions, 1e-6)
        ref.assert_rows_close(k_cache.flatten(0, 1)[tab.slot_mapping.long()], expected, size)

    step([0], [600], [[3, 9, 4]])                      # the shared prompt; two whole pages of it can be shared
    own = [[3, 9, 10], [3, 9, 11, 12], [3, 9, 13]]     # the rest of it is each request's own
    step([512, 512, 512], [120, 300, 90], own)
    cached = [632, 812, 602]
    for _ in range(3):
        step(cached, [1, 1, 1], own, ([0, 3], [600]))
        cached = [c + 1 for c in cached]
    assert _native.device_error() == 0


def test_streams_and_graphs(cuda_device):
    """Another stream than the current one's default, and captured calls that share no
    workspace, replayed with other lengths, tables and groups."""
    dev = cuda_device
    case = shared_case([(600, [3, 130, 200]), (256, [1, 2, 3])], 8, 2, dev)
    pre = prefill_case([(100, 60), (0, 90)], 8, 2, dev)
    q, k, v = views("fused", 6, 8, 2, dev)
    cos_sin = rotary(2000, 128, dev)
    tables, context, starts, prefix = (i32(x, dev) for x in case[3:])
    ptables, pcontext, pstarts = (i32(x, dev) for x in pre[3:])
    positions, slots = torch.arange(6, device=dev), i32([-1] * 6, dev)
    ws = shared_prefix_workspace(6, 2, 8, 2, dev), prefill_attention_workspace(150, 2, 8, 2, dev)

    def calls():
        a = append_kv(q, k, v, cos_sin, positions, slots, case[1], case[2])
        b = shared_prefix_attention(*case[:3], tables, context, starts, prefix, scale=SCALE, workspace=ws[0])
        c = paged_prefill_attention(*pre[:3], ptables, pcontext, pstarts, scale=SCALE, workspace=ws[1])
        return a, b, c

    eager = calls()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = calls()
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(eager, on_side))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = calls()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(eager, captured))
    context.copy_(i32([500, 0, 800, 257, 1, 259], dev))
    starts.copy_(i32([0, 2, 6], dev))
    prefix.copy_(i32([0, 0], dev))
    pcontext.copy_(i32([150, 120], dev))
    pstarts.copy_(i32([0, 100, 150], dev))
    graph.replay()
    torch.cuda.synchronize()
    ref.assert_attention_close(captured[1], *ref.decode(*case[:4], context.tolist(), SCALE))
    want, size, rows = ref.prefill(*pre[:4], pcontext.tolist(), pstarts.tolist(), SCALE)
    close_prompt(captured[2], want, size)
    assert _native.device_error() == 0


def test_two_calls_at_once(cuda_device):
    """Overlapping calls on two streams, a workspace each (here torch's allocator's)."""
    dev = cuda_device
    a, b = prefill_case([(2000, 100)], 8, 2, dev), shared_case([(2048, [30] * 8)], 8, 2, dev, seed=3)
    args_a, args_b = [i32(x, dev) for x in a[3:]], [i32(x, dev) for x in b[3:]]
    want_a = paged_prefill_attention(*a[:3], *args_a, scale=SCALE)
    want_b = shared_prefix_attention(*b[:3], *args_b, scale=SCALE)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(10):
        with torch.cuda.stream(streams[0]):
            outs.append((paged_prefill_attention(*a[:3], *args_a, scale=SCALE), want_a))
        with torch.cuda.stream(streams[1]):
            outs.append((shared_prefix_attention(*b[:3], *args_b, scale=SCALE), want_b))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in outs)
