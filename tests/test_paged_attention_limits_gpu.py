"""The operators of requests that share cached tokens where test_paged_attention_gpu.py
does not go: waits that give up, and the sizes at which the kernels take other branches."""
import pytest
import torch

import paged_reference as ref
from nanovllm import _native
from test_paged_attention_gpu import D, PAGE, SCALE, caches, prefill_case, rand, run_prefill, run_shared, shared_case

pytestmark = pytest.mark.gpu

PEER_TIMEOUT = 5


def absent_pages(case):
    """Some pages outside the cache: tiles of no keys among tiles of some."""
    tables = [list(t) for t in case[3]]
    for b in range(0, len(tables), 3):
        tables[b][max(0, case[4][b] - 1) // PAGE] = -1
    return (*case[:3], tables, *case[4:])


GIVEN_UP = {
    "prompts side by side": lambda d: (run_prefill, prefill_case(
        [(37 * i, 700 - 13 * i) for i in range(6)], 32, 8, d)),
    "short prompts": lambda d: (run_prefill, prefill_case([(11 * i % 700, 1 + i % 9) for i in range(300)], 8, 2, d)),
    "decode": lambda d: (run_shared, shared_case([(600, [3 + i for i in range(9)])] * 9, 16, 4, d, before=5, after=5)),
}


@pytest.mark.parametrize("name", GIVEN_UP)
def test_a_wait_that_gave_up_ends_the_call(cuda_device, name):
    """An earlier wait ran out (a peer that never comes) and its error has not been read: waits of later calls
    give up as soon as they would have to go on waiting.  The call ends whatever it computes; once the error is
    read the next one is right again."""
    call, case = GIVEN_UP[name](cuda_device)
    cases = case, absent_pages(case)
    want = [call(*c) for c in cases]
    assert _native.device_error() == 6
    buffers = [_native.peer_buffer_alloc(32 * 4096, cuda_device)[0] for _ in range(2)]
    x = torch.zeros(32 * 4096, dtype=torch.bfloat16, device=cuda_device)
    try:
        _native.peer_allreduce_bf16(buffers, 0, x, x.numel(), 32 * 4096)
        for _ in range(3):
            for c in cases:
                call(*c)
        assert _native.device_error() == PEER_TIMEOUT
    finally:
        torch.cuda.synchronize()
        for b in buffers:
            _native.peer_buffer_free(b, cuda_device)
    assert all(torch.equal(call(*c), w) for c, w in zip(cases, want))
    assert _native.device_error() == 6


# ------------------------------------------------------------------ many requests and heads
def check_shared(case):
    out = run_shared(*case)
    ref.assert_attention_close(out, *ref.decode(*case[:5], SCALE))
    assert _native.device_error() == 0


def check_prefill(case):
    out = run_prefill(*case)
    ref.assert_attention_close(out, *ref.prefill(*case, SCALE)[:2], terms=1)
    assert _native.device_error() == 0


RAGGED = [(1000, [5, 90, 3, 700]), (700, [1 + 7 * i for i in range(40)]), (2000, [4, 4]), (100, [3, 600, 2]),
          (256, [1 + 3 * i % 50 for i in range(70)]), (3000, [10, 300, 20])]


@pytest.mark.parametrize("hq,hkv,copies", [(32, 8, 1), (8, 8, 1), (48, 3, 1), (10, 2, 2)])
def test_shared_join_of_many_rows(cuda_device, hq, hkv, copies):
    """More (request, KV head) pairs than are joined by 512 threads each: groups of at most a quarter of a block's
    rows and larger ones, cut and whole blocks, padding, requests of no group."""
    case = shared_case(RAGGED * copies, hq, hkv, cuda_device, seed=hq, before=3, after=6)
    assert len(case[4]) * hkv > 2 * 160
    for b in (0, 9, 20, len(case[4]) - 1):
        case[4][b] = 0
    check_shared(case)


@pytest.mark.parametrize("hq,hkv", [(32, 8), (48, 3)])
def test_shared_join_of_many_rows_in_whole_blocks(cuda_device, hq, hkv):
    """Blocks of a tile or two: most are not cut."""
    case = shared_case([(256, [1 + (i + j) % 40 for i in range(2 + j % 5)]) for j in range(30)], hq, hkv, cuda_device)
    assert len(case[4]) * hkv > 2 * 160
    check_shared(case)


def many_prompts(count, most, hq, hkv, device, seed=0):
    """Ragged prompts: some without new tokens, some with nothing cached, some with a context that is none."""
    lens = [((7 * i + 300 * (i % 61 == 0)) % 500 if i % 3 else 0, i % (most + 1)) for i in range(count)]
    case = prefill_case(lens, hq, hkv, device, seed=seed)
    for b in range(0, count, 97):
        case[4][b] = -b
    return case


@pytest.mark.parametrize("count,most,hq,hkv", [(513, 2, 2, 1), (1100, 5, 2, 1), (1100, 5, 6, 2), (3000, 3, 3, 1),
                                               (600, 40, 16, 1), (1030, 25, 16, 1)])
def test_prefill_of_many_requests(cuda_device, count, most, hq, hkv):
    """More than the threads of the block table's CTA, once, twice and four times; with 16 heads more rows a request
    than a block has, and with 3000 requests more blocks than the table keeps on the chip."""
    check_prefill(many_prompts(count, most, hq, hkv, cuda_device))


def many_groups(groups, device, hq, hkv, prefix=1):
    """Groups of no to three requests, every seventh without a prefix, and requests of no group between some."""
    case = shared_case([(prefix * PAGE + 3 if i % 7 else 0, [1 + (i + j) % 9 for j in range(i % 4)])
                        for i in range(groups)], hq, hkv, device, before=2, after=2)
    for b in range(0, len(case[4]), 53):
        case[4][b] = 0
    return case


@pytest.mark.parametrize("groups,hq,hkv", [(511, 2, 1), (513, 4, 2), (1300, 2, 1)])
def test_shared_of_many_groups(cuda_device, groups, hq, hkv):
    """As many passes over the groups and requests; with 1300 groups more than 2048 blocks."""
    case = many_groups(groups, cuda_device, hq, hkv)
    of_prefix = sum(i % 7 > 0 and i % 4 > 1 for i in range(groups))  # a block each, but for padded rows
    assert groups < 1300 or len(case[4]) + of_prefix > 2048 + 100
    check_shared(case)


def test_shared_of_one_large_group(cuda_device):
    """2100 requests over one page, 17 blocks of prefix rows."""
    case = shared_case([(PAGE, [1 + i % 5 for i in range(2100)])], 1, 1, cuda_device)
    check_shared(case)


# ------------------------------------------------------------------ long walks
def long_case(batch, new, pages, hq, hkv, device, seed=0):
    """Contexts of so many pages each, all but a few of which name the same page, whose keys lie so far off that
    their probabilities are zero: the rest is the whole of the result, wherever the walks are cut.  A page behind
    the few holds the new tokens' keys and values, as far off."""
    few = 6
    g = torch.Generator().manual_seed(seed)
    k_cache, v_cache = caches(few + 1, hkv, device, seed)
    k_cache[..., 0] = 0
    k_cache[few] = 0
    k_cache[few, ..., 0] = -16384.0  # a score of -23,000 and more: exp(-23,000) is zero in FP32 and FP64
    q = rand((batch * new, hq, D), device, seed)
    q[..., 0] = 16.0
    tables, real = [[few] * pages for _ in range(batch)], []
    for b in range(batch):
        at = sorted(set(torch.randint(0, pages - 2, (4,), generator=g).tolist()))
        real.append([int(x) for x in torch.randint(0, few, (len(at),), generator=g)])
        for i, page in zip(at, real[-1]):
            tables[b][i] = page
    return q, k_cache, v_cache, tables, [pages * PAGE] * batch, real


@pytest.mark.parametrize("batch,hq,hkv,pages", [(256, 16, 8, 260), (270, 4, 1, 2000)])
def test_shared_walks_of_a_million_tiles(cuda_device, batch, hq, hkv, pages):
    """Costs that are divided in 64 bits, joined in both ways."""
    q, k_cache, v_cache, tables, context, real = long_case(batch, 1, pages, hq, hkv, cuda_device)
    assert batch * hkv * pages * 2 > 1 << 20
    out = run_shared(q, k_cache, v_cache, tables, context, [0], [])
    ref.assert_attention_close(out, *ref.decode(q, k_cache, v_cache, real, [PAGE * len(x) for x in real], SCALE))
    assert _native.device_error() == 0


@pytest.mark.parametrize("batch,new,hq,hkv,pages", [(300, 1, 8, 8, 230), (16, 130, 32, 8, 1800)])
def test_prefill_walks_of_a_million_tiles(cuda_device, batch, new, hq, hkv, pages):
    q, k_cache, v_cache, tables, context, real = long_case(batch, new, pages, hq, hkv, cuda_device)
    rows = 128 * hkv // hq * (2 if new > 128 * hkv // hq else 1)  # tokens of a block, or of two side by side
    assert batch * hkv * -(-new // rows) * (pages * 2 - 1) > 1 << 20
    out = run_prefill(q, k_cache, v_cache, tables, context, [new * b for b in range(batch + 1)])
    parts = [ref.attend(q[b * new:(b + 1) * new], k_cache, v_cache, real[b], [PAGE * len(real[b])] * new, SCALE)
             for b in range(batch)]
    ref.assert_attention_close(out, *(torch.cat(x) for x in zip(*parts)), terms=1)
    assert _native.device_error() == 0
