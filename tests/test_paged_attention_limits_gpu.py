"""The operators of requests that share cached tokens where test_paged_attention_gpu.py
does not go: waits that give up, and the sizes at which the kernels take other branches."""
import pytest
import torch

import paged_reference as ref
from nanovllm import _native
from test_paged_attention_gpu import PAGE, SCALE, prefill_case, run_prefill, run_shared, shared_case

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

