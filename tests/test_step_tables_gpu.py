"""Step tables built on the GPU against the engine's own lists (Sequence.slot and
the padded page lists)."""
import os
import subprocess
import sys

import pytest
import torch

from gpu_helpers import Guarded
from nanovllm import _native
from nanovllm.kernels.step_tables import StepTables, alloc_step_tables, build_step_tables

pytestmark = pytest.mark.gpu


def expected(cached, new, pages, max_pages, page_size, rows, tokens):
    tables, slots, positions, starts, at = [], [], [], [0], 0
    for c, n in zip(cached, new):
        count = -(-(c + n) // page_size)
        own = pages[at:at + count]
        at += count
        tables.append((own + [0] * max_pages)[:max_pages])
        positions += list(range(c, c + n))
        slots += [own[p // page_size] * page_size + p % page_size for p in range(c, c + n)]
        starts.append(len(slots))
    pad = rows - len(cached)
    return (torch.tensor(tables + [[0] * max_pages] * pad, dtype=torch.int32),
            torch.tensor([c + n for c, n in zip(cached, new)] + [0] * pad, dtype=torch.int32),
            torch.tensor(slots + [-1] * (tokens - len(slots)), dtype=torch.int32),
            torch.tensor(positions + [0] * (tokens - len(slots)), dtype=torch.int64),
            torch.tensor(starts + [len(slots)] * pad, dtype=torch.int32))


def guarded(rows, tokens, max_pages, device):
    make = lambda shape, dtype: Guarded(shape, dtype, device, canary=12345, fill=-77)  # noqa: E731
    return [make((rows, max_pages), torch.int32), make((rows,), torch.int32), make((tokens,), torch.int32),
            make((tokens,), torch.int64), make((rows + 1,), torch.int32)]


CASES = [  # cached, new, page_size
    ([0], [1], 256), ([255], [1], 256), ([256], [1], 256), ([0], [257], 256), ([5, 0, 0, 300], [1, 0, 700, 1], 256),
    ([0, 0, 0], [0, 0, 0], 256), ([7, 9, 0], [3, 0, 5], 1), ([100, 3], [28, 61], 16), ([10, 20, 30], [5, 5, 5], 7),
    ([(37 * i) % 2000 for i in range(513)], [1] * 513, 256), ([0] * 1000, [(13 * i) % 40 for i in range(1000)], 256),
    ([3 * i for i in range(4097)], [i % 3 for i in range(4097)], 256), ([i % 700 for i in range(28672)], [1] * 28672, 256)]


@pytest.mark.parametrize("cached,new,page_size", CASES, ids=range(len(CASES)))
@pytest.mark.parametrize("padding", [0, 5])
def test_against_lists(cuda_device, cached, new, page_size, padding):
    need = [-(-(c + n) // page_size) for c, n in zip(cached, new)]
    pages = torch.randperm(sum(need) + 10, generator=torch.Generator().manual_seed(len(cached))).tolist()
    max_pages, tokens, rows = max(max(need), 1) + 1, sum(new) + padding, len(cached) + padding
    outs = guarded(rows, tokens, max_pages, cuda_device)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)  # noqa: E731
    c, n, p = dev(cached), dev(new), dev(pages)
    got = build_step_tables(c, n, p, num_tokens=sum(new), max_pages=max_pages, page_size=page_size,
                            out=StepTables(*(o.view for o in outs)))
    for o, want, name in zip(got, expected(cached, new, pages, max_pages, page_size, rows, tokens), StepTables._fields):
        assert torch.equal(o.cpu(), want), name
    assert all(o.intact() for o in outs)
    assert torch.equal(p.cpu(), torch.tensor(pages, dtype=torch.int32))
    plain = build_step_tables(c, n, p, num_tokens=sum(new), max_pages=max_pages, page_size=page_size)
    assert torch.equal(plain.slot_mapping, got.slot_mapping[:sum(new)])
    assert torch.equal(plain.block_tables, got.block_tables[:len(cached)])
    assert _native.device_error() == 0


def test_missing_and_bad_pages(cuda_device):
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)  # noqa: E731
    # request 0 needs 2 pages (one negative), request 1 needs 2, of which one is not listed
    t = build_step_tables(dev([250, 0]), dev([8, 300]), dev([4, -3, 9]), num_tokens=308, max_pages=3)
    assert _native.device_error() == 6
    assert t.slot_mapping[:8].tolist() == [4 * 256 + 250 + i for i in range(6)] + [-1, -1]
    assert t.slot_mapping[8:264].tolist() == list(range(9 * 256, 10 * 256)) and (t.slot_mapping[264:] == -1).all()
    assert t.block_tables.tolist() == [[4, -3, 0], [9, 0, 0]]
    assert t.positions[-1].item() == 299 and t.context_lens.tolist() == [258, 300]
    # a context longer than the table, a page whose slots pass 31 bits, negative lengths
    t = build_step_tables(dev([0, -4, 255]), dev([513, 3, -1]), dev([1, 2, 3, 2 ** 24, 7]), num_tokens=516, max_pages=2)
    assert _native.device_error() == 6
    assert (t.slot_mapping[:512] >= 0).all() and t.slot_mapping[512].item() == -1
    assert (t.slot_mapping[513:] == -1).all()  # page 2^24 * 256 has no 32-bit slot
    assert t.context_lens.tolist() == [513, 3, 255] and t.query_starts.tolist() == [0, 513, 516, 516]
    # fewer tokens asked for than there are: the rest is dropped
    t = build_step_tables(dev([0]), dev([10]), dev([5]), num_tokens=4, max_pages=1)
    assert t.slot_mapping.tolist() == [1280, 1281, 1282, 1283] and t.query_starts.tolist() == [0, 10]
    assert _native.device_error() == 0
    # lengths whose sum passes 32 bits
    t = build_step_tables(dev([2 ** 31 - 1] * 3), dev([2 ** 31 - 1, 1, 5]), dev([]), num_tokens=2, max_pages=1,
                          page_size=2 ** 24)
    assert _native.device_error() == 6
    assert t.slot_mapping.tolist() == [-1, -1] and t.context_lens[0].item() == 2 ** 31 - 1


def test_in_a_graph(cuda_device):
    b, max_pages = 6, 4
    cached, new = (torch.zeros(b, dtype=torch.int32, device=cuda_device) for _ in range(2))
    pages = torch.arange(100, 100 + b * max_pages, dtype=torch.int32, device=cuda_device)
    out = alloc_step_tables(b, b, max_pages, cuda_device)
    call = lambda: build_step_tables(cached, new, pages, num_tokens=b, max_pages=max_pages, out=out)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for lens in ([1, 256, 300, 1000, 0, 5], [700, 2, 2, 2, 513, 0]):
        ones = [int(i < 5) for i in range(b)]
        cached.copy_(torch.tensor(lens, dtype=torch.int32))
        new.copy_(torch.tensor(ones, dtype=torch.int32))
        graph.replay()
        for o, want in zip(out, expected(lens, ones, pages.tolist(), max_pages, 256, b, b)):
            assert torch.equal(o.cpu(), want)


def test_batches_around_48_kb_of_shared_memory(cuda_device):
    """In a process of its own, so that no larger batch came before."""
    program = """
import sys, torch
sys.path[:0] = sys.argv[1:]
from nanovllm.kernels.step_tables import build_step_tables
for b in (6128, 6143, 6127, 6142, 6144, 28672, 1):
    one = torch.ones(b, dtype=torch.int32, device="cuda")
    pages = torch.arange(b, dtype=torch.int32, device="cuda")
    t = build_step_tables(one, one, pages, num_tokens=b, max_pages=1)
    assert torch.equal(t.block_tables[:, 0], pages) and (t.context_lens == 2).all() and (t.positions == 1).all(), b
    assert torch.equal(t.slot_mapping, pages * 256 + 1), b
    assert torch.equal(t.query_starts, torch.arange(b + 1, dtype=torch.int32, device="cuda")), b
"""
    package = os.path.dirname(os.path.dirname(os.path.abspath(_native.__file__)))
    done = subprocess.run([sys.executable, "-c", program, package], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
