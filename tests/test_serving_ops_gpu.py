"""What the Python entry points of the 4-bit cache, the step tables and the
log-probabilities refuse on a GPU, before any launch: tensors of another device,
not contiguous or not aligned; and their use on other streams."""
import io

import pytest
import torch

from nanovllm import _native
from nanovllm.kernels.kv4_cache import (alloc_kv4_cache, kv4_attention_workspace, paged_decode_attention_kv4,
                                        qk_norm_rope_store_kv4)
from nanovllm.kernels.step_tables import alloc_step_tables, build_step_tables
from nanovllm.kernels.token_logprobs import token_logprobs

pytestmark = pytest.mark.gpu


def shifted(x):
    """The same values, one element behind an aligned address."""
    y = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)[1:].view(x.shape)
    return y.copy_(x)


def spaced(x):
    """The same values, not contiguous."""
    return torch.stack([x, x], dim=-1)[..., 0]


def variants(x):
    return x.cpu(), spaced(x)


def calls(dev):
    cache = alloc_kv4_cache(4, 2, dev)
    for c in cache:
        c.zero_()
    t, hq, hkv = 3, 4, 2
    store = dict(qkv=torch.randn(t, (hq + 2 * hkv) * 128, device=dev).bfloat16(),
                 q_weight=torch.ones(128, device=dev).bfloat16(), k_weight=torch.ones(128, device=dev).bfloat16(),
                 cos_sin=torch.ones(16, 128, device=dev), positions=torch.arange(t, device=dev),
                 slot_mapping=torch.arange(t, dtype=torch.int32, device=dev))
    attend = dict(q=torch.randn(2, hq, 128, device=dev).bfloat16(),
                  block_tables=torch.zeros(2, 2, dtype=torch.int32, device=dev),
                  context_lens=torch.ones(2, dtype=torch.int32, device=dev))
    tables = dict(cached_lens=torch.tensor([3, 300], dtype=torch.int32, device=dev),
                  new_lens=torch.tensor([2, 1], dtype=torch.int32, device=dev),
                  pages=torch.arange(3, dtype=torch.int32, device=dev))
    probs = dict(logits=torch.randn(4, 100, device=dev), targets=torch.arange(4, device=dev))
    return cache, [(lambda **a: qk_norm_rope_store_kv4(cache=cache, num_heads=hq, num_kv_heads=hkv, eps=1e-6, **a), store),
                   (lambda **a: paged_decode_attention_kv4(cache=cache, scale=0.1, **a), attend),
                   (lambda **a: build_step_tables(num_tokens=3, max_pages=2, **a), tables),
                   (lambda **a: token_logprobs(top_k=3, **a), probs)]


@pytest.mark.parametrize("which", range(4))
def test_other_devices_and_strides(cuda_device, which):
    _, table = calls(cuda_device)
    call, args = table[which]
    call(**args)
    for name, x in args.items():
        for bad in variants(x):
            with pytest.raises(ValueError, match="contiguous"):
                call(**(args | {name: bad}))
    assert _native.device_error() == 0


def test_alignment(cuda_device):
    """Vector loads need 16 bytes: refused, but for logits, whose rows may start anywhere."""
    cache, table = calls(cuda_device)
    for which, names in ((0, ("qkv", "q_weight", "k_weight", "cos_sin")), (1, ("q",))):
        call, args = table[which]
        for name in names:
            with pytest.raises(ValueError):
                call(**(args | {name: shifted(args[name])}))
    call, args = table[3]
    want, got = call(**args), call(**(args | dict(logits=shifted(args["logits"]))))
    assert torch.equal(want.top_ids, got.top_ids) and torch.equal(want.ranks, got.ranks)
    torch.testing.assert_close(want.logprobs, got.logprobs)


def test_outputs_and_workspaces(cuda_device):
    cache, table = calls(cuda_device)
    call, args = table[1]
    q = args["q"]
    for out in (torch.empty_like(q).cpu(), spaced(q), torch.empty_like(q)[:1], torch.empty_like(q).float(), shifted(q)):
        with pytest.raises(ValueError):
            call(**args, out=out)
    ws = kv4_attention_workspace(2, 4, 2, cuda_device)
    for bad in (ws[:-16], ws.cpu(), shifted(ws)):
        with pytest.raises(ValueError):
            call(**args, workspace=bad)
    call, args = table[2]
    good = alloc_step_tables(3, 5, 2, cuda_device)
    call(**args, out=good)
    for name, x in good._asdict().items():
        for bad in (x.cpu(), spaced(x), x[:1]):
            with pytest.raises(ValueError):
                call(**args, out=good._replace(**{name: bad}))
    assert _native.device_error() == 0


def test_two_streams_at_once(cuda_device):
    """The four calls on two streams, with no synchronisation between them, give what one stream gives."""
    _, table = calls(cuda_device)
    big = [(table[1][0], dict(q=torch.randn(64, 16, 128, device=cuda_device).bfloat16(),
                              block_tables=torch.randint(0, 4, (64, 16), dtype=torch.int32, device=cuda_device),
                              context_lens=torch.randint(0, 4096, (64,), dtype=torch.int32, device=cuda_device))),
           (table[3][0], dict(logits=torch.randn(7, 50003, device=cuda_device), targets=torch.arange(7, device=cuda_device))),
           table[2]]
    flat = lambda r: [r] if torch.is_tensor(r) else list(r)
    want = [[x.clone() for x in flat(c(**a))] for c, a in big]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda_device) for _ in range(2)]
    kept = []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                kept.append([flat(c(**a)) for c, a in big])
    torch.cuda.synchronize()
    for run in kept:
        for got, wanted in zip(run, want):
            assert all(torch.equal(x, y) for x, y in zip(got, wanted))
    assert _native.device_error() == 0


@pytest.mark.parametrize("inference", [False, True])
def test_outputs_are_ordinary_tensors(cuda_device, inference):
    """Contiguous, aligned, apart from one another, alive after the others are gone; writable and copyable."""
    with torch.inference_mode(inference):
        _, table = calls(cuda_device)
        for which, types in ((2, [torch.int32, torch.int32, torch.int32, torch.int64, torch.int32]),
                             (3, [torch.float32, torch.int64, torch.float32, torch.float32, torch.int64])):
            call, args = table[which]
            want = [x.clone() for x in call(**args)]
            got = list(call(**args))
            spans = sorted((x.data_ptr(), x.data_ptr() + x.numel() * x.element_size()) for x in got)
            assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
            for x, t in zip(got, types):
                assert x.dtype == t and x.is_contiguous() and x.data_ptr() % 16 == 0 and x.device == cuda_device
                assert not x.requires_grad and x.is_inference() == inference
            first = got[0]
            first.fill_(7)
            assert all(torch.equal(x, y) for x, y in zip(got[1:], want[1:]))
            last = got[-1]
            del got
            other = [torch.full((1 << 12,), -1, dtype=torch.int32, device=cuda_device) for _ in range(8)]
            assert torch.equal(last, want[-1]) and (first == 7).all() and len(other) == 8
            assert torch.equal(last.reshape(-1).cpu(), want[-1].reshape(-1).cpu())
            assert (last[1:].contiguous() == want[-1][1:]).all()
    none = token_logprobs(torch.empty(0, 10, device=cuda_device), torch.empty(0, dtype=torch.int64, device=cuda_device), top_k=2)
    assert [tuple(x.shape) for x in none] == [(0,), (0,), (0,), (0, 2), (0, 2)]
    for over in (dict(max_pages=(1 << 24) + 1), dict(num_tokens=(1 << 30) + 1)):
        with pytest.raises(ValueError):
            build_step_tables(**table[2][1], **(dict(num_tokens=3, max_pages=2) | over))


def test_outputs_in_a_captured_graph(cuda_device):
    _, table = calls(cuda_device)
    args, probs = table[2][1], table[3][1]
    table[2][0](**args), table[3][0](**probs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tables, found = table[2][0](**args), table[3][0](**probs)
    args["cached_lens"].copy_(torch.tensor([7, 400], dtype=torch.int32))
    probs["logits"].copy_(torch.randn(4, 100, device=cuda_device))
    graph.replay()
    for got, want in ((tables, table[2][0](**args)), (found, table[3][0](**probs))):
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_outputs_have_storage_of_their_own(cuda_device):
    """They can be saved together, and one that is kept keeps no other alive."""
    _, table = calls(cuda_device)
    for which in (2, 3):
        call, args = table[which]
        got = list(call(**args))
        for x in got:
            assert x.untyped_storage().nbytes() == x.numel() * x.element_size() and x.storage_offset() == 0
        assert len({x.untyped_storage().data_ptr() for x in got}) == len(got)
        file = io.BytesIO()
        torch.save(got, file)
        file.seek(0)
        assert all(torch.equal(a, b) for a, b in zip(torch.load(file), got))


def test_step_tables_in_place_are_refused(cuda_device):
    """Advancing a batch in place: the lengths may not be both input and output."""
    _, table = calls(cuda_device)
    call, args = table[2]
    good = alloc_step_tables(2, 3, 2, cuda_device)
    for out in (good._replace(context_lens=args["cached_lens"]), good._replace(context_lens=args["new_lens"]),
                good._replace(query_starts=args["pages"]), good._replace(slot_mapping=good.query_starts)):
        with pytest.raises(ValueError):
            call(**args, out=out)
    want = call(**args)
    assert all(torch.equal(a, b) for a, b in zip(call(**args, out=good), want))


def test_returned_values_are_the_caches_rounded_to_bf16(cuda_device):
    """The decode attention reads code * scale unrounded, up to 11 significant bits."""
    import kv4_reference as ref
    cache, table = calls(cuda_device)
    call, args = table[0]
    _, k, v = call(**args, return_values=True)
    for got, held in ((k, ref.read_k(cache)), (v, ref.read_v(cache))):
        held = held[0, :, :3].transpose(0, 1)
        got = got.cpu()
        assert torch.equal(got, held.bfloat16()) and not torch.equal(got.double(), held)
        assert ((got.double() - held).abs() <= 2.0 ** -8 * held.abs()).all()


def test_logprobs_of_logits_that_require_a_gradient(cuda_device):
    _, table = calls(cuda_device)
    call, args = table[3]
    got = call(**(args | dict(logits=args["logits"].clone().requires_grad_())))
    assert all(torch.equal(a, b) and not a.requires_grad for a, b in zip(got, call(**args)))
