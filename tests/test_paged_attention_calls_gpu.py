"""How the operators of requests that share cached tokens are called: gradients, inference
mode, the workspaces that captured calls allocate, layouts that are refused."""
import pytest
import torch

from nanovllm import _native
from nanovllm.kernels.paged_attention import append_kv, paged_prefill_attention, shared_prefix_attention
from test_paged_attention_gpu import D, SCALE, caches, i32, prefill_case, rand, rotary, shared_case, views

pytestmark = pytest.mark.gpu


def calls(dev):
    """(function, arguments) of the three, the first for five tokens behind each other."""
    q, k, v = views("separate", 5, 8, 2, dev)
    k_cache, v_cache = caches(2, 2, dev)
    append = dict(q=q, k=k, v=v, cos_sin=rotary(64, 128, dev), positions=torch.arange(5, device=dev),
                  slot_mapping=i32([300, 301, 302, -1, 0], dev), k_cache=k_cache, v_cache=v_cache,
                  q_weight=1 + rand(D, dev, 1, 0.2), k_weight=1 + rand(D, dev, 2, 0.2))
    case = prefill_case([(300, 70), (0, 90)], 8, 2, dev)
    prefill = dict(zip(("q", "k_cache", "v_cache", "block_tables", "context_lens", "query_starts"),
                       (*case[:3], *(i32(x, dev) for x in case[3:]))), scale=SCALE)
    case = shared_case([(600, [3, 130, 200]), (256, [1, 2])], 8, 2, dev)
    shared = dict(zip(("q", "k_cache", "v_cache", "block_tables", "context_lens", "group_starts", "prefix_lens"),
                      (*case[:3], *(i32(x, dev) for x in case[3:]))), scale=SCALE)
    return (append_kv, append), (paged_prefill_attention, prefill), (shared_prefix_attention, shared)


@pytest.mark.parametrize("inference", [False, True])
def test_outputs_are_ordinary_tensors(cuda_device, inference):
    with torch.inference_mode(inference):
        for call, args in calls(cuda_device):
            want = call(**args).clone()
            got = call(**args)
            assert torch.equal(got, want) and got.shape == args["q"].shape and got.dtype == torch.bfloat16
            assert got.is_contiguous() and got.data_ptr() % 32 == 0 and got.is_inference() == inference
            assert got.untyped_storage().nbytes() == got.numel() * 2 and not got.requires_grad


def test_outputs_carry_no_gradient(cuda_device):
    for call, args in calls(cuda_device):
        want = call(**args)
        leaf = {n: x.clone().requires_grad_() for n, x in args.items()
                if n in ("q", "k", "v", "q_weight", "k_weight")}
        got = call(**(args | leaf))
        assert torch.equal(got, want) and not got.requires_grad and got.grad_fn is None


def test_captured_calls_allocate_their_own_workspaces(cuda_device):
    """Two graphs, replayed in turn and over new lengths, without one handed in."""
    table = calls(cuda_device)
    graphs = []
    for call, args in table:
        call(**args)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = call(**args), call(**args)
        graphs.append((graph, outs))
    table[1][1]["context_lens"].copy_(i32([333, 90], cuda_device))
    table[2][1]["context_lens"].copy_(i32([601, 0, 800, 257, 258], cuda_device))
    table[0][1]["positions"].add_(3)
    for _ in range(3):
        for graph, _ in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for (call, args), (_, outs) in zip(table, graphs):
        assert all(torch.equal(x, call(**args)) for x in outs)
    assert _native.device_error() == 0


def test_layouts_that_are_refused(cuda_device):
    """Strided queries, caches, tables and outputs of the attentions; overlapping or unaligned tokens of the append."""
    dev = cuda_device
    (append, a), (prefill, p), (shared, s) = calls(dev)

    def other(x):  # the same shape in other strides
        return torch.empty(*x.shape[:-1], 2 * x.shape[-1], dtype=x.dtype, device=dev)[..., ::2]

    for call, args in ((prefill, p), (shared, s)):
        for name in [n for n in args if n != "scale"]:
            with pytest.raises(ValueError):
                call(**(args | {name: other(args[name])}))
            with pytest.raises(ValueError):
                call(**(args | {name: args[name].cpu()}))
        out = torch.empty_like(args["q"])
        off = torch.empty(out.numel() + 8, dtype=out.dtype, device=dev)[8:].view(out.shape)  # 16 bytes off 32
        for bad in (dict(out=other(out)), dict(out=args["q"]), dict(out=off),
                    dict(workspace=torch.empty(64, dtype=torch.uint8, device=dev))):
            with pytest.raises(ValueError):
                call(**(args | bad))
    token = a["k"][:1].expand(5, 2, D)                                    # every token the same memory
    odd = rand((5, 2 * D + 4), dev, 3)[:, :2 * D].unflatten(1, (2, D))    # 4 channels, 8 bytes, further on
    swapped = a["k"].transpose(0, 1).contiguous().transpose(0, 1)         # heads further apart than a row
    for bad in (token, odd, swapped):
        for name in ("k", "v"):
            with pytest.raises(ValueError):
                append(**(a | {name: bad}))
    for name in ("cos_sin", "positions", "slot_mapping", "k_cache", "v_cache", "q_weight"):
        with pytest.raises(ValueError):
            append(**(a | {name: other(a[name])}))
        with pytest.raises(ValueError):
            append(**(a | {name: a[name].cpu()}))
    fused = rand((5, 8 + 2 + 2, D), dev, 4)
    with pytest.raises(ValueError):  # q in place in a fused projection: tokens apart
        append(**(a | dict(q=fused[:, :8], q_out=fused[:, :8])))
    assert _native.device_error() == 0
