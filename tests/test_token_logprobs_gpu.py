"""Token log-probabilities against float64 on the CPU."""
import math

import pytest
import torch

from gpu_helpers import Guarded
from nanovllm import _native
from nanovllm.kernels.token_logprobs import TokenLogprobs, token_logprobs

pytestmark = pytest.mark.gpu
INF = math.inf


def reference(x, targets, k):
    """Float64, ties to the lowest index."""
    x = x.double().cpu()
    t, v = x.shape
    top = x.amax(-1, keepdim=True)
    logp = (x - top) - (x - top).exp().sum(-1, keepdim=True).log()  # x - top first: x alone may absorb the logarithm
    p = logp.exp()
    given = (targets >= 0) & (targets < v)
    at = targets.clamp(0, v - 1)[:, None]
    lp = torch.where(given, logp.gather(1, at)[:, 0], torch.zeros(t, dtype=torch.float64))
    ranks = torch.where(given, (x > x.gather(1, at)).sum(-1) + 1, 0)
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
    order = torch.sort(x, dim=-1, descending=True, stable=True)
    ids = order.indices[:, :k]
    top = logp.gather(1, ids)
    if ids.shape[1] < k:
        ids = torch.nn.functional.pad(ids, (0, k - ids.shape[1]), value=-1)
        top = torch.nn.functional.pad(top, (0, k - top.shape[1]), value=-INF)
    gone = top == -INF
    ids = torch.where(gone, -1, ids)
    return lp, ranks, entropy, top, ids


def check(got, x, targets, k):
    lp, ranks, entropy, top, ids = reference(x, targets.cpu(), k)
    assert torch.equal(got.ranks.cpu(), ranks)
    # x - m is exact or off by 2^-24 |x - m|; exp, the sum of up to V terms (pairwise over
    # threads: depth some tens to a few hundred adds) and log add a few 2^-24 each, absolute
    size = x.double().cpu().clamp(-1e4, 1e4).abs().amax(-1) + 1
    tol = 2.0 ** -24 * (16 + 4 * size) + 2e-6
    finite = lp > -INF
    assert torch.equal(got.logprobs.cpu() > -INF, finite)
    assert ((got.logprobs.double().cpu() - lp).abs()[finite] <= (tol + 2.0 ** -23 * lp.abs())[finite]).all()
    assert ((got.entropy.double().cpu() - entropy).abs() <= tol + 2e-6 * entropy).all()
    if k:
        assert torch.equal(got.top_ids.cpu(), ids)
        ok = top > -INF
        assert torch.equal(got.top_logprobs.cpu() > -INF, ok)
        err = (got.top_logprobs.double().cpu() - top).abs()
        assert (err[ok] <= (tol[:, None] + 2.0 ** -23 * top.abs())[ok]).all()
    else:
        assert got.top_ids is None and got.top_logprobs is None


def logits(t, v, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(t, v, generator=g) * spread).to(dtype), torch.randint(0, v, (t,), generator=g)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,v,k", [(1, 1, 1), (1, 7, 3), (3, 31, 32), (5, 255, 20), (2, 256, 5), (2, 257, 32), (4, 1000, 0),
                                   (1, 8191, 20), (33, 4099, 5), (2, 151936, 20), (1, 151937, 32), (300, 2050, 1),
                                   (1, 1000003, 20)])
def test_shapes(cuda_device, dtype, t, v, k):
    x, targets = logits(t, v, dtype, seed=t + v)
    got = token_logprobs(x.to(cuda_device), targets.to(cuda_device), top_k=k)
    check(got, x, targets, k)
    again = token_logprobs(x.to(cuda_device), targets.to(cuda_device), top_k=k)
    assert all(a is None or torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["constant", "rising", "falling", "two values", "one high", "large", "blocks"])
def test_hard_rows(cuda_device, dtype, kind):
    """Ties over the whole row, every order of arrival, peaked and huge logits."""
    t, v, k = 3, 20011, 20
    i = torch.arange(v, dtype=torch.float32)
    x = {"constant": torch.full((v,), -2.5), "rising": i / 100, "falling": -i / 100, "two values": (i % 997 == 3).float(),
         "one high": torch.where(i == 12345, 90.0, -90.0), "large": (i % 13) * 1e4 - 5e4,
         "blocks": (i // 256) % 5}[kind]
    x = torch.stack((x, x.flip(0), x.roll(5000))).to(dtype)
    targets = torch.tensor([12345, 0, v - 1])
    check(token_logprobs(x.to(cuda_device), targets.to(cuda_device), top_k=k), x, targets, k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_equal_logits_over_many_parts(cuda_device, dtype):
    """Every part of a split row holds more candidates than are ranked at once."""
    v, k = 1000003, 32
    x = torch.zeros(2, v, dtype=dtype)
    x[1, 500000:] = 1.0
    targets = torch.tensor([v - 1, 3])
    check(token_logprobs(x.to(cuda_device), targets.to(cuda_device), top_k=k), x, targets, k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masks(cuda_device, dtype):
    """-inf and the type's lowest value, few or no tokens left, targets masked or outside."""
    v, k = 5003, 20
    x, _ = logits(9, v, dtype, seed=4)
    low = torch.finfo(dtype).min
    x[0, torch.rand(v, generator=torch.Generator().manual_seed(1)) < 0.9] = -INF
    x[1, torch.rand(v, generator=torch.Generator().manual_seed(2)) < 0.9] = low
    x[2] = -INF
    x[2, 4000] = 1.5          # one token left
    x[3] = low
    x[3, [17, 4999]] = 0.25   # two left, the rest at the lowest value
    x[4] = -INF               # nothing left
    x[5] = low                # all at the lowest value: uniform
    x[6, ::2] = -INF
    targets = torch.tensor([int(x[0].isinf().logical_not().nonzero()[0]), 5, 4000, 17, 9, 77, 2, -1, v])
    d = token_logprobs(x.to(cuda_device), targets.to(cuda_device), top_k=k)
    rows = [0, 1, 2, 3, 5, 6, 7, 8]
    keep = TokenLogprobs(*(f[rows] for f in d))
    # row 1's target may be at the lowest value: its logprob is then about that value
    check(keep, x[rows], targets[rows], k)
    assert d.logprobs[4].item() == -INF and d.entropy[4].item() == 0.0 and d.ranks[4].item() == 1
    assert (d.top_ids[4] == -1).all() and (d.top_logprobs[4] == -INF).all()
    assert d.logprobs[7].item() == 0 and d.ranks[7].item() == 0 and d.ranks[8].item() == 0
    assert d.logprobs[6].item() == -INF
    assert d.entropy[2].item() == 0 and d.logprobs[2].item() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_nan_and_infinite_rows(cuda_device, dtype):
    v, k = 3001, 5
    x, targets = logits(4, v, dtype, seed=5)
    x[0, 2999] = float("nan")
    x[1, 100] = INF
    x[2, :] = float("nan")
    d = token_logprobs(x.to(cuda_device), targets.to(cuda_device), top_k=k)
    for r in (0, 1, 2):
        assert d.logprobs[r].isnan() and d.entropy[r].isnan()
    assert d.top_logprobs[:2].isnan().all()
    others = x[0].clone()
    others[2999] = -INF
    assert d.top_ids[0].tolist() == torch.sort(others.float(), descending=True, stable=True).indices[:k].tolist()
    assert d.top_ids[1, 0].item() == 100
    assert (d.top_ids[2] == -1).all()
    assert d.ranks[0].item() == 1 + int((x[0] > x[0, targets[0]]).sum())
    check(TokenLogprobs(*(f[3:] for f in d)), x[3:], targets[3:], k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_and_unaligned_rows(cuda_device, dtype):
    """A slice of a padded vocabulary, starting at any element; what lies between the rows is not read into them."""
    wide, targets = logits(6, 3000, dtype, seed=6)
    for lo, hi in ((0, 2995), (1, 2900), (3, 2000), (7, 8)):
        y = wide.clone()
        y[:, :lo] = float("nan")
        y[:, hi:] = float("nan")
        x = y.to(cuda_device)[:, lo:hi]
        t = targets % (hi - lo)
        check(token_logprobs(x, t.to(cuda_device), top_k=4), wide[:, lo:hi], t, 4)


def test_outputs_stay_in_their_bounds(cuda_device):
    t, v, k = 37, 5000, 7
    x, targets = logits(t, v, torch.bfloat16, seed=7)
    outs = [Guarded(s, d, cuda_device, canary=9, fill=-5) for s, d in (
        ((t,), torch.float32), ((t,), torch.int64), ((t,), torch.float32), ((t, k), torch.float32), ((t, k), torch.int64))]
    xd, td = x.to(cuda_device), targets.to(cuda_device)
    lib = _native.load()
    ws = torch.empty(lib.nv4_token_logprobs_workspace_bytes(t, v, k), dtype=torch.uint8, device=cuda_device)
    _native.check(lib.nv4_token_logprobs(xd.data_ptr(), 0, td.data_ptr(), *(o.view.data_ptr() for o in outs[:3]),
                                         outs[3].view.data_ptr(), outs[4].view.data_ptr(), ws.data_ptr(), ws.numel(), t,
                                         v, v, k, torch.cuda.current_stream().cuda_stream), "nv4_token_logprobs")
    check(TokenLogprobs(*(o.view for o in outs)), x, targets, k)
    assert all(o.intact() for o in outs)
    empty = token_logprobs(x[:0].to(cuda_device), targets[:0].to(cuda_device), top_k=k)
    assert empty.logprobs.shape == (0,) and empty.top_ids.shape == (0, k)


def test_beyond_32_bit_offsets(cuda_device):
    """Rows beyond 2^31 elements of the logits."""
    t, v = 15000, 151936
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    x = torch.zeros(t, v, dtype=torch.bfloat16, device=cuda_device)
    last, _ = logits(2, v, torch.bfloat16, seed=8)
    x[-2:] = last.to(cuda_device)
    targets = torch.full((t,), 5, device=cuda_device)
    d = token_logprobs(x, targets, top_k=3)
    check(TokenLogprobs(*(f[-2:] for f in d)), last, targets[-2:], 3)
    assert torch.allclose(d.logprobs[:-2], torch.full_like(d.logprobs[:-2], -math.log(v)), rtol=1e-6)
    assert (d.top_ids[:-2] == torch.arange(3, device=cuda_device)).all()


def test_in_a_graph_and_on_streams(cuda_device):
    x, targets = logits(4, 30001, torch.float32, seed=9)
    xd, td = x.to(cuda_device), targets.to(cuda_device)
    token_logprobs(xd, td, top_k=5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = token_logprobs(xd, td, top_k=5)
    for seed in (10, 11):
        x, targets = logits(4, 30001, torch.float32, seed=seed)
        xd.copy_(x)
        td.copy_(targets)
        graph.replay()
        check(got, x, targets, 5)
    streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], []
    torch.cuda.synchronize()
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(token_logprobs(xd, td, top_k=5))
    torch.cuda.synchronize()
    for o in outs:
        check(o, x, targets, 5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("v", [5003, 40003], ids=["one CTA a row", "split rows"])
@pytest.mark.parametrize("power", [24, 25, 30, 31, 32, 33, 36, 39, 40, 60])
def test_maxima_of_any_size(cuda_device, dtype, v, power):
    """Maxima around and beyond where m - 1 and m - 110 round to m, of either sign, beside zeros, -inf, the type's
    lowest value and the next number below."""
    rows = []
    for m in (2.0 ** power, 1.4 * 2.0 ** power, -(2.0 ** power), -1.4 * 2.0 ** power):
        m = torch.tensor(m, dtype=dtype)
        below = torch.nextafter(m, torch.tensor(-INF, dtype=dtype))
        for other in ([0.0] if m > 0 else []) + [-INF, torch.finfo(dtype).min, below.item(), 2 * m.item() if m < 0 else -m.item()]:
            row = torch.full((v,), other, dtype=dtype)
            row[[3, v // 2, v - 1][:1 + len(rows) % 3]] = m
            rows.append(row)
    x = torch.stack(rows)
    targets = torch.arange(len(rows)) % 2 * 7 + 3  # the maximum, another
    check(token_logprobs(x.to(cuda_device), targets.to(cuda_device), top_k=5), x, targets, 5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_large_maximum_among_ordinary_logits(cuda_device, dtype):
    """A forced token, wherever it stands: logprob 0, entropy 0."""
    x, _ = logits(9, 20000, dtype, seed=12)
    at = torch.tensor([0, 511, 512, 7777, 19999, 8191, 4096, 100, 15000])
    x[torch.arange(9), at] = torch.tensor([2e9, 3e9, 1e10, 1e11, 1e12, 5e9, 2.5e9, 4.3e9, 1e30]).to(dtype)
    got = token_logprobs(x.to(cuda_device), at.to(cuda_device), top_k=3)
    check(got, x, at, 3)
    assert not got.logprobs.any() and not got.entropy.any()
