"""The operators of requests that share cached tokens, in 64 bits and from their
definitions, with the bounds their tests use."""
import torch

D, PAGE = 128, 256


def norm_rope(x, weight, cos_sin, positions, eps):
    """float64 (values, sizes) of [T, H, 128]: size bounds what the rotation adds up."""
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    cos, sin = cos_sin.double()[positions].unsqueeze(1).chunk(2, -1)
    half = cos.shape[-1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return (torch.cat((a * cos - b * sin, b * cos + a * sin, rest), -1),
            torch.cat((a.abs() + b.abs(), a.abs() + b.abs(), rest.abs()), -1))


def assert_rows_close(got, ref, size):
    """BF16's rounding is off by 2^-8 of the value at most; 2^-18 of the addends covers
    the FP32 steps before it (a sum of 128 squares, rsqrt, two products, one sum)."""
    bound = 2.0 ** -8 * ref.abs() + 2.0 ** -18 * size + 1e-38
    worst = ((got.double() - ref).abs() / bound).max().item()
    assert torch.isfinite(got).all() and worst <= 1.0, worst


def attend(q, k_cache, v_cache, table, seen, scale):
    """(out, sum p |v|) in float64 of queries q [n, Hq, 128] of one request, query i
    over the first seen[i] tokens that ``table`` names (pages outside the cache hold none)."""
    n, hq, _ = q.shape
    pages, _, hkv, _ = k_cache.shape
    most = max([0] + [min(int(s), len(table) * PAGE) for s in seen])
    out = torch.zeros(n, hq, D, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    if not most:
        return out, size
    token = torch.arange(most, device=q.device)
    page = torch.as_tensor(table, device=q.device).long()[token // PAGE]
    there = (page >= 0) & (page < pages)
    page = page.clamp(0, pages - 1)
    seen = torch.as_tensor([int(s) for s in seen], device=q.device)
    mask = there & (token[None] < seen[:, None])
    for h in range(hkv):
        of = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
        k, v = (c[page, token % PAGE, h].double() for c in (k_cache, v_cache))
        scores = torch.einsum("ngd,td->gnt", q[:, of].double(), k) * scale
        p = torch.softmax(scores.masked_fill(~mask, -float("inf")), -1)
        p = torch.where(mask.any(-1)[:, None], p, 0.0)
        out[:, of] = torch.einsum("gnt,td->ngd", p, v)
        size[:, of] = torch.einsum("gnt,td->ngd", p, v.abs())
    return out, size


def prefill(q, k_cache, v_cache, tables, context, starts, scale):
    """(out, size, rows that belong to a request)."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    size, rows = torch.zeros_like(out), torch.zeros(q.shape[0], dtype=torch.bool, device=q.device)
    for b, ctx in enumerate(context):
        lo, hi = starts[b], starts[b + 1]
        if hi > lo:
            seen = [ctx - (hi - lo) + i + 1 for i in range(hi - lo)]
            out[lo:hi], size[lo:hi] = attend(q[lo:hi], k_cache, v_cache, tables[b], seen, scale)
            rows[lo:hi] = True
    return out, size, rows


def decode(q, k_cache, v_cache, tables, context, scale):
    parts = [attend(q[b:b + 1], k_cache, v_cache, tables[b], [c], scale) for b, c in enumerate(context)]
    return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])


def assert_attention_close(got, ref, size, terms=2):
    """The output's rounding to BF16 is off by 2^-8 |ref| at most.  Everything before is
    FP32 but the probabilities: in one BF16 term each is off by up to 2^-8 of itself, so the
    sum by 2^-8 of sum p |v| (size); in two by 2^-14.  A score of 128 products is off by up
    to 128 * 2^-22 of the sum of their magnitudes (below 10 here, scaled), 2^-12, and sums
    over up to 2^12 tokens by 2^-12; 2^-10 of size covers those."""
    bound = 2.0 ** -8 * ref.abs() + (2.0 ** -10 + (2.0 ** -8 if terms == 1 else 0)) * size + 1e-30
    worst = ((got.double() - ref).abs() / bound).max().item() if ref.numel() else 0.0
    assert torch.isfinite(got).all() and worst <= 1.0, worst
