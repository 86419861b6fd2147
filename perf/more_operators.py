"""Measured cases of the operators for requests that share cached tokens.

Each case names one operator and its sizes; ``run`` makes one pass, in plain
torch (``own`` false) or through the framework's entry points (``own`` true), all
of them in ``nanovllm.kernels.paged_attention``:

* ``append``   keys and values appended to the paged BF16 cache, the rotation (and,
               where the model has it, the q/k RMSNorm) applied on the way
               (``append_kv``);
* ``prefill``  new tokens of several requests, each over the tokens that its
               request already has in the cache (``paged_prefill_attention``);
* ``shared``   one query token per request, requests in groups that share the pages
               of a long prefix (``shared_prefix_attention``).

The cache: BF16 [pages, 256, kv_heads, 128] for K and for V, token t of a request
in page ``block_tables[request, t // 256]`` at row ``t % 256``.
"""
import math
import os
import random
import sys

import torch

own = False

D, PAGE = 128, 256
PACKAGE = os.path.join(os.getcwd(), "nano-vllm-int4_b200")


# ------------------------------------------------------------------ cases
def listed():
    return [
        # the decode step of the benchmark's 32 requests: views of the fused projection, q/k norm
        dict(name="append-decode-32", op="append", tokens=32, q_heads=32, kv_heads=8, rotary=128, norm=True,
             fused=True, padding=0.1),
        # a prompt of odd length, separate projections without norm, half of the channels rotated
        dict(name="append-prompt-301", op="append", tokens=301, q_heads=40, kv_heads=8, rotary=64, norm=False,
             fused=False, padding=0.0),
        # a full prefill step (the default of max_num_batched_tokens), separate projections as the GPTQ model's
        dict(name="append-prefill-16384", op="append", tokens=16384, q_heads=32, kv_heads=8, rotary=128, norm=True,
             fused=False, padding=0.0),
        # the next turn of a chat: a short message over a cached conversation
        dict(name="prefill-turn-37-over-3k", op="prefill", batch=1, new=37, cached=3100, ragged=False, q_heads=32,
             kv_heads=8, lens_seed=1),
        # ragged prompts behind a cached instruction, five query heads a KV head
        dict(name="prefill-8-ragged", op="prefill", batch=8, new=700, cached=1500, ragged=True, q_heads=40, kv_heads=8,
             lens_seed=2),
        # one prompt's slice over what is cached of a long document
        dict(name="prefill-2048-over-14k", op="prefill", batch=1, new=2048, cached=14336, ragged=False, q_heads=32,
             kv_heads=8, lens_seed=3),
        # a full prefill step: prompts of the benchmark's length, nothing cached
        dict(name="prefill-4x4096", op="prefill", batch=4, new=4096, cached=0, ragged=False, q_heads=32, kv_heads=8,
             lens_seed=4),
        # four samples of one question, just begun
        dict(name="shared-4-over-900", op="shared", groups=1, rows=4, prefix=900, own=40, q_heads=32, kv_heads=8,
             padding=0, lens_seed=5),
        # 32 answers to one prompt of the benchmark's length, up to its 256 tokens long
        dict(name="shared-32-over-4k", op="shared", groups=1, rows=32, prefix=4096, own=256, q_heads=32, kv_heads=8,
             padding=0, lens_seed=6),
        # several long documents with several questions each, and the padding of a captured batch
        dict(name="shared-12x8-ragged-16k", op="shared", groups=12, rows=8, prefix=16384, own=900, q_heads=32,
             kv_heads=8, padding=3, lens_seed=7),
        # one long instruction before every request of a large batch
        dict(name="shared-256-over-2k", op="shared", groups=1, rows=256, prefix=2000, own=700, q_heads=32, kv_heads=8,
             padding=0, lens_seed=8),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "prefill", "shared"])
    kv = rng.choice([1, 2, 4, 8])
    heads = dict(q_heads=kv * rng.choice([1, 2, 4, 5, 8]), kv_heads=kv)
    if op == "append":
        most = min(16384, 16384 * 48 // (heads["q_heads"] + 2 * kv))
        return dict(op=op, tokens=_log_int(rng, 1, most), **heads, rotary=rng.choice([128, 128, 64, 32]),
                    norm=rng.choice([True, False]), fused=rng.choice([True, False]), padding=rng.choice([0.0, 0.1]))
    if op == "prefill":
        batch = _log_int(rng, 1, 64)
        new = _log_int(rng, 1, max(1, 8192 // batch))
        cached = rng.choice([0, _log_int(rng, 1, max(1, min(16384, 65536 // batch)))])
        while batch * new * (new + cached) * heads["q_heads"] > 4096 * 4096 * 2 * 32:
            new, cached = max(1, new * 3 // 4), cached * 3 // 4
        return dict(op=op, batch=batch, new=new, cached=cached, ragged=rng.random() < 0.8, **heads,
                    lens_seed=rng.randrange(1 << 30))
    groups = _log_int(rng, 1, 16)
    prefix = _log_int(rng, 1, 16384)
    rows = _log_int(rng, 1, max(1, min(256, 10 * 16384 * 8 * 32 // (groups * (prefix + 500) * heads["q_heads"]),
                                    256 // groups)))
    return dict(op=op, groups=groups, rows=rows, prefix=prefix,
                own=_log_int(rng, 1, max(1, min(1024, 65536 // (groups * rows)))), **heads,
                padding=rng.choice([0, 0, 3]), lens_seed=rng.randrange(1 << 30))


def _lengths(case):
    """Lengths of the requests: of a prefill (cached, new) pairs, of a shared batch
    (prefix, [own tokens of each row]) per group; the same whatever the inputs' seed."""
    rng = random.Random(case["lens_seed"])
    if case["op"] == "prefill":
        b, new, cached = case["batch"], case["new"], case["cached"]
        if not case["ragged"]:
            return [(cached, new)] * b
        return [(rng.randint(cached // 2, cached), rng.randint((new + 1) // 2, new)) for _ in range(b)]
    many = case["groups"] > 1
    groups = []
    for _ in range(case["groups"]):
        rows = rng.randint((case["rows"] + 1) // 2, case["rows"]) if many else case["rows"]
        prefix = rng.randint((case["prefix"] + 3) // 4, case["prefix"]) if many else case["prefix"]
        groups.append((prefix, [rng.randint(1, case["own"]) for _ in range(rows)]))
    return groups


# ------------------------------------------------------------------ inputs
def _cache(pages, heads, g):
    """K with a few strong channels, as after its norm weight, and V."""
    k = torch.randn(pages, PAGE, heads, D, device="cuda", generator=g, dtype=torch.bfloat16)
    k *= 1 + 4 * (torch.rand(heads, D, device="cuda", generator=g) > 0.95).bfloat16()
    return k, torch.randn(pages, PAGE, heads, D, device="cuda", generator=g, dtype=torch.bfloat16)


def _prepare_append(case, seed, g):
    t, hq, hkv, r = case["tokens"], case["q_heads"], case["kv_heads"], case["rotary"]
    heads = hq + 2 * hkv
    x = torch.randn(t, heads, D, device="cuda", generator=g)
    x *= 0.5 + 2 * torch.rand(t, 1, 1, device="cuda", generator=g)
    parts = x.bfloat16().split([hq, hkv, hkv], 1)
    q, k, v = parts if case["fused"] else (p.contiguous() for p in parts)
    length = 40960
    inverse = 1.0 / (1e6 ** (torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r))
    angle = torch.arange(length, dtype=torch.float64, device="cuda")[:, None] * inverse
    pages = -(-t // PAGE) + 3
    slots = torch.randperm(pages * PAGE, device="cuda", generator=g)[:t].int()
    slots[torch.rand(t, device="cuda", generator=g) < case["padding"]] = -1
    k_cache, v_cache = _cache(pages, hkv, g)
    qw, kw = (1 + 0.5 * torch.randn(2, D, device="cuda", generator=g)).bfloat16()
    return dict(q=q, k=k, v=v, q_weight=qw if case["norm"] else None, k_weight=kw if case["norm"] else None, eps=1e-6,
                cos_sin=torch.cat((angle.cos(), angle.sin()), -1).float(), slots=slots,
                stored=(slots >= 0).nonzero()[:, 0], k_cache=k_cache, v_cache=v_cache,
                positions=torch.randint(0, length, (t,), device="cuda", generator=g))


def _tables(counts, seed):
    """Block tables of requests with that many pages each (a list: shared leading pages, then own)."""
    total = sum(counts)
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    out, at = [], 0
    for n in counts:
        out.append(order[at:at + n])
        at += n
    return out, total


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _prepare_prefill(case, seed, g):
    lens = _lengths(case)
    pages, total = _tables([-(-(c + n) // PAGE) for c, n in lens], seed)
    width = max(len(p) for p in pages)
    starts = [0]
    for _, n in lens:
        starts.append(starts[-1] + n)
    k_cache, v_cache = _cache(total, case["kv_heads"], g)
    return dict(q=torch.randn(starts[-1], case["q_heads"], D, device="cuda", generator=g).bfloat16(), lens=lens,
                k_cache=k_cache, v_cache=v_cache, tables=_int32([p + [0] * (width - len(p)) for p in pages]),
                context=_int32([c + n for c, n in lens]), starts=_int32(starts), scale=D ** -0.5)


def _prepare_shared(case, seed, g):
    groups = _lengths(case)
    counts = []
    for prefix, own_lens in groups:  # whole pages are shared; the rest of the prefix is in the row's own pages
        common = prefix // PAGE
        counts += [common] + [-(-(prefix + n) // PAGE) - common for n in own_lens]
    pages, total = _tables(counts, seed)
    tables, context, starts, at = [], [], [0], 0
    for prefix, own_lens in groups:
        common, at = pages[at], at + 1
        for n in own_lens:
            tables.append(common + pages[at])
            context.append(prefix + n)
            at += 1
        starts.append(len(tables))
    tables += [[]] * case["padding"]
    context += [0] * case["padding"]
    width = max(len(p) for p in tables)
    k_cache, v_cache = _cache(total, case["kv_heads"], g)
    return dict(q=torch.randn(len(tables), case["q_heads"], D, device="cuda", generator=g).bfloat16(),
                lens=context, rows=starts, prefix=[p for p, _ in groups], k_cache=k_cache, v_cache=v_cache,
                tables=_int32([p + [0] * (width - len(p)) for p in tables]), context=_int32(context),
                starts=_int32(starts), prefix_lens=_int32([p for p, _ in groups]), scale=D ** -0.5)


_PREPARE = dict(append=_prepare_append, prefill=_prepare_prefill, shared=_prepare_shared)


def prepare(case, seed):
    state = _PREPARE[case["op"]](case, seed, torch.Generator(device="cuda").manual_seed(seed))
    state["op"] = case["op"]
    return state


# ------------------------------------------------------------------ plain forms
def _turned(x, weight, s):
    x = x.float()
    if weight is not None:
        x = x * (x.square().mean(-1, keepdim=True) + s["eps"]).rsqrt() * weight.float()
    cos, sin = s["cos_sin"][s["positions"]].unsqueeze(1).chunk(2, -1)
    half = cos.shape[-1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, rest), -1).bfloat16()


def _plain_append(s):
    rows = s["stored"]
    slot = s["slots"][rows].long()
    s["k_cache"].flatten(0, 1)[slot] = _turned(s["k"], s["k_weight"], s)[rows]
    s["v_cache"].flatten(0, 1)[slot] = s["v"][rows]
    return {"q": _turned(s["q"], s["q_weight"], s), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _context(cache, pages, start, end):
    """FP32 [kv_heads, end - start, D] of the tokens start..end-1 (start on a page) of a request."""
    x = cache[pages[start // PAGE:-(-end // PAGE)].long()].flatten(0, 1)[:end - start]
    return x.transpose(0, 1).float()


def _plain_prefill(s):
    hq, hkv = s["q"].shape[1], s["k_cache"].shape[2]
    out, at = torch.empty_like(s["q"]), 0
    for i, (cached, new) in enumerate(s["lens"]):
        k, v = (_context(s[c], s["tables"][i], 0, cached + new) for c in ("k_cache", "v_cache"))
        for lo in range(0, new, 1024):
            hi = min(lo + 1024, new)
            seen = cached + hi
            q = s["q"][at + lo:at + hi].float().view(hi - lo, hkv, hq // hkv, D).permute(1, 2, 0, 3)
            scores = q.flatten(1, 2) @ k[:, :seen].transpose(1, 2) * s["scale"]
            scores = scores.view(hkv, hq // hkv, hi - lo, seen)
            behind = torch.arange(seen, device=q.device) > torch.arange(cached + lo, seen, device=q.device)[:, None]
            scores.masked_fill_(behind, -math.inf)
            e = (scores - scores.amax(-1, keepdim=True)).exp()
            o = (e.flatten(1, 2) @ v[:, :seen]).view(hkv, hq // hkv, hi - lo, D) / e.sum(-1, keepdim=True)
            out[at + lo:at + hi] = o.permute(2, 0, 1, 3).reshape(hi - lo, hq, D).bfloat16()
        at += new
    return {"out": out}


def _plain_shared(s):
    hq, hkv = s["q"].shape[1], s["k_cache"].shape[2]
    out = torch.zeros_like(s["q"])
    for g, prefix in enumerate(s["prefix"]):
        lo, hi = s["rows"][g], s["rows"][g + 1]
        n, common = hi - lo, prefix // PAGE * PAGE
        q = s["q"][lo:hi].float().view(n, hkv, hq // hkv, D)
        longest = max(s["lens"][lo:hi])
        pages = s["tables"][lo:hi, common // PAGE:-(-longest // PAGE)].long()
        k, v = (s[c][pages].flatten(1, 2).transpose(1, 2).float() for c in ("k_cache", "v_cache"))  # [n, hkv, t, D]
        scores = q @ k.transpose(2, 3) * s["scale"]
        t = torch.arange(common, common + k.shape[2], device=q.device)
        scores.masked_fill_((t >= s["context"][lo:hi, None])[:, None, None], -math.inf)
        top = scores.amax(-1, keepdim=True)
        if common:
            pk, pv = (_context(s[c], s["tables"][lo], 0, common) for c in ("k_cache", "v_cache"))
            of_prefix = (q.transpose(0, 1).reshape(hkv, -1, D) @ pk.transpose(1, 2) * s["scale"])
            of_prefix = of_prefix.view(hkv, n, hq // hkv, common).transpose(0, 1)
            top = torch.maximum(top, of_prefix.amax(-1, keepdim=True))
            e = (of_prefix - top).exp()
            total = e.sum(-1, keepdim=True)
            o = (e.transpose(0, 1).reshape(hkv, -1, common) @ pv).view(hkv, n, hq // hkv, D).transpose(0, 1)
        else:
            total, o = 0.0, 0.0
        e = (scores - top).exp()
        out[lo:hi] = ((o + e @ v) / (total + e.sum(-1, keepdim=True))).reshape(n, hq, D).bfloat16()
    return {"out": out}


_PLAIN = dict(append=_plain_append, prefill=_plain_prefill, shared=_plain_shared)


# ------------------------------------------------------------------ the framework's calls
def _own_append(s):
    from nanovllm.kernels import paged_attention
    q = paged_attention.append_kv(s["q"], s["k"], s["v"], s["cos_sin"], s["positions"], s["slots"], s["k_cache"],
                                  s["v_cache"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=s["eps"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_prefill(s):
    from nanovllm.kernels import paged_attention
    return {"out": paged_attention.paged_prefill_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"],
                                                           s["context"], s["starts"], scale=s["scale"])}


def _own_shared(s):
    from nanovllm.kernels import paged_attention
    return {"out": paged_attention.shared_prefix_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"],
                                                           s["context"], s["starts"], s["prefix_lens"],
                                                           scale=s["scale"])}


_OWN = dict(append=_own_append, prefill=_own_prefill, shared=_own_shared)


def run(state):
    if own:
        if PACKAGE not in sys.path:  # the package's folder, as the tests and the benchmark put it there
            sys.path.insert(0, PACKAGE)
        return _OWN[state["op"]](state)
    return _PLAIN[state["op"]](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    hq, hkv = case["q_heads"], case["kv_heads"]
    if case["op"] == "append":
        t = case["tokens"]
        stored = t * (1 - case["padding"])
        # q, k, v, the position, its cos and sin, the slot in; q and the stored rows out
        return {"bytes": t * ((hq + 2 * hkv) * 2 * D + 8 + 4 * case["rotary"] + 4) + t * hq * 2 * D
                + stored * hkv * 4 * D, "flops": t * (hq + hkv) * D * (8 if case["norm"] else 3)}
    lens = _lengths(case)
    if case["op"] == "prefill":
        tokens, queries = sum(c + n for c, n in lens), sum(n for _, n in lens)
        pairs = sum(n * c + n * (n + 1) // 2 for c, n in lens)
    else:
        queries = sum(len(o) for _, o in lens) + case["padding"]
        tokens = sum(p // PAGE * PAGE + sum(p % PAGE + n for n in o) for p, o in lens)
        pairs = sum(p + n for p, o in lens for n in o)
    return {"bytes": tokens * hkv * 4 * D + queries * hq * 4 * D, "flops": 4 * pairs * hq * D}


# ------------------------------------------------------------------ the same in 64 bits
def _exact_append(s):
    t = s["positions"].numel()
    angle = s["cos_sin"][s["positions"]].double()
    half = angle.shape[1] // 2
    turn = torch.complex(angle[:, :half], angle[:, half:])[:, None]

    def rotated(x, w):
        x = x.double()
        if w is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / D + s["eps"]).sqrt() * w.double()
        z = torch.complex(x[..., :half], x[..., half:2 * half]) * turn
        return torch.cat((z.real, z.imag, x[..., 2 * half:]), -1)

    out = {"q": rotated(s["q"], s["q_weight"])}
    k, v = rotated(s["k"], s["k_weight"]), s["v"].double()
    for name, x in (("k_cache", k), ("v_cache", v)):
        cache = s[name].double()
        pages, rows = s["slots"].long() // PAGE, s["slots"].long() % PAGE
        keep = torch.arange(t, device="cuda")[s["slots"] >= 0]
        cache[pages[keep], rows[keep]] = x[keep]
        out[name] = cache
    return out


def _attend(q, s, row, seen):
    """softmax(scale q K^T) V in 64 bits of queries q [n, Hq, D] of a request, query i over its first seen[i] tokens."""
    hkv = s["k_cache"].shape[2]
    n, hq, _ = q.shape
    most = int(seen.max())
    page = s["tables"][row, torch.arange(most, device="cuda") // PAGE].long()
    offset = torch.arange(most, device="cuda") % PAGE
    gone = torch.arange(most, device="cuda")[None] >= seen[:, None]
    out = torch.empty(n, hq, D, dtype=torch.float64, device="cuda")
    for h in range(hkv):
        of = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
        k, v = (s[c][page, offset, h].double() for c in ("k_cache", "v_cache"))
        scores = torch.einsum("ngd,td->gnt", q[:, of].double(), k) * s["scale"]
        p = torch.softmax(scores.masked_fill_(gone, -math.inf), -1)
        out[:, of] = torch.einsum("gnt,td->ngd", p, v)
    return out


def _exact_prefill(s):
    at, parts = 0, []
    for i, (cached, new) in enumerate(s["lens"]):
        for lo in range(0, new, 512):
            hi = min(lo + 512, new)
            seen = torch.arange(cached + lo + 1, cached + hi + 1, device="cuda")
            parts.append(_attend(s["q"][at + lo:at + hi], s, i, seen))
        at += new
    return {"out": torch.cat(parts)}


def _exact_shared(s):
    return {"out": torch.cat([_attend(s["q"][i:i + 1], s, i, torch.tensor([n], device="cuda")) if n
                              else torch.zeros(1, s["q"].shape[1], D, dtype=torch.float64, device="cuda")
                              for i, n in enumerate(s["lens"])])}


def exact(case, seed):
    return dict(append=_exact_append, prefill=_exact_prefill, shared=_exact_shared)[case["op"]](prepare(case, seed))
