"""Measured cases of the 4-bit KV cache and token log-probability operators.

Each case names one operator and its sizes; ``run`` makes one pass, in plain
torch (``own`` false) or through the framework's entry points (``own`` true):

* ``attention``  decode attention over a paged cache held in 4 bits
                 (``nanovllm.kernels.kv4_cache.paged_decode_attention_kv4``);
* ``store``      q/k RMSNorm + rotary embedding of a fused QKV projection, K and V
                 quantised into that cache (``qk_norm_rope_store_kv4``);
* ``tables``     block tables, slot map, positions and context lengths of a step
                 (``nanovllm.kernels.step_tables.build_step_tables``);
* ``logprobs``   log-probability and rank of given tokens, entropy and the top
                 alternatives (``nanovllm.kernels.token_logprobs.token_logprobs``).

The 4-bit cache: codes uint8 [pages, kv_heads, 256, 64] and BF16 scales [pages,
kv_heads, 256, 4] for K and for V, one scale per 32 of the 128 channels.  A
group's scale is s = bf16(absmax / 7) (1 when all are zero); a value's code is
round-half-even(x / s) in [-7, 7], held as code + 8.  Four consecutive channels
of a token make a 16-bit unit (lowest channel in the lowest nibble).  With
g = channel // 32 and r = channel % 32, a K unit lies at byte
``(r // 8) * 16 + g * 4 + (r % 8) // 4 * 2`` of its token's 64 bytes; a V unit at
byte ``((r // 4) ^ (2 * (pair % 4))) * 16 + g * 4 + token % 2 * 2`` of the 128
bytes of its token pair (pair = token // 2).
"""
import math
import os
import random
import sys

import torch

own = False

D, PAGE, GROUP = 128, 256, 32
PACKAGE = os.path.join(os.getcwd(), "nano-vllm-int4_b200")


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one user, a short chat: the latency of a single token
        dict(name="attention-one-short", op="attention", batch=1, q_heads=32, kv_heads=8, max_len=700, spread="even"),
        # the framework's own decode benchmark: 32 prompts of 4096 tokens, 256 tokens further at most
        dict(name="attention-32x4k", op="attention", batch=32, q_heads=32, kv_heads=8, max_len=4352, spread="even"),
        # long documents beside short chats: ragged lengths up to 16k, some rows of the batch empty
        dict(name="attention-64-ragged-16k", op="attention", batch=64, q_heads=32, kv_heads=8, max_len=16384,
             spread="ragged"),
        # the decode step's tokens, some of them the padding of a captured batch
        dict(name="store-decode-32", op="store", tokens=32, q_heads=32, kv_heads=8, padding=0.1),
        # a prompt of odd length on another head layout (five query heads a KV head)
        dict(name="store-prompt-301", op="store", tokens=301, q_heads=40, kv_heads=8, padding=0.0),
        # a full prefill step (the default of max_num_batched_tokens)
        dict(name="store-prefill-16384", op="store", tokens=16384, q_heads=32, kv_heads=8, padding=0.0),
        # decode steps of 32 and of 512 requests (the default of max_num_seqs), one new token each
        dict(name="tables-decode-32", op="tables", batch=32, cached=4096, new=1, max_pages=17),
        dict(name="tables-decode-512", op="tables", batch=512, cached=4000, new=1, max_pages=16),
        # a prefill step: prompts of ragged lengths, nothing cached
        dict(name="tables-prefill-40", op="tables", batch=40, cached=0, new=400, max_pages=16),
        # the sampled token of one request with five alternatives
        dict(name="logprobs-one", op="logprobs", rows=1, vocab=151936, dtype="bfloat16", top_k=5, masked=0.0),
        # a batch of requests under a grammar mask, FP32 logits, twenty alternatives, odd vocabulary
        dict(name="logprobs-48-fp32", op="logprobs", rows=48, vocab=100003, dtype="float32", top_k=20, masked=0.3),
        # the prompt's own tokens scored, a slice of the prompt at a time
        dict(name="logprobs-prompt-1024", op="logprobs", rows=1024, vocab=151936, dtype="bfloat16", top_k=0, masked=0.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "store", "tables", "logprobs"])
    if op == "attention":
        kv = rng.choice([1, 2, 4, 8])
        batch = _log_int(rng, 1, 256)
        most = min(40960, 64 * 16384 * 8 // (batch * kv * 2))
        return dict(op=op, batch=batch, q_heads=kv * rng.choice([1, 2, 4, 5, 8]), kv_heads=kv,
                    max_len=_log_int(rng, 1, most), spread=rng.choice(["even", "ragged"]))
    if op == "store":
        kv = rng.choice([1, 2, 4, 8])
        return dict(op=op, tokens=_log_int(rng, 1, 16384), q_heads=kv * rng.choice([1, 2, 4, 5]), kv_heads=kv,
                    padding=rng.choice([0.0, 0.1]))
    if op == "tables":
        if rng.random() < 0.5:
            pages = _log_int(rng, 1, 64)
            return dict(op=op, batch=_log_int(rng, 1, 512), cached=pages * PAGE - rng.randint(1, PAGE - 1), new=1,
                        max_pages=pages)
        batch = _log_int(rng, 1, 128)
        new = _log_int(rng, 1, 16384 // batch)
        cached = rng.choice([0, _log_int(rng, 1, 8192)])
        return dict(op=op, batch=batch, cached=cached, new=new, max_pages=(cached + 2 * new) // PAGE + 1)
    dtype = rng.choice(["bfloat16", "float32"])
    rows = _log_int(rng, 1, 1024)
    vocab = _log_int(rng, 1000, 160000)
    if dtype == "float32":
        rows = min(rows, 256)
    if rows * vocab > 1024 * 151936:
        vocab = 1024 * 151936 // rows
    return dict(op=op, rows=rows, vocab=vocab, dtype=dtype, top_k=rng.choice([0, 1, 5, 20]),
                masked=rng.choice([0.0, 0.3]))


# ------------------------------------------------------------------ the cache's layout
def _k_position(token, channel):
    """Nibble index, within 8 tokens (1024 nibbles), of a K code."""
    g, r = channel // GROUP, channel % GROUP
    byte = token * 64 + (r // 8) * 16 + g * 4 + (r % 8) // 4 * 2
    return byte * 2 + r % 4


def _v_position(token, channel):
    g, r = channel // GROUP, channel % GROUP
    pair = token // 2
    byte = pair * 128 + ((r // 4) ^ (2 * (pair % 4))) * 16 + g * 4 + token % 2 * 2
    return byte * 2 + r % 4


def _positions(of, device):
    token = torch.arange(8, device=device)[:, None]
    channel = torch.arange(D, device=device)[None, :]
    return of(token, channel).reshape(-1)


def _quantise(x):
    """(code + 8, scale) of float32 values [..., 128]."""
    groups = x.double().unflatten(-1, (4, GROUP))
    top = groups.abs().amax(-1)
    scale = (top / 7.0).float().clamp_min(2.0 ** -126).bfloat16()
    scale = torch.where(top == 0, torch.ones_like(scale), scale)
    codes = torch.round(groups / scale.double().unsqueeze(-1)).clamp(-7, 7) + 8
    return codes.to(torch.uint8).flatten(-2), scale


def _pack(codes, positions):
    """uint8 codes [pages, heads, 256, 128] -> bytes [pages, heads, 256, 64]."""
    source = torch.empty_like(positions)
    source[positions] = torch.arange(positions.numel(), device=positions.device)
    nibbles = codes.reshape(*codes.shape[:2], 32, 1024).index_select(-1, source)
    return (nibbles[..., ::2] | (nibbles[..., 1::2] << 4)).reshape(*codes.shape[:3], 64)


def _unpack(packed, positions):
    """bytes [..., 256, 64] -> centred codes, float32 [..., 256, 128]."""
    flat = packed.reshape(*packed.shape[:-2], 32, 512)
    nibbles = torch.stack((flat & 15, flat >> 4), -1).flatten(-2)
    return nibbles.index_select(-1, positions).reshape(*packed.shape[:-1], D).float() - 8.0


# ------------------------------------------------------------------ inputs
def _lengths(case, rng):
    b, most = case["batch"], case["max_len"]
    if case["spread"] == "even":
        low = max(1, most - most // 16)
        lens = [rng.randint(low, most) for _ in range(b)]
    else:
        lens = [0 if rng.random() < 0.05 else _log_int(rng, max(1, most // 32), most) for _ in range(b)]
    lens[rng.randrange(b)] = most
    return lens


def _cache(pages, heads, g):
    """A cache filled with quantised K and V: K with a few strong channels, as after its norm weight."""
    out = []
    for of in (_k_position, _v_position):
        positions = _positions(of, "cuda")
        x = torch.randn(pages, heads, PAGE, D, device="cuda", generator=g)
        if of is _k_position:
            x *= 1 + 4 * (torch.rand(heads, 1, D, device="cuda", generator=g) > 0.95)
        codes, scale = _quantise(x.bfloat16().float())
        del x
        out.append((_pack(codes, positions), scale, positions))
    return out


def _prepare_attention(case, seed, g, rng):
    lens = _lengths(case, rng)
    max_pages = max(1, -(-max(lens) // PAGE))
    used = [-(-n // PAGE) for n in lens]
    total = max(1, sum(used))
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    tables, at = [], 0
    for n in used:
        tables.append(order[at:at + n] + [0] * (max_pages - n))
        at += n
    (kc, ks, kp), (vc, vs, vp) = _cache(total, case["kv_heads"], g)
    q = torch.randn(case["batch"], case["q_heads"], D, device="cuda", generator=g).bfloat16()
    return dict(q=q, k_codes=kc, k_scales=ks, v_codes=vc, v_scales=vs, k_positions=kp, v_positions=vp,
                tables=torch.tensor(tables, dtype=torch.int32, device="cuda"),
                lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), scale=D ** -0.5)


def _prepare_store(case, seed, g, rng):
    t, hq, hkv = case["tokens"], case["q_heads"], case["kv_heads"]
    pages = -(-t // PAGE) + 3
    qkv = torch.randn(t, hq + 2 * hkv, D, device="cuda", generator=g)
    qkv *= 0.5 + 2 * torch.rand(t, 1, 1, device="cuda", generator=g)
    qw, kw = (1 + 0.5 * torch.randn(2, D, device="cuda", generator=g)).bfloat16()
    length = 40960
    inverse = 1.0 / (1e6 ** (torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D))
    angle = torch.arange(length, dtype=torch.float64, device="cuda")[:, None] * inverse
    cos_sin = torch.cat((angle.cos(), angle.sin()), -1).float()
    slots = torch.randperm(pages * PAGE, device="cuda", generator=g)[:t].int()
    slots[torch.rand(t, device="cuda", generator=g) < case["padding"]] = -1
    state = dict(qkv=qkv.bfloat16().view(t, -1), q_weight=qw, k_weight=kw, cos_sin=cos_sin, slots=slots,
                 positions=torch.randint(0, length, (t,), device="cuda", generator=g), eps=1e-6, hq=hq, hkv=hkv,
                 stored=(slots >= 0).nonzero()[:, 0])
    for name in ("k", "v"):
        state[name + "_codes"] = torch.randint(0, 256, (pages, hkv, PAGE, 64), device="cuda", generator=g,
                                               dtype=torch.uint8)
        state[name + "_scales"] = torch.rand(pages, hkv, PAGE, 4, device="cuda", generator=g).bfloat16()
    return state


def _prepare_tables(case, seed, g, rng):
    b, cached, new = case["batch"], case["cached"], case["new"]
    limit = case["max_pages"] * PAGE
    cached = [rng.randint(cached // 2, cached) for _ in range(b)]
    news = [new] * b  # ragged in pairs, so that the step's tokens are as many for every seed
    for i in range(0, b - 1, 2):
        d = rng.randint(0, new // 2)
        news[i], news[i + 1] = new + d, new - d
    news = [max(1, n) for n in news]
    cached = [min(c, limit - n) for c, n in zip(cached, news)]
    need = sum(-(-(c + n) // PAGE) for c, n in zip(cached, news))
    pages = torch.randperm(need + 100, generator=torch.Generator().manual_seed(seed))[:need]
    return dict(cached=torch.tensor(cached, dtype=torch.int32, device="cuda"),
                new=torch.tensor(news, dtype=torch.int32, device="cuda"), pages=pages.int().cuda(),
                tokens=sum(news), max_pages=case["max_pages"])


def _prepare_logprobs(case, seed, g, rng):
    t, v = case["rows"], case["vocab"]
    dtype = getattr(torch, case["dtype"])
    x = torch.randn(t, v, device="cuda", generator=g) * (1 + 2 * torch.rand(t, 1, device="cuda", generator=g))
    likely = torch.randint(0, v, (t,), device="cuda", generator=g)
    x[torch.arange(t, device="cuda"), likely] += 12 * torch.rand(t, device="cuda", generator=g)
    any_token = torch.randint(0, v, (t,), device="cuda", generator=g)
    targets = torch.where(torch.rand(t, device="cuda", generator=g) < 0.7, likely, any_token)
    if case["masked"]:
        gone = torch.rand(t, v, device="cuda", generator=g) < case["masked"]
        gone[torch.arange(t, device="cuda"), targets] = False  # a given token is one that the grammar allows
        x.masked_fill_(gone, -math.inf)
        lowest = torch.rand(t, 1, device="cuda", generator=g) < 0.5  # half the rows: the type's lowest value instead
        x = torch.where(gone & lowest, torch.full_like(x, torch.finfo(dtype).min), x)
        del gone
    return dict(logits=x.to(dtype), targets=targets, top_k=case["top_k"])


_PREPARE = dict(attention=_prepare_attention, store=_prepare_store, tables=_prepare_tables, logprobs=_prepare_logprobs)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = _PREPARE[case["op"]](case, seed, g, random.Random(seed))
    state["op"] = case["op"]
    return state


# ------------------------------------------------------------------ plain forms
def _plain_attention(s):
    b, hq, _ = s["q"].shape
    hkv, width = s["k_codes"].shape[1], s["tables"].shape[1]
    pages = s["tables"].long()

    def values(codes, scales, positions):
        x = _unpack(codes[pages], positions).unflatten(-1, (4, GROUP))
        x *= scales[pages].float().unsqueeze(-1)
        return x.flatten(-2).transpose(1, 2).reshape(b, hkv, width * PAGE, D)

    q = s["q"].float().view(b, hkv, hq // hkv, D)
    scores = q @ values(s["k_codes"], s["k_scales"], s["k_positions"]).transpose(-1, -2) * s["scale"]
    gone = torch.arange(width * PAGE, device=q.device) >= s["lens"][:, None]
    scores = scores.masked_fill(gone[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-3e38)
    e = (scores - top).exp()
    out = e @ values(s["v_codes"], s["v_scales"], s["v_positions"])
    out = torch.where(s["lens"][:, None, None, None] > 0, out / e.sum(-1, keepdim=True), 0.0)
    return {"out": out.view(b, hq, D).bfloat16()}


def _norm_rope(x, w, s, dtype):
    x = x.to(dtype)
    x = x * (x.square().mean(-1, keepdim=True) + s["eps"]).rsqrt() * w.to(dtype)
    cos, sin = s["cos_sin"][s["positions"]].to(dtype).unsqueeze(1).chunk(2, -1)
    x1, x2 = x.chunk(2, -1)
    return torch.cat((x1 * cos - x2 * sin, x2 * cos + x1 * sin), -1)


def _plain_store(s):
    hq, hkv = s["hq"], s["hkv"]
    q, k, v = s["qkv"].view(-1, hq + 2 * hkv, D).split([hq, hkv, hkv], 1)
    q_out = _norm_rope(q, s["q_weight"], s, torch.float32).bfloat16()
    k_codes, k_scale = _quantise(_norm_rope(k, s["k_weight"], s, torch.float64).float())  # 64 bits: codes next to a border
    v_codes, v_scale = _quantise(v.float())
    rows = s["stored"]
    slot = s["slots"][rows].long()
    page, token = slot // PAGE, slot % PAGE
    heads = torch.arange(hkv, device=slot.device)
    base = (page[:, None] * hkv + heads) * (PAGE * 64)  # first byte of the (page, head) tile
    byte = torch.arange(64, device=slot.device)
    # K: units (8-channel run, group, half); V: units (4-channel run, group)
    units = k_codes[rows].view(-1, hkv, 4, 4, 2, 4).transpose(2, 3).flatten(2)
    at = base[..., None] + (token * 64)[:, None, None] + byte
    s["k_codes"].view(-1)[at] = units[..., ::2] | (units[..., 1::2] << 4)
    units = v_codes[rows].view(-1, hkv, 4, 8, 4).transpose(2, 3).flatten(2)
    pair = (token // 2)[:, None, None]
    at = (base[..., None] + pair * 128 + ((byte // 8) ^ (2 * (pair % 4))) * 16 + byte % 8 // 2 * 4
          + (token % 2)[:, None, None] * 2 + byte % 2)
    s["v_codes"].view(-1)[at] = units[..., ::2] | (units[..., 1::2] << 4)
    s["k_scales"][page, :, token] = k_scale[rows]
    s["v_scales"][page, :, token] = v_scale[rows]

    def values(codes, scale):
        return ((codes.float() - 8).unflatten(-1, (4, GROUP)) * scale.float().unsqueeze(-1)).flatten(-2).bfloat16()

    return {"q": q_out, "k_values": values(k_codes, k_scale), "v_values": values(v_codes, v_scale),
            "cache": [s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"]]}


def _plain_tables(s):
    cached, new, pages, width = s["cached"].long(), s["new"].long(), s["pages"], s["max_pages"]
    context = cached + new
    count = (context + PAGE - 1) // PAGE
    first = count.cumsum(0) - count
    column = torch.arange(width, device=cached.device)
    at = (first[:, None] + column).clamp_max(pages.numel() - 1)
    tables = torch.where(column < count[:, None], pages[at], 0)
    ends = new.cumsum(0)
    token = torch.arange(s["tokens"], device=cached.device)
    row = torch.searchsorted(ends, token, right=True)
    position = cached[row] + token - (ends - new)[row]
    slot = tables[row, position // PAGE] * PAGE + position % PAGE
    starts = torch.cat((torch.zeros_like(ends[:1]), ends))
    return {"block_tables": tables.int(), "context_lens": context.int(), "slot_mapping": slot.int(),
            "positions": position, "query_starts": starts.int()}


def _plain_logprobs(s):
    x, targets, k = s["logits"].float(), s["targets"], s["top_k"]
    top = x.amax(-1, keepdim=True)
    d = x - top
    e = d.exp()
    total = e.sum(-1, keepdim=True)
    log_total = total.log()
    d.masked_fill_(e == 0, 0.0)
    entropy = log_total[:, 0] - (e * d).sum(-1) / total[:, 0]
    del d, e
    chosen = x.gather(1, targets[:, None])
    out = {"logprobs": (chosen - top - log_total)[:, 0], "ranks": (x > chosen).sum(-1) + 1, "entropy": entropy}
    if k:
        bits = (x + 0.0).view(torch.int32)
        order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()
        lowest_first = 0xFFFFFFFF - torch.arange(x.shape[1], device=x.device)
        keys = ((order << 32) + lowest_first).topk(k, -1).values
        out["top_ids"] = 0xFFFFFFFF - (keys & 0xFFFFFFFF)
        out["top_logprobs"] = x.gather(1, out["top_ids"]) - top - log_total
    return out


_PLAIN = dict(attention=_plain_attention, store=_plain_store, tables=_plain_tables, logprobs=_plain_logprobs)


# ------------------------------------------------------------------ the framework's calls
def _own_attention(s):
    from nanovllm.kernels import kv4_cache
    cache = kv4_cache.Kv4Cache(s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"])
    return {"out": kv4_cache.paged_decode_attention_kv4(s["q"], cache, s["tables"], s["lens"], scale=s["scale"])}


def _own_store(s):
    from nanovllm.kernels import kv4_cache
    cache = kv4_cache.Kv4Cache(s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"])
    q, k, v = kv4_cache.qk_norm_rope_store_kv4(s["qkv"], s["q_weight"], s["k_weight"], s["cos_sin"], s["positions"],
                                               s["slots"], cache, num_heads=s["hq"], num_kv_heads=s["hkv"],
                                               eps=s["eps"], return_values=True)
    return {"q": q, "k_values": k, "v_values": v,
            "cache": [cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales]}


def _own_tables(s):
    from nanovllm.kernels import step_tables
    t = step_tables.build_step_tables(s["cached"], s["new"], s["pages"], num_tokens=s["tokens"],
                                      max_pages=s["max_pages"])
    return {"block_tables": t.block_tables, "context_lens": t.context_lens, "slot_mapping": t.slot_mapping,
            "positions": t.positions, "query_starts": t.query_starts}


def _own_logprobs(s):
    from nanovllm.kernels import token_logprobs
    r = token_logprobs.token_logprobs(s["logits"], s["targets"], top_k=s["top_k"])
    out = {"logprobs": r.logprobs, "ranks": r.ranks, "entropy": r.entropy}
    if s["top_k"]:
        out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
    return out


_OWN = dict(attention=_own_attention, store=_own_store, tables=_own_tables, logprobs=_own_logprobs)


def run(state):
    if own:
        if PACKAGE not in sys.path:  # the package's folder, as the tests and the benchmark put it there
            sys.path.insert(0, PACKAGE)
        return _OWN[state["op"]](state)
    return _PLAIN[state["op"]](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "attention":
        b, hq, hkv, most = case["batch"], case["q_heads"], case["kv_heads"], case["max_len"]
        # mean lengths of the two spreads: uniform over the top sixteenth; log-uniform from max_len / 32, 5% empty
        mean = most * 31 / 32 if case["spread"] == "even" else 0.95 * most * (1 - 1 / 32) / math.log(32)
        tokens = (b - 1) * mean + most
        row = 2 * (D // 2 + D // GROUP * 2)
        return {"bytes": tokens * hkv * row + b * (4 * D * hq + 4) + 4 * tokens / PAGE, "flops": 4 * tokens * hq * D}
    if op == "store":
        t, hq, hkv = case["tokens"], case["q_heads"], case["kv_heads"]
        stored = t * (1 - case["padding"]) * hkv * 2 * (D // 2 + D // GROUP * 2)
        # qkv, the position and its cos and sin, the slot in; q, the values and the stored rows out
        return {"bytes": t * ((hq + 2 * hkv) * 2 * D + 8 + 4 * D + 4) + t * (hq + 2 * hkv) * 2 * D + stored,
                "flops": t * (hq + hkv) * D * 8}
    if op == "tables":
        b, cached = case["batch"], case["cached"] * 3 / 4
        tokens = b * case["new"]
        pages = b * ((cached + case["new"]) / PAGE + 0.5)
        return {"bytes": 8 * b + 4 * pages + 4 * b * case["max_pages"] + 4 * b + 4 * (b + 1) + 12 * tokens, "flops": 0}
    t, v, k = case["rows"], case["vocab"], case["top_k"]
    return {"bytes": t * v * (2 if case["dtype"] == "bfloat16" else 4) + t * (8 + 16 + 12 * k), "flops": 5 * t * v}


# ------------------------------------------------------------------ the same in 64 bits
def _exact_attention(s):
    """Per sequence and from the byte formulas: every (token, channel) looked up by its own address."""
    b, hq, _ = s["q"].shape
    hkv = s["k_codes"].shape[1]
    c = torch.arange(D, device="cuda")
    t = torch.arange(PAGE, device="cuda")[:, None]
    run8, quad = c % 32 // 8, c % 32 // 4
    k_byte = 64 * t + 16 * run8 + 4 * (c // 32) + 2 * (c // 4 % 2) + c % 4 // 2
    v_byte = 128 * (t // 2) + 16 * (quad ^ (2 * (t // 2 % 4))) + 4 * (c // 32) + 2 * (t % 2) + c % 4 // 2
    shift = (4 * (c % 2)).to(torch.uint8)
    out = torch.zeros(b, hq, D, dtype=torch.float64, device="cuda")
    for i, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        page = s["tables"][i, :-(-n // PAGE)].long()

        def dense(codes, scales, byte):
            nibble = (codes[page].flatten(2)[:, :, byte] >> shift) & 15
            x = (nibble.double() - 8) * scales[page].double().repeat_interleave(32, -1)
            return x.transpose(0, 1).reshape(hkv, -1, D)[:, :n]

        q = s["q"][i].double().view(hkv, hq // hkv, D)
        p = torch.softmax(torch.einsum("hgd,htd->hgt", q, dense(s["k_codes"], s["k_scales"], k_byte)) * s["scale"], -1)
        out[i] = torch.einsum("hgt,htd->hgd", p, dense(s["v_codes"], s["v_scales"], v_byte)).reshape(hq, D)
    return {"out": out}


def _exact_store(s):
    hq, hkv = s["hq"], s["hkv"]
    x = s["qkv"].double().view(-1, hq + 2 * hkv, D)
    angle = s["cos_sin"][s["positions"]].double()
    turn = torch.complex(angle[:, :64], angle[:, 64:])[:, None]

    def rotated(h, w):
        h = h / (h.pow(2).sum(-1, keepdim=True) / D + s["eps"]).sqrt() * w.double()
        h = torch.complex(h[..., :64], h[..., 64:]) * turn
        return torch.cat((h.real, h.imag), -1)

    def held(h):
        h = h.float().double().view(*h.shape[:-1], 4, 32)
        most = h.abs().max(-1, keepdim=True).values
        step = torch.where(most > 0, (most / 7).float().bfloat16().double(), 1.0)
        return ((h / step).round() * step).view(*h.shape[:-2], D)

    return {"q": rotated(x[:, :hq], s["q_weight"]), "k_values": held(rotated(x[:, hq:hq + hkv], s["k_weight"])),
            "v_values": held(x[:, hq + hkv:]), "cache": [None, None, None, None]}


def _exact_logprobs(s):
    x = s["logits"].double()
    logp = x - torch.logsumexp(x, -1, keepdim=True)
    p = logp.exp()
    out = {"logprobs": logp.gather(1, s["targets"][:, None])[:, 0], "ranks": None,
           "entropy": -torch.where(p > 0, p * logp, 0.0).sum(-1)}
    if s["top_k"]:
        out["top_ids"], out["top_logprobs"] = None, logp.topk(s["top_k"], -1).values
    return out


def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers
    return dict(attention=_exact_attention, store=_exact_store, logprobs=_exact_logprobs)[case["op"]](
        prepare(case, seed))
