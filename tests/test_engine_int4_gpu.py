"""The engine with a 4-bit KV cache and with log-probabilities asked for, on a
small random-init Qwen3; and one step's operators in a row against 64 bits."""
import gc
import math

import pytest
import torch

import kv4_reference as ref
from nanovllm import _native
from nanovllm.kernels.kv4_cache import alloc_kv4_cache, paged_decode_attention_kv4, qk_norm_rope_store_kv4
from nanovllm.kernels.step_tables import build_step_tables
from nanovllm.kernels.token_logprobs import token_logprobs
from nanovllm.layers.common import rotary_cos_sin
from nanovllm.utils import synthetic

pytestmark = pytest.mark.gpu

TINY = dict(num_hidden_layers=2, hidden_size=1024, intermediate_size=2048, num_attention_heads=8,
            num_key_value_heads=2, vocab_size=4099, max_position_embeddings=4096)


@pytest.fixture(scope="module")
def model_dir(tmp_path_factory):
    return synthetic.write_qwen3_config(str(tmp_path_factory.mktemp("qwen3_kv4")), **TINY)


def prompts(lengths=(7, 100, 257, 600, 3), seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, TINY["vocab_size"], (k,), generator=g).tolist() for k in lengths]


def generate(model_dir, params=None, record=None, texts=None, **kw):
    from nanovllm import LLM, SamplingParams
    args = dict(load_format="dummy", max_model_len=1024, max_num_batched_tokens=2048, max_num_seqs=8,
                num_kvcache_blocks=48, seed=3)
    args.update(kw)
    llm = LLM(model_dir, **args)
    try:
        if record is not None:
            model = llm.runner.model
            inner = model.compute_logits

            def compute_logits(hidden):
                logits = inner(hidden)
                record.append(logits.clone())
                return logits
            model.compute_logits = compute_logits
        base = dict(temperature=0.0, max_tokens=24, ignore_eos=True)
        out = llm.generate(texts or prompts(), SamplingParams(**(base | (params or {}))))
        blocks = llm.runner.config.num_kvcache_blocks
        assert _native.device_error() == 0
        return out, blocks
    finally:
        llm.exit()
        del llm
        gc.collect()
        torch.cuda.empty_cache()


@pytest.mark.parametrize("flavour", [dict(w4a4_checkpoint="random"), dict(), dict(use_w4a16=True)],
                         ids=["w4a4", "bf16", "w4a16"])
def test_graph_decode_matches_eager(cuda_device, model_dir, flavour):
    graph, _ = generate(model_dir, kv_cache_dtype="int4", **flavour)
    eager, _ = generate(model_dir, kv_cache_dtype="int4", enforce_eager=True, **flavour)
    assert [o["token_ids"] for o in graph] == [o["token_ids"] for o in eager]
    assert all(len(o["token_ids"]) == 24 for o in graph)
    assert all("logprobs" not in o and "prompt_logprobs" not in o for o in graph)


def test_more_pages_and_preemption(cuda_device, model_dir):
    """A pool that the memory alone limits holds about 512 / 144 times the pages;
    one that is too small preempts, and every request still ends."""
    _, small = generate(model_dir, num_kvcache_blocks=-1, gpu_memory_utilization=0.1, params=dict(max_tokens=1))
    _, large = generate(model_dir, num_kvcache_blocks=-1, gpu_memory_utilization=0.1, params=dict(max_tokens=1),
                        kv_cache_dtype="int4")
    assert 3.3 * small < large < 3.8 * small
    out, _ = generate(model_dir, kv_cache_dtype="int4", num_kvcache_blocks=5, texts=prompts((250, 250, 250, 250)))
    assert all(len(o["token_ids"]) == 24 for o in out)


def row_reference(row, token, k):
    x = row.double().cpu()
    logp = (x - x.max()) - (x - x.max()).exp().sum().log()
    order = torch.sort(x, descending=True, stable=True).indices[:k].tolist()
    return (logp[token].item(), int((x > x[token]).sum()) + 1, -(logp.exp() * logp).sum().item(),
            [(i, logp[i].item()) for i in order])


def assert_described(found, row, token, k):
    lp, rank, entropy, top = row_reference(row, token, k)
    assert found["token_id"] == token and found["rank"] == rank
    # FP32 sums of 4099 exponentials of logits within some tens: see the operator's own tests
    assert math.isclose(found["logprob"], lp, rel_tol=2e-6, abs_tol=4e-6)
    assert math.isclose(found["entropy"], entropy, rel_tol=4e-6, abs_tol=4e-6)
    assert [i for i, _ in found["top"]] == [i for i, _ in top]
    assert all(math.isclose(a, b, rel_tol=2e-6, abs_tol=4e-6) for (_, a), (_, b) in zip(found["top"], top))


@pytest.mark.parametrize("cache", ["bf16", "int4"])
def test_logprobs_of_generated_and_prompt_tokens(cuda_device, model_dir, cache, monkeypatch):
    import nanovllm.engine.runner as runner
    monkeypatch.setattr(runner, "LOGPROB_ROWS", 256)  # the 600-token prompt goes in three parts
    texts, record = prompts((7, 600, 1)), []
    plain, _ = generate(model_dir, kv_cache_dtype=cache, texts=texts)
    out, _ = generate(model_dir, kv_cache_dtype=cache, texts=texts, record=record,
                      params=dict(logprobs=3, prompt_logprobs=2, max_tokens=10))
    assert [o["token_ids"] for o in out] == [o["token_ids"][:10] for o in plain]
    # the prompts' positions come first, in order, then one set of logits a step
    at = 0
    for o, text in zip(out, texts):
        rows = []
        while len(rows) < len(text) - 1:
            rows += list(record[at])
            at += 1
        assert len(o["prompt_logprobs"]) == len(rows) == len(text) - 1
        for found, row, token in list(zip(o["prompt_logprobs"], rows, text[1:]))[::37]:
            assert_described(found, row, token, 2)
    steps = record[at:]
    assert len(steps) == 10
    for i, o in enumerate(out):
        assert len(o["logprobs"]) == 10
        for found, logits, token in zip(o["logprobs"], steps, o["token_ids"]):
            assert found["rank"] == 1
            assert_described(found, logits[i], token, 3)


def test_each_request_its_own_logprobs(cuda_device, model_dir):
    from nanovllm import LLM, SamplingParams
    llm = LLM(model_dir, load_format="dummy", max_model_len=512, max_num_batched_tokens=1024, max_num_seqs=4,
              num_kvcache_blocks=16, seed=3, kv_cache_dtype="int4")
    try:
        params = [SamplingParams(temperature=0.0, max_tokens=3 + i, ignore_eos=True, logprobs=k)
                  for i, k in enumerate((None, 0, 5))]
        out = llm.generate(prompts((5, 6, 7)), params)
    finally:
        llm.exit()
    assert "logprobs" not in out[0]
    assert [len(d["top"]) for d in out[1]["logprobs"]] == [0] * 4
    assert [len(d["top"]) for d in out[2]["logprobs"]] == [5] * 5
    assert all(d["top"][0][0] == d["token_id"] for d in out[2]["logprobs"])


def test_a_step_of_operators_against_64_bits(cuda_device):
    """Tables from lengths, prompts stored, a decode step's token stored and attended, its logits scored."""
    hq, hkv, d, vocab, eps, scale = 8, 2, 128, 500, 1e-6, 128 ** -0.5
    lens, pages_all = [300, 1, 257, 40], 12
    g = torch.Generator().manual_seed(1)
    dev = lambda x, dtype=torch.int32: torch.tensor(x, dtype=dtype, device=cuda_device)  # noqa: E731
    cache = alloc_kv4_cache(pages_all, hkv, cuda_device)
    for x in cache:
        x.zero_()
    w = (1 + 0.2 * torch.randn(2, d, generator=g)).bfloat16()
    cos_sin = rotary_cos_sin(d, 1024, 1e6)
    order = torch.randperm(pages_all, generator=g).tolist()
    history = []
    for cached, new in (([0] * 4, lens), (lens, [1] * 4)):
        need = sum(-(-(c + n) // 256) for c, n in zip(cached, new))
        # the pages of a request keep their order over the steps: the longest need comes first
        flat, at = [], 0
        for total in (n + 1 for n in lens):
            own = order[at:at + -(-total // 256)]
            at += len(own)
            flat.append(own)
        listed = [p for own, c, n in zip(flat, cached, new) for p in own[:-(-(c + n) // 256)]]
        assert len(listed) == need
        t = build_step_tables(dev(cached), dev(new), dev(listed), num_tokens=sum(new), max_pages=4)
        qkv = torch.randn(sum(new), (hq + 2 * hkv) * d, generator=g).bfloat16()
        q = qk_norm_rope_store_kv4(qkv.to(cuda_device), w[0].to(cuda_device), w[1].to(cuda_device), cos_sin.to(cuda_device),
                                   t.positions, t.slot_mapping, cache, num_heads=hq, num_kv_heads=hkv, eps=eps)
        history.append((qkv.view(-1, hq + 2 * hkv, d), cached, new))
    out = paged_decode_attention_kv4(q, cache, t.block_tables, t.context_lens, scale=scale)
    head = torch.randn(vocab, hq * d, generator=g) / 32
    logits = out.view(4, -1).float() @ head.T.to(cuda_device)
    targets = torch.randint(0, vocab, (4,), generator=g)
    got = token_logprobs(logits, targets.to(cuda_device), top_k=3)

    # the same from the inputs alone, in 64 bits
    for i in range(4):
        ks, vs = [], []
        for qkv, cached, new in history:
            at = sum(new[:i])
            part = qkv[at:at + new[i]]
            pos = torch.arange(cached[i], cached[i] + new[i])
            kc, kscale = ref.quantise(ref.norm_rope(part[:, hq:hq + hkv], w[1], cos_sin, pos, eps).float())
            vc, vscale = ref.quantise(part[:, hq + hkv:].float())
            ks.append(kc * kscale.repeat_interleave(32, -1))
            vs.append(vc * vscale.repeat_interleave(32, -1))
            qq = ref.norm_rope(part[-1:, :hq], w[0], cos_sin, pos[-1:], eps)[0]
        k, v = torch.cat(ks).transpose(0, 1), torch.cat(vs).transpose(0, 1)
        s = torch.einsum("hgd,htd->hgt", qq.view(hkv, -1, d), k) * scale
        p = torch.softmax(s, -1)
        o = torch.einsum("hgt,htd->hgd", p, v).reshape(-1)
        size = torch.einsum("hgt,htd->hgd", p, v.abs()).reshape(-1)
        # q's rounding to BF16 moves a score by 2^-8 sum |q k| scale at most, a probability by twice that
        moved = 2 * 2.0 ** -8 * (torch.einsum("hgd,htd->hgt", qq.abs().view(hkv, -1, d), k.abs()) * scale).amax().item()
        bound = 2.0 ** -8 * o.abs() + (2.0 ** -8 + 2.0 ** -10 + moved) * size
        assert ((out[i].double().cpu().reshape(-1) - o).abs() <= bound).all()
        x = head.double() @ o
        off = (head.double().abs() @ bound).max().item()  # of a logit
        logp = torch.log_softmax(x, -1)
        assert abs(got.logprobs[i].item() - logp[targets[i]].item()) <= 2 * off + 1e-5
        assert abs(got.top_logprobs[i, 0].item() - logp.max().item()) <= 2 * off + 1e-5
    assert _native.device_error() == 0


@pytest.mark.parametrize("cache", ["int4", "bf16"])
def test_tokens_up_to_the_end_of_the_last_page(cuda_device, model_dir, cache):
    """max_model_len within a page: requests may grow to the page's end, as with the next multiple of 256."""
    texts = prompts((990, 1))
    short, _ = generate(model_dir, kv_cache_dtype=cache, max_model_len=1000, texts=texts)
    whole, _ = generate(model_dir, kv_cache_dtype=cache, max_model_len=1024, texts=texts)
    assert [o["token_ids"] for o in short] == [o["token_ids"] for o in whole]


def test_preemption_happens_and_keeps_what_was_generated(cuda_device, model_dir, monkeypatch):
    from nanovllm.engine.scheduler import Scheduler
    preempted, inner = [], Scheduler._preempt

    def preempt(self, seq):
        preempted.append(seq.num_completion_tokens)
        inner(self, seq)
    monkeypatch.setattr(Scheduler, "_preempt", preempt)
    texts, params = prompts((250, 250, 250, 250)), dict(logprobs=1)
    plain, _ = generate(model_dir, kv_cache_dtype="int4", texts=texts, params=params)
    assert not preempted
    out, _ = generate(model_dir, kv_cache_dtype="int4", num_kvcache_blocks=5, texts=texts, params=params)
    # the 257th token needs a second page for each of the four, and one page is free: the last is preempted for the
    # second's, the third for want of one
    assert preempted == [7, 7]
    for o, p in zip(out, plain):
        assert len(o["logprobs"]) == len(o["token_ids"]) == 24
        assert [d["token_id"] for d in o["logprobs"]] == o["token_ids"]
        assert o["token_ids"][:7] == p["token_ids"][:7] and o["logprobs"][:7] == p["logprobs"][:7]
