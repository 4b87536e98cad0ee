"""A multi-adapter decoder on its paged cache: prompts, steps and logit rules
together give what forwards over the whole sequences give without a cache."""


import pytest
import torch

from polylora_b200 import PolyLoraConfig, PolyLoraModel
from polylora_b200.graphed import GraphedForward
from polylora_b200.kv_cache import PagedKVCache
from polylora_b200.logits import LogitRules
from polylora_b200.store import CpuLayerWeights

pytestmark = pytest.mark.gpu

TARGETS = ["q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "down_proj"]
VOCAB = 300


def _model(dev, dtype, heads=4, kv_heads=2, head_dim=32, layers=2, window=None):
    from transformers import LlamaConfig, LlamaForCausalLM, MistralConfig, MistralForCausalLM

    kw = dict(vocab_size=VOCAB, hidden_size=heads * head_dim, intermediate_size=256, num_hidden_layers=layers,
              num_attention_heads=heads, num_key_value_heads=kv_heads, max_position_embeddings=512)
    torch.manual_seed(0)
    torch.set_default_dtype(dtype)
    try:
        with torch.device(dev):
            base = (MistralForCausalLM(MistralConfig(sliding_window=window, **kw)) if window
                    else LlamaForCausalLM(LlamaConfig(**kw))).eval()
    finally:
        torch.set_default_dtype(torch.float32)
    shapes = {n: (m.in_features, m.out_features) for n, m in base.named_modules()
              if isinstance(m, torch.nn.Linear) and any(n.endswith("." + t) for t in TARGETS)}
    model = PolyLoraModel(base, PolyLoraConfig(max_gpu_adapters=3, max_rank=16, target_modules=TARGETS,
                                               enforce_right_padding=False))
    g = torch.Generator().manual_seed(1)
    for a in range(4):
        r = [4, 8, 16, 16][a]
        model.adapter_store.add_adapter(f"a{a}", {
            name: CpuLayerWeights(A=torch.randn(k, r, generator=g) * 0.1, B=torch.randn(r, n, generator=g) * 0.1, rank=r,
                                  scale=1.0) for name, (k, n) in shapes.items()})
    return model


def _whole(model, seq, adapter):
    """Logits of every position of one sequence, without a cache."""
    ids = torch.tensor([seq], device=model.base_model.device)
    return model(input_ids=ids, adapter_ids=[adapter], use_cache=False).logits[0]


def _close(got, want, dtype):
    """Two orders of the same fp32 sums through two layers; 16-bit activations
    round at each of their ~20 steps: eps / 2 each of values near the logits' size."""
    tol = (2e-4 if dtype == torch.float32 else 20 * torch.finfo(dtype).eps) * float(want.float().abs().max())
    assert float((got.float() - want.float()).abs().max()) <= tol


@pytest.mark.parametrize("dtype,window,page", [(torch.float32, None, 16), (torch.float32, None, 5), (torch.bfloat16, None, 16),
                                               (torch.float32, 20, 8)])
def test_prompts_and_steps_match_whole_sequences(cuda_status_clean, dtype, window, page):
    dev = torch.device("cuda")
    model = _model(dev, dtype, window=window)
    cache = PagedKVCache(2, 60, page, 2, 32, dtype, dev)
    model.attach_kv_cache(cache)
    g = torch.Generator().manual_seed(2)
    seqs = {n: torch.randint(0, VOCAB, (k,), generator=g).tolist() for n, k in (("x", 30), ("y", 7), ("z", 1))}
    adapters = {"x": "a0", "y": "__base__", "z": "a2"}
    with torch.inference_mode():
        names = ["x", "y", "z"]
        batch = cache.batch(names, [len(seqs[n]) for n in names])
        ids = torch.zeros(3, batch.max_new, dtype=torch.long, device=dev)
        for b, n in enumerate(names):
            ids[b, :len(seqs[n])] = torch.tensor(seqs[n])
        out = model(input_ids=ids, adapter_ids=[adapters[n] for n in names], paged=batch).logits
        for b, n in enumerate(names):
            _close(out[b, :len(seqs[n])], _whole(model, seqs[n], adapters[n]), dtype)
        for step in range(5):  # rows change order, one leaves and a new one joins
            if step == 2:
                cache.free("y")
                names, seqs["w"], adapters["w"] = ["w", "z", "x"], [3], "a3"
            new = torch.randint(0, VOCAB, (3,), generator=g).tolist()
            if step == 2:
                new[0] = 3
            for n, t in zip(names, new):
                if not (step == 2 and n == "w"):
                    seqs[n].append(t)
            out = model(input_ids=torch.tensor(new, device=dev)[:, None], adapter_ids=[adapters[n] for n in names],
                        paged=cache.batch(names)).logits
            for b, n in enumerate(names):
                _close(out[b, 0], _whole(model, seqs[n], adapters[n])[-1], dtype)
        # several tokens at once after a history, fewer of them in one row
        more = torch.randint(0, VOCAB, (2, 4), generator=g)
        seqs["x"] += more[0].tolist()
        seqs["z"] += more[1, :2].tolist()
        out = model(input_ids=more.to(dev), adapter_ids=["a0", "a2"], paged=cache.batch(["x", "z"], [4, 2])).logits
        _close(out[0], _whole(model, seqs["x"], "a0")[-4:], dtype)
        _close(out[1, :2], _whole(model, seqs["z"], "a2")[-2:], dtype)
        # a step taken back and made again
        cache.truncate("x", len(seqs["x"]) - 4)
        out2 = model(input_ids=more[:1].to(dev), adapter_ids=["a0"], paged=cache.batch(["x"], [4])).logits
        _close(out2[0], out[0], dtype)


def test_captured_steps_with_rules_match_eager(cuda_status_clean):
    """Append, attention and rules in one captured step, replayed over growing
    sequences and changing adapters and rules, equal the eager steps bit for bit."""
    dev, dtype = torch.device("cuda"), torch.bfloat16
    model = _model(dev, dtype, heads=8, kv_heads=2, head_dim=64)
    caches = [PagedKVCache(2, 80, 16, 2, 64, dtype, dev) for _ in range(2)]
    g = torch.Generator().manual_seed(3)
    names, ids = ["p", "q", "r"], ["a0", "__base__", "a1"]
    prompt = torch.randint(0, VOCAB, (3, 40), generator=g).to(dev)
    lens = [40, 13, 1]

    def rules(step):
        h = torch.Generator().manual_seed(10 + step)
        r = LogitRules(tokens=torch.randint(0, VOCAB, (3, 50), generator=h),
                       token_lens=torch.tensor([50, 20 + step, 0], dtype=torch.int32),
                       prompt_lens=torch.tensor([10, 0, 0], dtype=torch.int32), repetition_penalty=torch.rand(3, generator=h) + 1,
                       frequency_penalty=torch.rand(3, generator=h), bias_tokens=torch.randint(-1, VOCAB, (3, 6), generator=h),
                       bias_values=torch.randn(3, 6, generator=h),
                       allowed=torch.randint(-2**31, 2**31, (3, (VOCAB + 31) // 32), generator=h).to(torch.int32))
        return LogitRules(**{k: v.to(dev) if v is not None else None for k, v in vars(r).items()})

    with torch.inference_mode():
        token = prompt[:, :1]
        for cache in caches:
            model.attach_kv_cache(cache)
            model(input_ids=prompt, adapter_ids=ids, paged=cache.batch(names, lens))
        model.attach_kv_cache(caches[0])
        eager, feed = [], token
        steps = [(ids, 0), (["a2", "a0", "a2"], 1), (["a3", "a3", "__base__"], 2), (ids, 3)]
        for who, step in steps:
            out = model(input_ids=feed, adapter_ids=who, paged=caches[0].batch(names, width=8), logit_rules=rules(step)).logits
            assert bool(torch.isinf(out).any()) and not bool(torch.isnan(out).any())
            eager.append(out.clone())
            feed = out[:, 0].argmax(-1, keepdim=True)
        model.attach_kv_cache(caches[1])
        first = caches[1].batch(names, width=8)
        graphed = GraphedForward(model, ids, output=lambda o: o.logits, paged=first, logit_rules=rules(0), input_ids=token)
        feed = token
        for i, (who, step) in enumerate(steps):
            batch = first if i == 0 else caches[1].batch(names, width=8)
            out = graphed(who, paged=batch, logit_rules=rules(step), input_ids=feed)
            assert torch.equal(out, eager[i]), i
            feed = out[:, 0].argmax(-1, keepdim=True)
        with pytest.raises(ValueError):
            graphed(ids, input_ids=feed)
        with pytest.raises(ValueError):
            graphed(ids, paged=caches[1].batch(names), input_ids=feed)


def test_gradients_are_refused(cuda_status_clean):
    from polylora_b200.logits import apply_logit_rules
    from polylora_b200.paged import paged_append, paged_attention

    dev = torch.device("cuda")
    kc, table, lens = torch.zeros(1, 1, 4, 16, device=dev), torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.ones(1, device=dev)
    q = torch.zeros(1, 2, 16, device=dev, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        paged_attention(q, kc, kc, table, lens)
    with pytest.raises(RuntimeError, match="no gradient"):
        paged_append(None, q[None, :, :1], q[None, :, :1], kc, kc.clone(), table, lens)
    with pytest.raises(RuntimeError, match="no gradient"):
        apply_logit_rules(q[0], LogitRules())
    with torch.no_grad():
        assert paged_attention(q, kc, kc, table, lens).shape == (1, 2, 16)
