"""Which decoders the paged forward is attached to: those whose own attention
gives the same.  Random models of the installed transformers, on the CPU."""

import pytest
import torch

from polylora_b200 import PolyLoraConfig, PolyLoraModel
from polylora_b200.kv_cache import PagedKVCache, attach, attention_modules
from polylora_b200.kv_check import paged_formula
from polylora_b200.paged import paged_append, paged_attention, rotary_phases

YARN = dict(rope_type="yarn", rope_theta=1e4, factor=4.0, original_max_position_embeddings=64, beta_fast=32.0, beta_slow=1.0)


def _base(name, dtype=torch.float32, **kw):
    transformers = pytest.importorskip("transformers")
    sizes = dict(vocab_size=100, hidden_size=128, intermediate_size=64, num_hidden_layers=4, num_attention_heads=8,
                 num_key_value_heads=2, head_dim=16, max_position_embeddings=256, pad_token_id=0, bos_token_id=1, eos_token_id=2)
    if not hasattr(transformers, name + "Config"):
        pytest.skip(f"no {name} in this transformers")
    torch.manual_seed(0)
    torch.set_default_dtype(dtype)
    try:
        return getattr(transformers, name + "ForCausalLM")(getattr(transformers, name + "Config")(**{**sizes, **kw})).eval()
    finally:
        torch.set_default_dtype(torch.float32)


def _attach(base, pages=20, **kw):
    modules = attention_modules(base)
    dim = int(modules[0].head_dim)
    cache = PagedKVCache(len(modules), pages, 16, modules[0].k_proj.out_features // dim, dim, torch.float32, "cpu")
    attach(base, cache, **kw)


@pytest.mark.parametrize("name,kw,interleaved", [
    ("Llama", {}, False), ("Mistral", dict(sliding_window=40), False), ("Mistral", dict(sliding_window=None), False),
    ("Qwen2", {}, False), ("Granite", {}, False), ("Gemma", {}, False), ("StableLm", {}, False),
    ("Starcoder2", {}, False), ("Mixtral", {}, False), ("Llama", dict(rope_parameters=YARN), False),
    ("Cohere", {}, True), ("Glm", {}, True), ("Glm4", {}, True), ("Helium", {}, True),
    ("Ernie4_5", {}, True),
])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attaches_to_decoders_of_one_rotation(name, kw, interleaved, dtype):
    base = _base(name, dtype, **kw)
    ids = torch.arange(14).view(2, 7)
    with torch.no_grad():
        want = base(input_ids=ids).logits
    names, training = sorted(base.state_dict()), [m.training for m in base.modules()]
    modules = attention_modules(base)
    forwards = [m.forward for m in modules]
    with pytest.raises(ValueError, match="pass interleaved=" + str(interleaved)):
        _attach(base, interleaved=not interleaved)
    assert forwards == [m.forward for m in modules]  # nothing attached, all as it was
    _attach(base, interleaved=interleaved)
    assert sorted(base.state_dict()) == names and [m.training for m in base.modules()] == training
    assert forwards == [m.forward.original for m in modules]
    with torch.no_grad():
        assert torch.equal(base(input_ids=ids).logits, want)
    # once more, as wrapped layers in training
    model = PolyLoraModel(base.train(), PolyLoraConfig(max_gpu_adapters=2, max_rank=8, target_modules=["q_proj", "o_proj"]))
    model.attach_kv_cache(modules[0].forward.cache, interleaved=interleaved)
    assert base.training and all(m.training for m in modules) and forwards == [m.forward.original for m in modules]


@pytest.mark.parametrize("name,kw,match", [
    ("Cohere2", dict(sliding_window=30), "layer 3"),  # its last layer does not rotate
    ("Ministral3", dict(rope_parameters=dict(YARN, llama_4_scaling_beta=0.1, mscale=1.0, mscale_all_dim=1.0)),
     "positions 232 to 255"),                                          # queries scaled by position
    ("MiniMax", {}, "mixes its tokens"),                               # linear attention between
])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_refuses_what_it_would_answer_differently(name, kw, match, dtype):
    interleaved = name == "Cohere2"
    for inv_freq in (None, "own"):
        base = _base(name, dtype, **kw)
        modules = attention_modules(base)
        forwards = [m.forward for m in modules]
        given = {} if inv_freq is None else dict(inv_freq=base.model.rotary_emb.inv_freq.clone(),
                                                 rotary_scale=base.model.rotary_emb.attention_scaling)
        with pytest.raises(ValueError, match=match):
            _attach(base, interleaved=interleaved, **given)
        assert forwards == [m.forward for m in modules]
    _attach(base, interleaved=interleaved, check=False)  # the caller knows better
    assert forwards != [m.forward for m in modules]


def test_positions_that_the_cache_cannot_hold_do_not_count():
    """Queries scaled from position 64 on, in a cache of 64 tokens."""
    beta = dict(YARN, llama_4_scaling_beta=0.1, mscale=1.0, mscale_all_dim=1.0)
    _attach(_base("Ministral3", rope_parameters=beta), pages=4)
    with pytest.raises(ValueError, match="positions 72 to 95"):
        _attach(_base("Ministral3", rope_parameters=beta), pages=6)


@pytest.mark.parametrize("change", ["scale", "window", "no window", "causal", "output", "one layer"])
def test_sees_changes_of_single_modules(change):
    """Terms that no attribute names."""
    base = _base("Mistral", sliding_window=40)
    modules = attention_modules(base)
    m = modules[2]
    original = m.forward
    if change == "window":      # the module says one thing and its mask another
        m.sliding_window = 30
    elif change == "no window":  # a mask that nothing names
        base.config.sliding_window = None
        for x in modules:
            x.sliding_window = None
        m.forward = lambda hidden_states, *a, **k: original(hidden_states, *a, **{**k, "attention_mask": _mask(hidden_states, 40)})
    elif change == "scale":
        m.forward = lambda hidden_states, *a, **k: (setattr(m, "scaling", 0.2), original(hidden_states, *a, **k))[1]
        m.scaling = 0.25
    elif change == "causal":
        m.forward = lambda hidden_states, *a, **k: original(hidden_states, *a, **{**k, "attention_mask": _mask(hidden_states, 0)})
    elif change == "output":
        m.forward = lambda hidden_states, *a, **k: _scaled(m, original, hidden_states, a, k)
    else:                       # turned by other angles
        def other(hidden_states, position_embeddings, *a, **k):
            cos, sin = position_embeddings
            return original(hidden_states, (cos, -sin), *a, **k)

        def wrong(hidden_states, position_embeddings, *a, **k):
            cos, sin = position_embeddings
            return original(hidden_states, (cos, sin.roll(1, -1)), *a, **k)

        m.forward = other  # turned the other way scores are different
        with pytest.raises(ValueError, match="layer 2"):
            _attach(base)
        m.forward = wrong
    with pytest.raises(ValueError, match="layer 2"):
        _attach(base)


def _mask(hidden, window):
    n = hidden.shape[1]
    at = torch.arange(n)
    seen = (at[None, :] <= at[:, None]) & (at[None, :] > at[:, None] - window) if window else torch.ones(n, n, dtype=torch.bool)
    return torch.zeros(n, n).masked_fill(~seen, torch.finfo(torch.float32).min)[None, None]


def _scaled(m, original, hidden, a, k):
    """Attention whose output is weighted by head before it is projected."""
    inner = m.o_proj

    class Weighted(torch.nn.Module):
        def forward(self, x):
            return inner(x * torch.linspace(0.8, 1, x.shape[-1]))

    m.o_proj = Weighted()
    try:
        return original(hidden, *a, **k)
    finally:
        m.o_proj = inner


def test_layers_that_a_forward_does_not_reach_and_models_it_cannot_run():
    base = _base("Llama")
    base.model.layers[3].forward = lambda hidden_states, *a, **k: hidden_states
    with pytest.raises(ValueError, match=r"does not reach its attention layers \[3\]"):
        _attach(base)

    class Bare(torch.nn.Module):
        def __init__(self, inner):
            super().__init__()
            self.inner = inner

        def forward(self, tokens):
            return self.inner(input_ids=tokens)

    with pytest.raises(ValueError, match="check=False"):
        _attach(Bare(_base("Llama")), inv_freq=torch.ones(8))
    _attach(Bare(_base("Llama")), inv_freq=torch.ones(8), check=False)


def test_frequencies_that_renew_themselves_are_put_back():
    """A rotary embedding that takes other frequencies past its length, given
    frequencies of the caller's."""
    base = _base("Llama", rope_parameters=dict(rope_type="dynamic", rope_theta=1e4, factor=4.0), max_position_embeddings=32)
    rotary = base.model.rotary_emb
    base.config.max_position_embeddings = 256
    held, keys = rotary.inv_freq, sorted(rotary.__dict__)
    _attach(base, inv_freq=held.clone())
    assert rotary.inv_freq is held and sorted(rotary.__dict__) == keys and rotary.max_seq_len_cached == 32


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved,window,pairs", [(False, 0, 16), (True, 0, 16), (False, 7, 8), (True, 30, 5)])
def test_the_formula_is_the_operators(cuda_status_clean, interleaved, window, pairs):
    g, dev = torch.Generator().manual_seed(1), torch.device("cuda")
    start, new, heads, kv, dim, page = 1000, 20, 6, 2, 32, 8
    freq = torch.rand(pairs, generator=g, dtype=torch.float64)
    q, k, v = (torch.randn(2, new, n, dim, generator=g) for n in (heads, kv, kv))
    table = torch.arange(2 * 130, dtype=torch.int32, device=dev).view(2, 130)
    kc, vc = (torch.zeros(260, kv, page, dim, device=dev) for _ in range(2))
    past = torch.full((2,), start, dtype=torch.int32, device=dev)
    turned, _ = paged_append(q.to(dev), k.to(dev), v.to(dev), kc, vc, table, past, phases=rotary_phases(freq.to(dev)),
                             interleaved=interleaved, rotary_scale=1.25)
    want = paged_formula(q, k, v, start, freq, interleaved=interleaved, rotary_scale=1.25, scale=0.2,
                         window=window or new, last=1)[:, 0]
    got = paged_attention(turned[:, -1], kc, vc, table, past + new, scale=0.2, window=min(window or new, new))  # its past is empty
    # sums of 32 products of rotated 32-bit numbers, and of 20 tokens: 2^-24 a step
    assert float((got.double().cpu() - want).abs().max()) <= 200 * 2.0**-24 * float(v.abs().max())
