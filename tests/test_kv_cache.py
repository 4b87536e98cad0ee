"""Host side of the paged cache: pages, lengths, batches, and what attach and
the forward refuse.  No GPU."""

import pytest
import torch

from polylora_b200 import PolyLoraConfig, PolyLoraModel
from polylora_b200.kv_cache import PagedKVCache, attention_modules, get_paged_batch
from polylora_b200.logits import LogitRules
from polylora_b200.model import apply_output_rules


def _cache(pages=10, size=4, layers=2, heads=2, dim=16):
    return PagedKVCache(layers, pages, size, heads, dim, torch.float32, "cpu")


def _used(batch, b, size=4):
    n = -(-int(batch.seq_lens[b]) // size)
    return batch.page_table[b, :n].tolist()


def test_batches_take_and_keep_pages():
    c = _cache()
    one = c.batch(["a", "b", "c"], [5, 0, 8])
    assert one.page_table.shape == (3, 2) and one.page_table.dtype == torch.int32 and one.max_new == 8 and one.fresh
    assert one.past_lens.tolist() == [0, 0, 0] and one.new_lens.tolist() == [5, 0, 8] and one.seq_lens.tolist() == [5, 0, 8]
    assert c.free_pages == 6 and c.length("a") == 5 and c.length("b") == 0
    assert one.page_table[1].tolist() == [-1, -1]
    pages = _used(one, 0) + _used(one, 2)
    assert len(set(pages)) == 4 and all(0 <= p < 10 for p in pages)
    two = c.batch(["c", "a"], width=5)  # one token each
    assert not two.fresh and two.max_new == 1 and two.page_table.shape == (2, 5)
    assert two.past_lens.tolist() == [8, 5] and two.seq_lens.tolist() == [9, 6]
    assert _used(two, 0)[:2] == _used(one, 2) and _used(two, 1) == _used(one, 0)
    assert c.free_pages == 5
    assert two.page_table.is_contiguous() and two.past_lens.is_contiguous()


def test_out_of_pages_takes_nothing():
    c = _cache(pages=3)
    c.batch(["a"], 9)
    with pytest.raises(RuntimeError, match="0 free pages"):
        c.batch(["a", "b"], [3, 1])
    assert c.length("a") == 9 and c.length("b") == 0 and c.free_pages == 0
    c.batch(["a"], 3)  # fits in the last page
    c.free("a")
    assert c.free_pages == 3 and c.length("a") == 0
    c.free("unknown")


def test_truncate_frees_whole_pages():
    c = _cache()
    c.batch(["a"], 13)
    c.truncate("a", 8)
    assert c.length("a") == 8 and c.free_pages == 8
    assert c.batch(["a"], 1).seq_lens.tolist() == [9] and c.free_pages == 7
    for bad in (-1, 10):
        with pytest.raises(ValueError):
            c.truncate("a", bad)


def test_batch_arguments():
    c = _cache()
    for kw in (dict(seqs=["a", "a"]), dict(seqs=["a"], new_lens=[1, 2]), dict(seqs=["a"], new_lens=[-1]),
               dict(seqs=["a"], new_lens=[3], max_new=2), dict(seqs=["a"], new_lens=[9], width=2)):
        with pytest.raises(ValueError):
            c.batch(**kw)
    assert c.free_pages == 10
    empty = c.batch([])
    assert empty.rows == 0 and empty.page_table.shape == (0, 1)
    for bad in ((0, 1, 1, 1, 8), (1, 1, 0, 1, 8)):
        with pytest.raises(ValueError):
            PagedKVCache(*bad, torch.float32, "cpu")


def test_captured_batches_keep_their_shape():
    c, other = _cache(), _cache()
    static = c.batch(["a", "b"], width=3).clone()
    new = c.batch(["b", "c"], width=3)
    with pytest.raises(ValueError):  # a prompt's batch is not a step's
        static.copy_(c.batch(["d", "e"], [2, 2], width=3))
    static2 = c.batch(["a", "b"], width=3).clone()
    static2.copy_(c.batch(["a", "b"], width=3))
    assert static2.past_lens.tolist() == [2, 3]
    for bad in (c.batch(["a"], width=3), c.batch(["a", "b"], width=4), other.batch(["a", "b"], width=3)):
        with pytest.raises(ValueError):
            static2.copy_(bad)
    assert new.rows == 2


def _llama(**kw):
    from transformers import LlamaConfig, LlamaModel

    cfg = LlamaConfig(vocab_size=50, hidden_size=64, intermediate_size=64, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, max_position_embeddings=64, **kw)
    return LlamaModel(cfg).eval()


def _wrapped(base):
    return PolyLoraModel(base, PolyLoraConfig(max_gpu_adapters=2, max_rank=8, target_modules=["q_proj", "o_proj"]))


def test_attach_keeps_names_and_plain_forwards():
    base = _llama()
    ids = torch.arange(12).view(2, 6)
    with torch.no_grad():
        want = base(input_ids=ids).last_hidden_state
    model = _wrapped(base)
    names = sorted(base.state_dict())
    assert len(attention_modules(base)) == 2
    model.attach_kv_cache(_cache())
    model.attach_kv_cache(_cache())  # another cache takes the first one's place
    assert sorted(base.state_dict()) == names
    with torch.no_grad():
        assert torch.equal(model(input_ids=ids).last_hidden_state, want)


def test_attach_refusals():
    model = _wrapped(_llama())
    for cache in (_cache(layers=3), _cache(heads=1), _cache(dim=32)):
        with pytest.raises(ValueError):
            model.attach_kv_cache(cache)
    model.base_model.rotary_emb.rope_type = "dynamic"
    with pytest.raises(ValueError, match="dynamic"):
        model.attach_kv_cache(_cache())
    model.attach_kv_cache(_cache(), inv_freq=torch.ones(8))  # given, none is looked for
    del model.base_model.rotary_emb.inv_freq
    with pytest.raises(ValueError, match="inv_freq"):
        model.attach_kv_cache(_cache())


@pytest.mark.parametrize("name,value,match", [
    ("sinks", torch.nn.Parameter(torch.zeros(4)), "sinks"), ("is_causal", False, "causal"), ("use_rope", 0, "rotate"),
    ("attn_logit_softcapping", 50.0, "softcapping"), ("config.clip_qkv", 8.0, "clip_qkv"),
    ("config.layer_types", ["full_attention", "chunked_attention"], "chunked"),
])
def test_attach_refuses_other_attention(name, value, match):
    """Terms that the paged forward leaves out, in any layer."""
    model = _wrapped(_llama())
    module = attention_modules(model.base_model)[1]
    owner = module.config if name.startswith("config.") else module
    setattr(owner, name.removeprefix("config."), value)
    forward = module.forward
    with pytest.raises(ValueError, match=match):
        model.attach_kv_cache(_cache())
    assert module.forward == forward  # nothing attached


def test_forward_refusals():
    model, cache = _wrapped(_llama()), _cache()
    model.attach_kv_cache(cache)
    batch = cache.batch(["a", "b"], 3)
    ids = torch.zeros(2, 3, dtype=torch.long)
    with pytest.raises(ValueError, match="attention_mask"):
        model(input_ids=ids, paged=batch, attention_mask=torch.ones(2, 3))
    with torch.no_grad():
        with pytest.raises(ValueError, match="2 x 3"):
            model(input_ids=ids[:, :2], paged=batch)
        with pytest.raises(ValueError, match="another cache"):
            model(input_ids=ids, paged=_cache().batch(["a", "b"], 3))
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            model(input_ids=ids, paged=batch)
    assert get_paged_batch() is None


def test_output_rules_refusals():
    with pytest.raises(ValueError, match="logits"):
        apply_output_rules(object(), LogitRules())
    with pytest.raises(ValueError, match="one token per row"):
        apply_output_rules(torch.zeros(2, 3, 5), LogitRules())
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        apply_output_rules(torch.zeros(2, 1, 5), LogitRules())
    r = LogitRules(tokens=torch.zeros(2, 3, dtype=torch.long), presence_penalty=torch.zeros(2))
    mine = r.clone()
    mine.copy_(LogitRules(tokens=torch.ones(2, 3, dtype=torch.long), presence_penalty=torch.ones(2)))
    assert mine.tokens.sum() == 6 and r.tokens.sum() == 0
    for bad in (LogitRules(), LogitRules(tokens=torch.ones(2, 4, dtype=torch.long), presence_penalty=torch.ones(2))):
        with pytest.raises(ValueError):
            mine.copy_(bad)
