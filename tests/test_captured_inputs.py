"""What the captured copies of rules and batches take, and leave alone.  No GPU."""

import pytest
import torch

from polylora_b200.graphed import GraphedForward
from polylora_b200.kv_cache import PagedKVCache
from polylora_b200.logits import LogitRules


def _rules(ids=torch.int64, value=1, **kw):
    r = LogitRules(tokens=torch.full((2, 3), value, dtype=ids), token_lens=torch.full((2,), value, dtype=torch.int32),
                   repetition_penalty=torch.full((2,), float(value)), bias_tokens=torch.full((2, 4), value, dtype=ids),
                   bias_values=torch.full((2, 4), float(value)), allowed=torch.full((2, 1), value, dtype=torch.int32))
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def _same(a, b):
    return all((x is None) == (y is None) and (x is None or torch.equal(x, y)) for x, y in zip(vars(a).values(), vars(b).values()))


@pytest.mark.parametrize("other", [
    _rules(value=2),                                                    # int64 ids into int32: 2^32 + 5 would be token 5
    _rules(torch.int32, 2, bias_tokens=torch.full((2, 4), 2**32 + 5)),
    _rules(torch.int32, 2, tokens=torch.full((2, 3), 2.0)),
    _rules(torch.int32, 2, allowed=torch.full((2, 1), 2**40)),
    _rules(torch.int32, 2, allowed=None),
    _rules(torch.int32, 2, allowed=torch.full((2, 2), 2, dtype=torch.int32)),
    _rules(torch.int32, 2, presence_penalty=torch.ones(2)),
])
def test_rules_that_are_refused_leave_the_captured_ones_alone(other):
    mine = _rules(torch.int32)
    with pytest.raises(ValueError):
        mine.copy_(other)
    assert _same(mine, _rules(torch.int32))


def test_rules_of_other_types_that_are_taken():
    mine = _rules(torch.int64)
    mine.copy_(_rules(torch.int32, 2, token_lens=torch.full((2,), 2), bias_values=torch.full((2, 4), 2.0, dtype=torch.float64)))
    assert _same(mine, _rules(torch.int64, 2))


def _cache():
    return PagedKVCache(1, 10, 4, 1, 8, torch.float32, "cpu")


def test_one_token_steps_take_first_tokens_and_later_ones():
    """A step of one token a row computes the same whether rows have a past or not."""
    c = _cache()
    first = c.batch(["a", "b"], width=2).clone()
    later = c.batch(["a", "b"], width=2)
    assert first.fresh and not later.fresh
    captured_first, captured_later = first.clone(), later.clone()
    captured_first.copy_(later)
    assert captured_first.past_lens.tolist() == [1, 1]
    c.free("a"), c.free("b")
    new = c.batch(["x", "y"], width=2)
    assert new.fresh
    captured_later.copy_(new)
    assert captured_later.past_lens.tolist() == [0, 0] and captured_later.seq_lens.tolist() == [1, 1]


def test_longer_rows_keep_apart():
    """Rows of a prompt attend among themselves, later ones over the cache."""
    c = _cache()
    prompt = c.batch(["a"], 3, width=3).clone()
    more = c.batch(["a"], 3, width=3)
    for one, other in ((prompt, more), (more.clone(), prompt)):
        with pytest.raises(ValueError):
            one.copy_(other)


def _captured(paged, rules, refuse):
    """A captured forward's host side, without its graph."""
    step = GraphedForward.__new__(GraphedForward)
    step.paged, step.rules, step.static = paged, rules, {}

    def host_part(adapter_ids):
        raise refuse

    step._host_part = host_part
    return step


def test_refused_calls_leave_batch_and_rules_alone():
    c = _cache()
    batch, rules = c.batch(["a", "b"], width=2), _rules(torch.int32)
    later = c.batch(["a", "b"], width=2)
    for paged, new, match in (
            (later, _rules(value=2), "bias_tokens|tokens"),                # rules refused, the batch is not taken
            (c.batch(["a", "b"], width=3), _rules(torch.int32, 2), "width"),  # the batch refused, the rules are not
            (later, _rules(torch.int32, 2), "no such adapter")):           # both well, but the adapters are not
        step = _captured(batch.clone(), rules.clone(), ValueError("no such adapter"))
        with pytest.raises(ValueError, match=match):
            step(["x", "y"], paged=paged, logit_rules=new)
        assert step.paged.past_lens.tolist() == [0, 0] and _same(step.rules, rules)


def test_masks_that_a_paged_forward_would_not_look_at():
    from test_kv_cache import _llama, _wrapped
    from test_kv_cache import _cache as cache_of_llama

    model, c = _wrapped(_llama()), cache_of_llama()
    model.attach_kv_cache(c)
    batch, ids, mask = c.batch(["a", "b"], 3), torch.zeros(2, 3, dtype=torch.long), torch.ones(2, 3)
    with pytest.raises(ValueError, match="attention_mask"):
        GraphedForward(model, ["__base__"] * 2, paged=batch, input_ids=ids, attention_mask=mask)
    with pytest.raises(ValueError, match="by name"):
        model(ids, mask, paged=batch)
    with torch.no_grad():
        for args in ((ids,), (ids, None)):
            with pytest.raises(RuntimeError, match="no CPU fallback"):
                model(*args, paged=batch)


def test_rules_for_several_tokens_are_refused_before_the_forward(monkeypatch):
    from transformers import LlamaConfig, LlamaForCausalLM

    from test_kv_cache import _wrapped
    from test_kv_cache import _cache as cache_of_llama

    base = LlamaForCausalLM(LlamaConfig(vocab_size=50, hidden_size=64, intermediate_size=64, num_hidden_layers=2,
                                        num_attention_heads=4, num_key_value_heads=2, max_position_embeddings=64)).eval()
    model, c = _wrapped(base), cache_of_llama()
    model.attach_kv_cache(c)
    appended = []
    monkeypatch.setattr("polylora_b200.kv_cache.paged_append", lambda *a, **k: appended.append(a) or 1 / 0)
    ids, rules = torch.zeros(2, 3, dtype=torch.long), LogitRules()
    with torch.no_grad():
        for kw in ({}, dict(logits_to_keep=0)):
            with pytest.raises(ValueError, match="one token per row"):
                model(input_ids=ids, paged=c.batch(["a", "b"], 3), logit_rules=rules, **kw)
        assert not appended
        for kw, n in ((dict(logits_to_keep=1), 3), ({}, 1)):  # one token's logits: the forward begins
            with pytest.raises(ZeroDivisionError):
                model(input_ids=ids[:, :n], paged=c.batch(["a", "b"], n), logit_rules=rules, **kw)
