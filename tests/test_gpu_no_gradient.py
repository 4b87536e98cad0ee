"""The serving operators have no gradient: every input that would lose one is refused."""

import pytest
import torch
from torch.autograd import forward_ad

from polylora_b200.logits import LogitRules, apply_logit_rules
from polylora_b200.paged import paged_append, paged_attention

pytestmark = pytest.mark.gpu


def _calls(dev):
    """(tensors by name, call of them)."""
    def tensors():
        return dict(q=torch.ones(1, 1, 2, 16, device=dev), k=torch.ones(1, 1, 1, 16, device=dev),
                    v=torch.ones(1, 1, 1, 16, device=dev), k_cache=torch.zeros(1, 1, 4, 16, device=dev),
                    v_cache=torch.zeros(1, 1, 4, 16, device=dev))

    table, one = torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    ids = torch.zeros(1, 2, dtype=torch.int64, device=dev)

    def append(q, k, v, k_cache, v_cache):
        return paged_append(q, k, v, k_cache, v_cache, table, one)[0]

    def attend(q, k, v, k_cache, v_cache):
        return paged_attention(q[0], k_cache, v_cache, table, one)

    def rules(logits, repetition_penalty, presence_penalty, frequency_penalty, bias_values):
        return apply_logit_rules(logits, LogitRules(tokens=ids, repetition_penalty=repetition_penalty,
                                                    presence_penalty=presence_penalty, frequency_penalty=frequency_penalty,
                                                    bias_tokens=ids, bias_values=bias_values))

    def of_rules():
        return dict(logits=torch.ones(1, 5, device=dev), bias_values=torch.ones(1, 2, device=dev),
                    **{n: torch.ones(1, device=dev) for n in ("repetition_penalty", "presence_penalty", "frequency_penalty")})

    return [(append, tensors, ("q", "k", "v", "k_cache", "v_cache")), (attend, tensors, ("q", "k_cache", "v_cache")),
            (rules, of_rules, tuple(of_rules()))]


@pytest.mark.parametrize("which", [0, 1, 2])
def test_gradients_and_tangents_are_refused(cuda_status_clean, which):
    call, make, names = _calls(torch.device("cuda"))[which]
    plain = call(**make())
    for name in names:
        t = make()
        t[name].requires_grad_()
        with pytest.raises(RuntimeError, match="no gradient"):
            call(**t)
        with torch.no_grad():
            assert torch.equal(call(**t), plain)
        t = make()
        with forward_ad.dual_level():
            t[name] = forward_ad.make_dual(t[name], torch.ones_like(t[name]))
            with pytest.raises(RuntimeError, match="tangent"):
                call(**t)
            assert torch.equal(call(**make()), plain)  # tensors without one
