"""Captured steps over sequences that begin, end and change."""

import pytest
import torch

from polylora_b200.graphed import GraphedForward
from polylora_b200.kv_cache import PagedKVCache
from test_gpu_decode import VOCAB, _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first", [True, False])
def test_a_step_captured_on_first_or_later_tokens_serves_both(cuda_status_clean, first):
    dev, dtype = torch.device("cuda"), torch.bfloat16
    model = _model(dev, dtype)
    ids = ["a0", "__base__"]
    g = torch.Generator().manual_seed(4)
    feed = torch.randint(0, VOCAB, (6, 2, 1), generator=g).to(dev)
    caches = [PagedKVCache(2, 20, 16, 2, 32, dtype, dev) for _ in range(2)]
    with torch.inference_mode():
        model.attach_kv_cache(caches[0])
        eager = []
        for step in range(6):
            if step == 3:
                caches[0].free("x"), caches[0].free("y")
            eager.append(model(input_ids=feed[step], adapter_ids=ids, paged=caches[0].batch(["x", "y"], width=4)).logits.clone())
        model.attach_kv_cache(caches[1])
        example = caches[1].batch(["x", "y"], width=4)
        if not first:  # capture on the second tokens
            model(input_ids=feed[0], adapter_ids=ids, paged=example)
            example = caches[1].batch(["x", "y"], width=4)
        step = GraphedForward(model, ids, output=lambda o: o.logits, paged=example, input_ids=feed[0 if first else 1])
        for i in range(0 if first else 1, 6):
            if i == 3:
                caches[1].free("x"), caches[1].free("y")
            batch = example if i == (0 if first else 1) else caches[1].batch(["x", "y"], width=4)
            assert torch.equal(step(ids, paged=batch, input_ids=feed[i]), eager[i]), i
