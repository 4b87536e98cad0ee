"""The paged forward around plain stand-ins for the two operators, on the CPU."""

import pytest
import torch

from polylora_b200 import kv_cache
from polylora_b200.kv_cache import PagedKVCache, attach, use_paged_batch
from test_kv_cache import _llama


def _append(q, k, v, kc, vc, table, past, news, *, phases, interleaved, rotary_scale, return_keys):
    pairs = phases.shape[0]
    angle = (past[:, None] + torch.arange(q.shape[1])).double()[..., None] * (phases.double() / 2.0**64 * 2 * torch.pi)
    c, s = (t[:, :, None].float() * rotary_scale for t in (angle.cos(), angle.sin()))

    def turned(x):
        a, b = x[..., :pairs], x[..., pairs:2 * pairs]
        return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * pairs:]], -1)

    q, k = turned(q), turned(k)
    page = kc.shape[2]
    for b in range(q.shape[0]):
        for m in range(int(news[b])):
            at = int(past[b]) + m
            kc[table[b, at // page], :, at % page], vc[table[b, at // page], :, at % page] = k[b, m], v[b, m]
    return q, k if return_keys else None


def _attend(limit):
    def attend(q, kc, vc, table, lens, *, scale, window=0, out=None):
        assert q.shape[0] <= limit and table.shape[0] == q.shape[0] == lens.shape[0]
        out = torch.empty_like(q) if out is None else out
        page, group = kc.shape[2], q.shape[1] // kc.shape[1]
        for b, n in enumerate(lens.tolist()):
            at = torch.arange(max(0, n - window) if window else 0, n)
            k, v = (c[table[b, at // page].long(), :, at % page].repeat_interleave(group, 1) for c in (kc, vc))
            p = torch.softmax(torch.einsum("hd,nhd->hn", q[b], k) * scale, -1)
            out[b] = torch.einsum("hn,nhd->hd", p, v)
        return out
    return attend


@pytest.mark.parametrize("limit", [1 << 20, 5, 1])
def test_tokens_after_a_history_take_as_many_calls_as_rows_fit(monkeypatch, limit):
    """3 rows of up to 4 tokens after histories: rows of the operator beyond its
    limit, cut inside a sequence too, against forwards over the whole sequences."""
    monkeypatch.setattr(kv_cache, "paged_append", _append)
    monkeypatch.setattr(kv_cache, "paged_attention", _attend(limit))
    monkeypatch.setattr(kv_cache, "_MOST_ROWS", limit)
    base = _llama()
    cache = PagedKVCache(2, 40, 4, 2, 16, torch.float32, "cpu")
    attach(base, cache)
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(0, 50, (3, 13), generator=g)
    names, first, then = ["a", "b", "c"], [9, 1, 4], [4, 3, 1]
    with torch.no_grad():
        for counts, begin in ((first, [0, 0, 0]), (then, first)):
            batch = cache.batch(names, counts)
            feed = torch.zeros(3, batch.max_new, dtype=torch.long)
            for b in range(3):
                feed[b, :counts[b]] = ids[b, begin[b]:begin[b] + counts[b]]
            with use_paged_batch(batch):
                got = base(input_ids=feed, use_cache=False).last_hidden_state
            for b in range(3):
                want = base(input_ids=ids[b:b + 1, :begin[b] + counts[b]], use_cache=False).last_hidden_state[0, begin[b]:]
                assert torch.allclose(got[b, :counts[b]], want, atol=2e-5), (b, counts)
