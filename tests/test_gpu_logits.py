"""Per-row logit rules against a plain 64-bit implementation."""

import math

import pytest
import torch

from polylora_b200.logits import LogitRules, apply_logit_rules

pytestmark = pytest.mark.gpu

BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32


def _reference(x, r):
    """(values, bound of the 32-bit roundings) in 64 bits, row by row."""
    y, slack = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    B, V = x.shape
    one = torch.ones(B)
    rep, pres, freq = (t if t is not None else d for t, d in ((r.repetition_penalty, one), (r.presence_penalty, 0 * one),
                                                             (r.frequency_penalty, 0 * one)))
    for b in range(B):
        if r.tokens is not None:
            n = int(r.token_lens[b]) if r.token_lens is not None else r.tokens.shape[1]
            p = int(r.prompt_lens[b]) if r.prompt_lens is not None else 0
            hist = r.tokens[b, :max(n, 0)].tolist()
            count = {}
            for i, t in enumerate(hist):
                if 0 <= t < V:
                    count[t] = count.get(t, 0) + (i >= p)
            for t, c in count.items():
                v = float(y[b, t])
                v = v / float(rep[b]) if v > 0 else v * float(rep[b])
                slack[b, t] += abs(v) if math.isfinite(v) else 0
                if c:
                    v -= float(freq[b]) * c + float(pres[b])
                    slack[b, t] += 2 * abs(float(freq[b])) * c + 2 * abs(float(pres[b]))
                y[b, t] = v
        if r.bias_tokens is not None:
            for t, v in zip(r.bias_tokens[b].tolist(), r.bias_values[b].tolist()):
                if 0 <= t < V:
                    slack[b, t] += abs(float(y[b, t])) + abs(v) if math.isfinite(float(y[b, t])) else 0
                    y[b, t] += v
        if r.allowed is not None:
            words = r.allowed[b].long() & 0xFFFFFFFF
            bits = (words[:, None] >> torch.arange(32)) & 1
            y[b, bits.flatten()[:V] == 0] = -math.inf
    # at most six roundings of 2^-24 on values no larger than what slack adds up
    return y, 6 * 2.0**-24 * slack


def _check(got, ref, slack, dtype):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf])
    fine = torch.isfinite(ref)
    half = torch.finfo(dtype).eps / 2
    tol = half * ref.abs() + slack * (1 + half) + torch.finfo(dtype).smallest_normal * half * 2
    assert bool(((got - ref).abs()[fine] <= tol[fine]).all()), float((got - ref).abs()[fine].max())


def _rules(g, B, V, L, K, mask, wide, everything=True):
    ids = torch.int64 if wide else torch.int32
    r = LogitRules()
    if L is not None:
        r.tokens = torch.randint(-2, V + 2, (B, L), generator=g).to(ids)  # some outside the vocabulary
        if L > 3:
            r.tokens[:, L // 2] = r.tokens[:, 0]  # repeats across prompt and answer
            r.tokens[:, -1] = r.tokens[:, L // 2 + 1]
        if everything:
            r.token_lens = torch.tensor([[L, 0, L // 2, L + 9, -1][b % 5] for b in range(B)], dtype=torch.int32).clamp(max=L)
            r.prompt_lens = torch.tensor([[L // 3, 0, L, 1][b % 4] for b in range(B)], dtype=torch.int32)
            r.repetition_penalty = torch.rand(B, generator=g) + 0.7
            r.frequency_penalty = torch.rand(B, generator=g) - 0.3
        r.presence_penalty = torch.rand(B, generator=g)
    if K is not None:
        r.bias_tokens = torch.randint(-1, V + 1, (B, K), generator=g).to(ids)
        r.bias_values = torch.randn(B, K, generator=g) * 4
        if K > 5:
            r.bias_tokens[:, 4] = r.bias_tokens[:, 1]
            r.bias_tokens[:, -1] = r.bias_tokens[:, 1]
    if mask:
        r.allowed = torch.randint(-2**31, 2**31, (B, (V + 31) // 32), generator=g).to(torch.int32)
        r.allowed[-1] = 0  # a row whose mask leaves nothing
    return r


def _to(r, dev):
    return LogitRules(**{k: (v.to(dev) if v is not None else None) for k, v in vars(r).items()})


CASES = [
    # B, V, history, biases, mask, dtype, wide
    (1, 128256, 300, 8, True, BF, True),
    (5, 50257, 1000, 300, True, FH, False),
    (4, 50257, 100, None, False, F32, True),
    (3, 8193, 40, 9, True, BF, False),        # one entry past a chunk
    (6, 1, 5, 3, True, F32, True),
    (2, 31, None, 40, True, BF, True),
    (2, 33, 7, None, True, FH, False),
    (3, 20000, None, None, True, BF, False),
    (3, 20001, None, None, False, F32, False),
    (2, 9000, 0, 0, False, BF, True),
    (2, 300, 5000, 4096, True, BF, True),     # lists longer than the vocabulary: many repeats
    (200, 3001, 60, 9, True, FH, True),       # rows by lists
    (170, 3001, 600, None, False, BF, False),
    (151, 900, None, 70, True, F32, True),
    (3, 300000, 9000, 20, True, BF, True),    # more than one part of the vocabulary
    (80, 300000, 40, 5, False, BF, True),
    (33, 50257, 200, 64, True, FH, True),     # small parts: one launch copies and applies
    (60, 40001, 70, 300, True, BF, True),     # larger ones: two kernels side by side
    (140, 17000, 30, 600, False, F32, False),
    (2, 40, 10, 900, True, F32, True),        # each token's biases many times
]


@pytest.mark.parametrize("B,V,L,K,mask,dtype,wide", CASES)
def test_rules_match_64_bits(cuda_status_clean, B, V, L, K, mask, dtype, wide):
    g, dev = torch.Generator().manual_seed(V + B), torch.device("cuda")
    x = (torch.randn(B, V, generator=g) * 4).to(dtype)
    x[0, V // 2], x[-1, V // 3] = -math.inf, 0.0
    r = _rules(g, B, V, L, K, mask, wide)
    ref, slack = _reference(x, r)
    xd, rd = x.to(dev), _to(r, dev)
    got = apply_logit_rules(xd, rd)
    _check(got, ref, slack, dtype)
    assert torch.equal(xd.cpu(), x)
    # in place, and into rows of a wider buffer at any alignment
    wide_rows = torch.full((B, V + 5), 3.0, dtype=dtype, device=dev)
    for start in (0, 1, 5):
        view = wide_rows[:, start:start + V]
        assert apply_logit_rules(xd, rd, out=view) is view
        assert torch.equal(view, got)
    view.copy_(xd)
    assert torch.equal(apply_logit_rules(view, rd, out=view), got)
    assert torch.equal(apply_logit_rules(xd.clone(), rd), got)


def test_rows_around_the_output_stay(cuda_status_clean):
    dev, g = torch.device("cuda"), torch.Generator().manual_seed(1)
    x = torch.randn(3, 1001, generator=g).to(BF).to(dev)
    buf = torch.full((5, 1010), 2.0, dtype=BF, device=dev)
    r = _to(_rules(g, 3, 1001, 20, 4, True, True), dev)
    apply_logit_rules(x, r, out=buf[1:4, 3:1004])
    keep = torch.ones_like(buf, dtype=torch.bool)
    keep[1:4, 3:1004] = False
    assert bool((buf[keep] == 2.0).all())


def test_masked_nan_and_single_rules(cuda_status_clean):
    """NaN and infinities behind the mask become -inf, NaN elsewhere stays; each
    rule alone leaves the others at their neutral values."""
    dev, g = torch.device("cuda"), torch.Generator().manual_seed(2)
    x = torch.randn(2, 64, generator=g)
    x[:, 3], x[:, 4], x[:, 5] = math.nan, math.inf, math.nan
    allowed = torch.full((2, 2), -1, dtype=torch.int32)
    allowed[:, 0] = ~((1 << 3) | (1 << 4))
    for kw in (dict(allowed=allowed), dict(tokens=torch.tensor([[1, 1, 2], [7, 8, 9]]), repetition_penalty=torch.tensor([1.5, 0.5])),
               dict(tokens=torch.tensor([[1, 1, 2], [7, 8, 9]]), frequency_penalty=torch.tensor([1.5, 0.5])),
               dict(bias_tokens=torch.tensor([[1, 1, 1], [0, 63, -5]]), bias_values=torch.tensor([[1., 2., 3.], [4., 5., 6.]])),
               dict()):
        r = LogitRules(**kw)
        ref, slack = _reference(x, r)
        _check(apply_logit_rules(x.to(dev), _to(r, dev)), ref, slack, F32)


def test_strided_lists_and_mixed_types(cuda_status_clean):
    dev, g = torch.device("cuda"), torch.Generator().manual_seed(3)
    B, V = 4, 5000
    x = torch.randn(B, V, generator=g).to(FH)
    r = _rules(g, B, V, 50, 12, True, True)
    ref, slack = _reference(x, r)
    d = _to(r, dev)
    d.tokens = torch.zeros(B, 80, dtype=torch.int64, device=dev)[:, 10:60].copy_(d.tokens)
    d.bias_tokens = d.bias_tokens.to(torch.int32)
    d.bias_values = d.bias_values.t().contiguous().t()
    d.allowed = torch.cat([d.allowed, torch.zeros_like(d.allowed)], dim=1)
    d.token_lens = d.token_lens.to(torch.int64)
    _check(apply_logit_rules(x.to(dev), d), ref, slack, FH)
    d.tokens = d.tokens[:1].expand(B, 50)  # one history for every row
    r.tokens = r.tokens[:1].expand(B, 50)
    ref, slack = _reference(x, r)
    _check(apply_logit_rules(x.to(dev), d), ref, slack, FH)


@pytest.mark.parametrize("B,V", [(3, 40000), (300, 5000)])  # rules by their finders, and by lists
def test_captured_rules_follow_their_buffers(cuda_status_clean, B, V):
    dev, g = torch.device("cuda"), torch.Generator().manual_seed(4)
    x = torch.randn(B, V, generator=g).to(BF).to(dev)
    r = _to(_rules(g, B, V, 64, 16, True, True), dev)
    out = torch.empty_like(x)
    gr = torch.cuda.CUDAGraph()
    apply_logit_rules(x, r, out=out)
    with torch.cuda.graph(gr):
        apply_logit_rules(x, r, out=out)
    for k in range(3):
        r.tokens.random_(0, V)
        r.token_lens.fill_(64 - k)
        x.mul_(0.5)
        gr.replay()
        assert torch.equal(out, apply_logit_rules(x, r))
        got = x.clone()
        assert torch.equal(apply_logit_rules(got, r, out=got), out)


def test_two_streams_of_listed_rules(cuda_status_clean):
    dev, g = torch.device("cuda"), torch.Generator().manual_seed(5)
    B, V = 300, 20000
    xs = [torch.randn(B, V, generator=g).to(BF).to(dev) for _ in range(2)]
    rs = [_to(_rules(g, B, V, 200, 16, True, True), dev) for _ in range(2)]
    want = [apply_logit_rules(x, r) for x, r in zip(xs, rs)]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(apply_logit_rules(xs[i], rs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_empty(cuda_status_clean):
    dev = torch.device("cuda")
    assert apply_logit_rules(torch.zeros(0, 10, device=dev), LogitRules()).shape == (0, 10)
    assert apply_logit_rules(torch.zeros(2, 0, device=dev), LogitRules()).shape == (2, 0)
