"""Paged cache operators against plain 64-bit implementations."""

import math

import pytest
import torch

from polylora_b200 import _native
from polylora_b200.paged import paged_append, paged_attention, rotary_phases

pytestmark = pytest.mark.gpu

HALF = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}  # a rounding is off by at most this, relative
BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32


def _dev():
    return torch.device("cuda")


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _table(lens, page, g, extra=2, width=None):
    need = [-(-n // page) for n in lens]
    pages = sum(need) + extra
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(lens), max(max(need, default=0), 1) if width is None else width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages


# ------------------------------------------------------------------ append
def _rotated(x, pos, freq, interleaved, scale):
    """x (heads, D) in 64 bits at one position."""
    out = x.clone()
    pairs = freq.numel()
    c, s = torch.cos(pos * freq) * scale, torch.sin(pos * freq) * scale
    i0 = torch.arange(pairs) * 2 if interleaved else torch.arange(pairs)
    i1 = i0 + 1 if interleaved else i0 + pairs
    out[:, i0] = x[:, i0] * c - x[:, i1] * s
    out[:, i1] = x[:, i1] * c + x[:, i0] * s
    return out


def _append_ref(q, k, v, kc, vc, table, past, news, freq, interleaved, scale):
    B, M = k.shape[:2]
    page = kc.shape[2]
    kc, vc = kc.double(), vc.double()
    qo = torch.zeros(q.shape, dtype=torch.float64) if q is not None else None
    ko = torch.zeros(k.shape, dtype=torch.float64)
    for b in range(B):
        for m in range(min(M, news[b])):
            pos = past[b] + m
            if q is not None:
                qo[b, m] = _rotated(q[b, m].double(), pos, freq, interleaved, scale)
            ko[b, m] = _rotated(k[b, m].double(), pos, freq, interleaved, scale)
            kc[table[b, pos // page], :, pos % page] = ko[b, m]
            vc[table[b, pos // page], :, pos % page] = v[b, m].double()
    return qo, ko, kc, vc


def _check_rotation(got, ref, dtype, biggest):
    """Off by the rounding of the result, and for each product by the angle:
    its fraction of a turn is rounded to 24 bits (pi 2^-24), sine and cosine are
    good to 2 ulp (2^-22), and the products and sum round (3 2^-24)."""
    tol = HALF[dtype] * ref.abs() + 2 * biggest * (math.pi * 2.0**-24 + 2.0**-22 + 3 * 2.0**-24) * (1 + HALF[dtype])
    err = (got.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), (err - tol).max()


APPEND = [
    # B, M, heads, kv_heads, D, page, pairs, interleaved, dtype, past
    (1, 1, 32, 8, 128, 16, 64, False, BF, [700]),
    (3, 1, 4, 4, 64, 1, 32, False, FH, [0, 5, 130000]),
    (4, 9, 8, 2, 128, 16, 64, False, BF, [0, 15, 16, 1000]),
    (2, 33, 3, 1, 80, 12, 16, True, F32, [7, 100001]),
    (2, 5, 2, 2, 96, 5, 12, False, BF, [3, 0]),     # halves that fill no 16-byte chunk
    (2, 5, 2, 1, 72, 8, 10, True, FH, [3, 90]),     # pairs that end inside a chunk; an odd number of chunks
    (2, 4, 6, 3, 256, 64, 128, False, F32, [60, 8000]),
    (1, 6, 1, 1, 8, 3, 4, False, BF, [2]),
    (3, 7, 2, 1, 40, 7, 0, False, FH, [0, 6, 50]),  # no rotation
    (2, 1400, 2, 1, 64, 16, 32, False, BF, [0, 3]),  # more tokens than one a CTA covers
]


@pytest.mark.parametrize("B,M,H,KV,D,page,pairs,inter,dtype,past", APPEND)
def test_append_matches_64_bits(cuda_status_clean, B, M, H, KV, D, page, pairs, inter, dtype, past):
    g = _gen(B * 1000 + D)
    news = [[M, max(M - 1, 0), 0, M + 5][(b + (M > 1)) % 4] if B > 1 else M for b in range(B)]
    table, pages = _table([p + min(n, M) for p, n in zip(past, news)], page, g)
    q, k, v = (torch.randn(B, M, h, D, generator=g).to(dtype) for h in (H, KV, KV))
    kc, vc = (torch.randn(pages, KV, page, D, generator=g).to(dtype) for _ in range(2))
    freq = (500000.0 ** -(torch.arange(pairs) / max(pairs, 1))).float()
    dev = _dev()
    kd, vd = kc.to(dev), vc.to(dev)
    scale = 1.0 if pairs != 64 else 1.25
    qo, ko = paged_append(q.to(dev), k.to(dev), v.to(dev), kd, vd, table.to(dev), torch.tensor(past, device=dev),
                          torch.tensor(news, dtype=torch.int32, device=dev),
                          phases=rotary_phases(freq.to(dev)) if pairs else None, interleaved=inter,
                          rotary_scale=scale, return_keys=True)
    rq, rk, rkc, rvc = _append_ref(q, k, v, kc, vc, table, past, news, freq.double(), inter,
                                   scale if pairs else 1.0)
    big = float(max(q.abs().max(), k.abs().max())) * scale
    _check_rotation(qo, rq, dtype, big)
    _check_rotation(ko, rk, dtype, big)
    _check_rotation(kd, rkc, dtype, big)
    assert torch.equal(vd.double().cpu(), rvc)  # values are copies
    touched = torch.zeros(kc.shape[:3], dtype=torch.bool)
    for b in range(B):
        for m in range(min(M, news[b])):
            touched[table[b, (past[b] + m) // page], :, (past[b] + m) % page] = True
    assert torch.equal(kd.cpu()[~touched], kc[~touched])  # bit for bit as they were
    for b in range(B):
        assert not qo[b, min(M, news[b]):].any() and not ko[b, min(M, news[b]):].any()
    # nothing asked for the queries: the cache gets the same bits
    k2, v2 = kc.to(dev), vc.to(dev)
    none = paged_append(None, k.to(dev), v.to(dev), k2, v2, table.to(dev), torch.tensor(past, device=dev),
                        torch.tensor(news, dtype=torch.int32, device=dev),
                        phases=rotary_phases(freq.to(dev)) if pairs else None, interleaved=inter, rotary_scale=scale)
    assert none == (None, None) and torch.equal(k2, kd) and torch.equal(v2, vd)


def test_append_strides_and_alignment(cuda_status_clean):
    """Heads sliced from a fused projection, rows in another order, tensors at
    odd addresses, caches whose pages lie apart, a page table with wide rows."""
    g, dev = _gen(5), _dev()
    B, M, H, KV, D, page = 3, 4, 4, 2, 64, 8
    fused = torch.randn(B, M, (H + 2 * KV) * D, generator=g).to(BF).to(dev)
    q, k, v = (t.view(B, M, -1, D) for t in fused.split([H * D, KV * D, KV * D], dim=-1))
    table, pages = _table([20, 21, 22], page, g)
    past, freq = torch.tensor([16, 17, 18], dtype=torch.int32, device=dev), torch.rand(32, generator=g).to(dev)
    ph = rotary_phases(freq)
    pool = torch.zeros(pages, 2, KV, page, D, dtype=BF, device=dev)
    wide = torch.full((3, 9), -7, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    out, _ = paged_append(q, k, v, pool[:, 0], pool[:, 1], wide.to(dev)[:, :3], past, phases=ph)
    kc, vc = torch.zeros(pages, KV, page, D, dtype=BF, device=dev), torch.zeros(pages, KV, page, D, dtype=BF, device=dev)
    want, _ = paged_append(q.contiguous(), k.contiguous(), v.contiguous(), kc, vc, table.to(dev), past, phases=ph)
    assert torch.equal(out, want) and torch.equal(pool[:, 0], kc) and torch.equal(pool[:, 1], vc)
    # tokens outermost, and an address that is no multiple of 16 bytes
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.empty(k.numel() + 1, dtype=BF, device=dev)[1:].view(k.shape).copy_(k)
    kc2, vc2 = torch.zeros_like(kc), torch.zeros_like(vc)
    got, _ = paged_append(qt, odd, v.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3), kc2, vc2, table.to(dev), past,
                          phases=ph)
    assert torch.equal(got, want) and torch.equal(kc2, kc) and torch.equal(vc2, vc)
    # one key for all heads, by a stride of 0
    one = k[:, :, :1].expand(B, M, KV, D)
    kc3, kc4 = torch.zeros_like(kc), torch.zeros_like(kc)
    paged_append(None, one, v, kc3, vc2, table.to(dev), past, phases=ph)
    paged_append(None, one.contiguous(), v, kc4, vc2, table.to(dev), past, phases=ph)
    assert torch.equal(kc3, kc4)


def test_append_without_a_page_raises_status(native):
    """Positions past the table, page ids outside the cache and negative
    lengths: those tokens are skipped, the others written."""
    g, dev = _gen(6), _dev()
    B, M, KV, D, page = 4, 2, 1, 16, 4
    k = torch.randn(B, M, KV, D, generator=g).to(BF).to(dev)
    kc, vc = torch.zeros(3, KV, page, D, dtype=BF, device=dev), torch.zeros(3, KV, page, D, dtype=BF, device=dev)
    table = torch.tensor([[0, 1], [2, -1], [3, 2], [1, 1]], dtype=torch.int32, device=dev)
    past = torch.tensor([7, 3, 0, -2], dtype=torch.int32, device=dev)  # position 8; page -1; page 3; negative
    native.device_status(clear=True)
    paged_append(None, k, k, kc, vc, table, past)
    assert native.device_status(clear=True) == _native.DEV_PAGE_RANGE
    want = torch.zeros_like(kc)
    want[1, 0, 3] = k[0, 0, 0]
    want[2, 0, 3] = k[1, 0, 0]
    assert torch.equal(kc, want) and torch.equal(vc, want)


# ------------------------------------------------------------------ attention
def _attend_ref(q, kc, vc, table, lens, window, scale):
    B, H, D = q.shape
    KV, page = kc.shape[1:3]
    out = torch.zeros(B, H, D, dtype=torch.float64)
    slack = torch.zeros(B, H, 1, dtype=torch.float64)
    for b, n in enumerate(lens):
        pos = torch.arange(max(0, n - window) if window else 0, n)
        if n == 0:
            continue
        where, slot = table[b].long()[pos // page], pos % page
        for h in range(H):
            k, v = kc[where, h // (H // KV), slot].double(), vc[where, h // (H // KV), slot].double()
            s = k @ q[b, h].double() * scale
            out[b, h] = torch.softmax(s, 0) @ v
            # scores: D products and sums in 32 bits, and the exponential; sums over the tokens
            ds = (D + 8) * 2.0**-24 * float((k.abs() @ q[b, h].double().abs()).max()) * abs(scale) + 2.0**-21
            slack[b, h] = (2 * ds + 2 * len(pos) * 2.0**-24 + PART[q.dtype]) * float(v.abs().max())
    return out, slack


# The products with the values take probabilities as a 16-bit number and a
# 16-bit remainder: 2^-9 2^-9 for bf16, 2^-12 2^-12 for fp16 (below its normal
# range 2^-25 of the largest, which the term of the sums covers).
PART = {BF: 2.0**-17, FH: 2.0**-22, F32: 0.0}

ATTEND = [
    # lens, heads, kv_heads, D, page, dtype, window
    ([1], 1, 1, 64, 16, BF, 0),
    ([200], 32, 8, 128, 16, BF, 0),
    ([0, 1, 15, 16, 17, 300, 0], 8, 2, 128, 16, BF, 0),
    ([0, 0], 4, 4, 64, 16, FH, 0),
    ([1000, 3, 77], 4, 4, 64, 1, FH, 0),
    ([129, 250], 14, 2, 96, 12, BF, 0),        # a group of seven
    ([40, 513], 16, 1, 256, 32, FH, 0),        # one shared head
    ([333], 20, 1, 80, 5, BF, 0),              # more query heads than a block
    ([100, 64], 40, 1, 64, 16, BF, 0),
    ([90, 41], 33, 1, 128, 16, FH, 0),
    ([90, 41, 7], 48, 1, 256, 16, BF, 0),
    ([5000], 4, 1, 128, 64, BF, 0),            # one item over many shares
    ([700, 64, 65, 1, 0], 4, 2, 128, 16, BF, 64),
    ([100, 33], 2, 2, 72, 7, FH, 1),
    ([100, 33], 2, 2, 72, 7, FH, 1000),
    ([700, 2, 0, 31], 15, 5, 80, 12, F32, 0),
    ([65, 400], 9, 1, 128, 16, F32, 0),
    ([65, 130], 3, 3, 256, 16, F32, 100),
    ([513], 4, 2, 8, 3, F32, 0),
    ([513, 20], 4, 2, 8, 3, BF, 0),
    ([31] * 300, 2, 1, 64, 16, BF, 0),         # more rows than threads of a CTA
    (list(range(700)), 4, 2, 32, 8, FH, 0),
    # few short rows: clusters of one to eight CTAs, warps without a tile, empty rows
    ([17], 4, 2, 128, 16, BF, 0),
    ([130, 0, 129], 4, 1, 128, 16, FH, 0),
    ([2000, 1, 900], 8, 2, 64, 16, BF, 0),
    ([1500, 0, 333, 12], 16, 1, 256, 16, BF, 0),
    ([1500, 200], 24, 1, 128, 8, BF, 0),
    ([600, 31], 3, 1, 128, 16, F32, 0),
    ([300, 0], 2, 1, 256, 16, F32, 0),
    ([600, 31, 5], 8, 1, 64, 4, F32, 50),
    ([40000, 20000], 4, 2, 64, 16, FH, 0),   # long rows: segments asked for
    ([50000, 33], 2, 1, 128, 16, F32, 0),
]


@pytest.mark.parametrize("lens,H,KV,D,page,dtype,window", ATTEND)
def test_attention_matches_64_bits(cuda_status_clean, lens, H, KV, D, page, dtype, window):
    g = _gen(len(lens) * 100 + H + D)
    B = len(lens)
    table, pages = _table(lens, page, g)
    q = (torch.randn(B, H, D, generator=g) * 2).to(dtype)
    kc, vc = (torch.randn(pages, KV, page, D, generator=g).to(dtype) for _ in range(2))
    ref, slack = _attend_ref(q, kc, vc, table, lens, window, D**-0.5)
    # places that no token fills hold NaN and infinities
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        pos = torch.arange(max(0, n - window) if window else 0, n)
        used[table[b].long()[pos // page], pos % page] = True
    free = (~used)[:, None, :, None].expand(kc.shape)
    kc[free], vc[free] = math.nan, math.inf
    dev = _dev()
    args = [t.to(dev) for t in (q, kc, vc, table, torch.tensor(lens, dtype=torch.int32))]
    got = paged_attention(*args, window=window)
    err = (got.double().cpu() - ref).abs()
    tol = HALF[dtype] * ref.abs() + slack * (1 + HALF[dtype])
    assert bool((err <= tol).all()), float((err - tol).max())
    for b, n in enumerate(lens):
        if n == 0:
            assert not got[b].any()
    assert torch.equal(paged_attention(*args, window=window), got)  # the same bits again


def test_attention_large_scores_and_masked_lowest(cuda_status_clean):
    """Scores of +-10^4, one-hot softmaxes, equal scores: no overflow, no NaN."""
    dev, D = _dev(), 64
    k = torch.zeros(4, 1, 16, D)
    k[..., 0] = torch.linspace(-1, 1, 64).view(4, 1, 16)
    v = torch.arange(64.0).view(4, 1, 16, 1).expand(4, 1, 16, D).contiguous()
    table = torch.arange(4, dtype=torch.int32).view(1, 4)
    q = torch.zeros(1, 3, D)
    q[0, 0, 0], q[0, 1, 0] = 1e4, -1e4
    for dtype in (BF, FH, F32):
        got = paged_attention(*(t.to(dev, dtype) for t in (q, k, v)), table.to(dev),
                              torch.tensor([64], dtype=torch.int32, device=dev), scale=1.0).float().cpu()
        assert torch.equal(got[0, 0], torch.full((D,), 63.0)) and torch.equal(got[0, 1], torch.zeros(D))
        assert torch.allclose(got[0, 2], torch.full((D,), 31.5), rtol=HALF[dtype] * 1.01 + 64 * 2.0**-24 + PART[dtype])


def test_attention_strides_shared_pages_and_out(cuda_status_clean):
    g, dev = _gen(9), _dev()
    H, KV, D, page = 8, 2, 64, 16
    pool = torch.randn(6, 2, KV, page, D, generator=g).to(BF).to(dev)
    table = torch.tensor([[4, 0, 9], [4, 0, 9], [5, 2, 9]], dtype=torch.int32, device=dev)  # a prefix of two rows
    lens = torch.tensor([20, 32, 17], device=dev)
    fused = torch.randn(3, 3, H * D, generator=g).to(BF).to(dev)
    q = fused[:, 1].view(3, H, D)
    want = paged_attention(q.contiguous(), pool[:, 0].contiguous(), pool[:, 1].contiguous(), table[:, :2].contiguous(), lens)
    out = torch.full((3, H, D), 7.0, dtype=BF, device=dev)
    got = paged_attention(q, pool[:, 0], pool[:, 1], table[:, :2], lens, out=out)
    assert got is out and torch.equal(out, want)
    flip = torch.arange(H - 1, -1, -1, device=dev)  # heads in another order are another call's heads
    odd = torch.empty(q.numel() + 3, dtype=BF, device=dev)[3:].view(q.shape).copy_(q)
    assert torch.equal(paged_attention(odd, pool[:, 0], pool[:, 1], table[:, :2], lens), want)
    assert not torch.equal(paged_attention(q[:, flip], pool[:, 0], pool[:, 1], table[:, :2], lens), want)


def test_attention_bad_page_and_length(native):
    """A page outside the cache reads as zeros and raises the status; lengths
    beyond the table are clamped, negative ones empty."""
    g, dev = _gen(10), _dev()
    kc, vc = (torch.randn(3, 1, 4, 16, generator=g).to(dev) for _ in range(2))
    q = torch.randn(3, 2, 16, generator=g).to(dev)
    table = torch.tensor([[0, 7], [1, 2], [0, 1]], dtype=torch.int32, device=dev)
    native.device_status(clear=True)
    got = paged_attention(q, kc, vc, table, torch.tensor([6, 100, -3], dtype=torch.int32, device=dev))
    assert native.device_status(clear=True) == _native.DEV_PAGE_RANGE
    padded_k, padded_v = torch.cat([kc, torch.zeros_like(kc[:1])]), torch.cat([vc, torch.zeros_like(vc[:1])])
    table[0, 1] = 3
    want = paged_attention(q, padded_k, padded_v, table, torch.tensor([6, 8, 0], dtype=torch.int32, device=dev))
    assert native.device_status(clear=True) == 0
    assert torch.equal(got, want) and not got[2].any()


def test_attention_past_32_bit_offsets(cuda_status_clean):
    """Pages whose elements lie beyond 2^31 (and 2^32 bytes) from the cache's start."""
    g, dev = _gen(11), _dev()
    KV, page, D, pages = 8, 64, 128, 33000  # 2.16e9 elements
    kc = torch.zeros(pages, KV, page, D, dtype=BF, device=dev)
    vc = torch.zeros(pages, KV, page, D, dtype=BF, device=dev)
    table = torch.tensor([[32999, 3, 32990]], dtype=torch.int32, device=dev)
    k, v, q = (torch.randn(1, 130, KV, D, generator=g).to(BF).to(dev) for _ in range(3))
    past = torch.zeros(1, dtype=torch.int32, device=dev)
    ph = rotary_phases(torch.rand(64, generator=g).to(dev))
    paged_append(q, k, v, kc, vc, table, past, phases=ph)
    sk, sv = torch.zeros(4, KV, page, D, dtype=BF, device=dev), torch.zeros(4, KV, page, D, dtype=BF, device=dev)
    small = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=dev)
    paged_append(q, k, v, sk, sv, small, past, phases=ph)
    assert torch.equal(kc[table[0].long()], sk[small[0].long()]) and torch.equal(vc[table[0].long()], sv[small[0].long()])
    lens = torch.tensor([130], dtype=torch.int32, device=dev)
    assert torch.equal(paged_attention(q[:, 0], kc, vc, table, lens), paged_attention(q[:, 0], sk, sv, small, lens))


@pytest.mark.parametrize("longest,width", [(3000, 256), (60000, 4096)])
def test_two_streams_and_two_graphs(cuda_status_clean, longest, width):
    """Calls on two streams at once, and two graphs captured one after the
    other and replayed at once with new lengths, give the single calls' bits;
    short rows (one launch) and long ones (a list of segments)."""
    g, dev = _gen(12), _dev()
    H, KV, D, page = 16, 4, 128, 16
    sets = []
    for n in (longest, longest - 500):
        lens = [n, 17, n // 2]
        table, pages = _table(lens, page, g, width=width)
        sets.append([torch.randn(3, H, D, generator=g).to(BF).to(dev)]
                    + [torch.randn(pages, KV, page, D, generator=g).to(BF).to(dev) for _ in range(2)]
                    + [table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)])
    want = [paged_attention(*s).clone() for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, (st, s) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(st):
                got[i] = paged_attention(*s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for s in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(paged_attention(*s))
        graphs.append(gr)
    new = [s[4] // 2 + 1 for s in sets]
    want2 = [paged_attention(*s[:4], n) for s, n in zip(sets, new)]
    for s, n in zip(sets, new):
        s[4].copy_(n)
    torch.cuda.synchronize()
    for _ in range(3):
        for st, gr in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want2))


def test_empty_calls(cuda_status_clean):
    dev = _dev()
    kc = torch.zeros(1, 2, 4, 16, device=dev)
    none = torch.zeros(0, 1, dtype=torch.int32, device=dev)
    assert paged_attention(torch.zeros(0, 4, 16, device=dev), kc, kc, none, torch.zeros(0, device=dev)).shape == (0, 4, 16)
    q, k = paged_append(torch.zeros(2, 0, 4, 16, device=dev), torch.zeros(2, 0, 2, 16, device=dev),
                        torch.zeros(2, 0, 2, 16, device=dev), kc, kc.clone(), torch.zeros(2, 1, dtype=torch.int32, device=dev),
                        torch.zeros(2, device=dev), return_keys=True)
    assert q.shape == (2, 0, 4, 16) and k.shape == (2, 0, 2, 16)


@pytest.mark.parametrize("lens", [[900, 300], [120000, 100000]])
def test_expired_wait_is_reported_and_clears(native, lens):
    """With the wait limit at 0 the attention's waits for its copies may run
    out: the call returns, the status says so, and the next call is whole.
    Copies of a small cache may all be there at the first look; the large one
    (225 MB, beyond the L2) has each warp wait some twenty times."""
    g, dev = _gen(13), _dev()
    table, pages = _table(lens, 16, g)
    args = [torch.randn(2, 8, 128, generator=g).to(BF).to(dev),
            *(torch.randn(pages, 2, 16, 128, generator=g).to(BF).to(dev) for _ in range(2)), table.to(dev),
            torch.tensor(lens, dtype=torch.int32, device=dev)]
    want = paged_attention(*args)
    native.device_status(clear=True)
    prev = native.set_wait_limit_ns(0)
    try:
        paged_attention(*args)
        status = native.device_status(clear=True)
    finally:
        native.set_wait_limit_ns(prev)
    assert status in ((0, _native.DEV_WAIT_TIMEOUT) if lens[0] < 1000 else (_native.DEV_WAIT_TIMEOUT,))
    assert torch.equal(paged_attention(*args), want)
    assert native.device_status(clear=True) == 0


def test_shared_prefix_of_many_rows_and_a_window_of_any_size(cuda_status_clean):
    """Rows that read the same pages, and windows beyond the tokens up to the
    largest number, agree with the plain call."""
    g, dev = _gen(14), _dev()
    kc, vc = (torch.randn(20, 2, 16, 64, generator=g).to(BF).to(dev) for _ in range(2))
    table = torch.arange(20, dtype=torch.int32, device=dev).view(1, 20).expand(300, 20).contiguous()
    lens = torch.arange(300, dtype=torch.int32, device=dev)
    q = torch.randn(1, 4, 64, generator=g).to(BF).to(dev).expand(300, 4, 64)
    want = paged_attention(q, kc, vc, table, lens)
    assert torch.equal(paged_attention(q, kc, vc, table, lens, window=2**63 - 1), want)
    one = paged_attention(q[250:251], kc, vc, table[:1], lens[250:251])
    assert torch.allclose(one.float(), want[250:251].float(), atol=2 * HALF[BF], rtol=2 * HALF[BF])
    assert torch.equal(paged_attention(q, kc, vc, table, lens, out=torch.empty_like(want)), want)


def test_queries_may_be_overwritten(cuda_status_clean):
    g, dev = _gen(15), _dev()
    for lens, width in (([70, 3], 8), ([30000, 20000], 2000)):
        table, pages = _table(lens, 16, g, width=width)
        q = torch.randn(2, 8, 128, generator=g).to(BF).to(dev)
        kc, vc = (torch.randn(pages, 2, 16, 128, generator=g).to(BF).to(dev) for _ in range(2))
        n = torch.tensor(lens, dtype=torch.int32, device=dev)
        want = paged_attention(q, kc, vc, table.to(dev), n)
        assert torch.equal(paged_attention(q, kc, vc, table.to(dev), n, out=q), want) and torch.equal(q, want)
