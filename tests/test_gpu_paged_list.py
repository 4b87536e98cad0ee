"""Paged attention over calls large enough that warps ask for segments of the
list of tiles, against 64 bits."""

import math

import pytest
import torch

from polylora_b200 import _native
from polylora_b200.paged import paged_attention
from polylora_b200.sgmv import dtype_code

BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32
TILE = 16


def _inputs(seed, lens, H, KV, D, page, dtype, device, pool=300):
    """Rows that read the pages of one small pool in orders of their own; the
    page a row ends on is its own, with NaN and infinities past its end."""
    g = torch.Generator().manual_seed(seed)
    width = max(-(-max(lens) // page), 1)
    table = torch.randint(0, pool, (len(lens), width), generator=g, dtype=torch.int32)
    kc, vc = (torch.randn(pool + len(lens), KV, page, D, generator=g).to(dtype) for _ in range(2))
    for b, n in enumerate(lens):
        last = -(-n // page)
        if last:
            table[b, last - 1] = pool + b
            kc[pool + b, :, n - (last - 1) * page:] = math.nan
            vc[pool + b, :, n - (last - 1) * page:] = math.inf
        table[b, last:] = -1
    q = (torch.randn(len(lens), H, D, generator=g) * 2).to(dtype)
    return [t.to(device) for t in (q, kc, vc, table, torch.tensor(lens, dtype=torch.int32))]


def _reference(q, kc, vc, table, lens, window, scale, drop=None):
    """Outputs in 64 bits, sum_j p_j |v_j|, and per head the largest |score| and
    sum |q||k|.  ``drop``: tokens (first, count) left out of every row."""
    B, H, D = q.shape
    KV, page = kc.shape[1:3]
    out, mean = (torch.zeros(B, H, D, dtype=torch.float64, device=q.device) for _ in range(2))
    top, span = (torch.zeros(B, H, 1, dtype=torch.float64, device=q.device) for _ in range(2))
    for b, n in enumerate(lens.tolist()):
        pos = torch.arange(max(0, n - window) if window else 0, n, device=q.device)
        if drop is not None:
            pos = pos[(pos < drop[0]) | (pos >= drop[0] + drop[1])]
        if len(pos) == 0:
            continue
        where, slot = table[b].long()[pos // page], pos % page
        for kv in range(KV):
            hs = slice(kv * (H // KV), (kv + 1) * (H // KV))
            k, v = kc[where, kv, slot].double(), vc[where, kv, slot].double()
            s = q[b, hs].double() @ k.t() * scale
            p = torch.softmax(s, 1)
            out[b, hs], mean[b, hs] = p @ v, p @ v.abs()
            top[b, hs, 0] = s.abs().amax(1)
            span[b, hs, 0] = (q[b, hs].double().abs() @ k.abs().t()).amax(1) * abs(scale)
    return out, mean, top, span


def _bound(ref, mean, top, span, dtype, dim, chain, parts, tokens):
    """How far an output may be off.  Scores: chains of dim / 32 tensor-core sums of
    17 terms, cut at 2^-23 of the largest each (CUDA cores: dim / 4 roundings); the
    factor and the difference from the maximum, 2^-24 each of scores up to twice the
    largest; the exponential, 2^-21.  An error
    e of all scores moves the output by 2 e of the mean of |v| at most.  Sums, of
    values and of probabilities: a tile is at most 16 additions and a scaling, 2^-24
    each, over a chain of tiles; a part is a product, an addition and a scaling, up
    to 32 of them in turn, or 32 runs of them and ten more.  Probabilities as two
    16-bit numbers (see the kernel)."""
    half = torch.finfo(dtype).eps / 2
    score = (dim / 32 * 17 + 8) * 2.0**-23 * span + 4 * 2.0**-24 * top + 2.0**-21
    sums = 2 * (17 * chain + 3 * (min(parts, 32) + parts / 32 + 10)) * 2.0**-24
    pair = {BF: 2.0**-18, FH: 2.0**-22, F32: 0.0}[dtype]
    slack = (2 * score + sums + pair) * mean
    if dtype is FH:  # below its smallest numbers half a step, 2^-40 of the largest probability, of |v| below 8
        slack = slack + tokens * 2.0**-40 * 8
    return half * ref.abs() + (1 + half) * slack + (torch.finfo(dtype).smallest_normal * half if dtype is FH else 0)


def _list(rows, H, KV, D, page, width, window, dtype):
    """(warps that segments are dealt to, query heads of a block), from the
    workspace: segments and two parts of each."""
    size = _native.load().plora_paged_attention_workspace(rows, H, KV, D, page, width, window, dtype_code(dtype))
    assert size > 0  # a call by the list
    group = H // KV
    most = 8 if dtype is F32 else (16 if D > 128 else 32)
    blocks = -(-group // most)
    heads = -(-group // blocks)
    more = 4 if heads <= 4 else (2 if heads <= 8 else 1)
    warps = int((size - 256 - rows * 8) / ((1 + more) * (16 + 2 * heads * (8 + 4 * D))))
    assert warps % 148 == 0, warps
    return warps, -(-group // heads)


def _tiles(lens, window):
    return [max(1, -(-n // TILE) - (max(0, n - window) // TILE if window else 0)) for n in lens]


def _ragged(rows, longest):
    """Rows of up to `longest` tokens, in no order, empty and single ones among them."""
    lens = [(longest * ((i * 101) % rows + 1)) // rows - (i % 3) for i in range(rows)]
    lens[1], lens[rows // 2], lens[-1] = 0, 1, 0
    return lens


LISTS = [
    # lens, heads, kv_heads, D, page, dtype, window
    (_ragged(64, 10500), 8, 2, 128, 16, BF, 0),      # copies by TMA
    ([310000], 8, 2, 128, 64, FH, 0),                # two items, each of hundreds of parts
    (_ragged(41, 16000), 6, 2, 128, 12, FH, 0),      # copies a lane, pages that end inside a tile
    (_ragged(40, 17000), 4, 2, 80, 5, BF, 0),        # heads padded to 128
    (_ragged(55, 12500), 8, 4, 64, 16, BF, 0),       # sixteen warps
    (_ragged(42, 12500), 16, 2, 256, 32, FH, 0),     # heads of 256, a block of eight
    (_ragged(37, 23500), 16, 1, 256, 32, BF, 0),     # and of sixteen heads
    (_ragged(38, 19000), 24, 2, 64, 16, BF, 0),      # twelve heads of 64
    (_ragged(37, 27500), 20, 1, 128, 16, BF, 0),     # a block of twenty
    (_ragged(37, 14500), 40, 1, 128, 16, BF, 0),     # and two of them
    (_ragged(150, 15000), 8, 2, 128, 16, BF, 2500),  # a window
    (_ragged(44, 11500), 6, 2, 128, 16, F32, 0),     # CUDA cores
    (_ragged(25, 14500), 18, 2, 64, 8, F32, 1 << 40),  # two blocks of five and four heads
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,H,KV,D,page,dtype,window", LISTS)
def test_asked_for_segments_match_64_bits(cuda_status_clean, lens, H, KV, D, page, dtype, window):
    dev = torch.device("cuda")
    args = _inputs(len(lens) + H + D, lens, H, KV, D, page, dtype, dev)
    warps, blocks = _list(len(lens), H, KV, D, page, args[3].shape[1], window, dtype)
    tiles = _tiles(lens, window)
    total = sum(tiles) * KV * blocks
    assert total >= 32 * warps, (total, 32 * warps)  # else all of them are dealt
    got = paged_attention(*args, window=window)
    ref, mean, top, span = _reference(*args, window, D**-0.5)
    # segments of 13/16 of an equal share at most, parts of eight tiles at least
    tol = _bound(ref, mean, top, span, dtype, D, total // warps + 1, max(tiles) // 8 + 2, max(lens))
    err = (got.double() - ref).abs()
    assert bool((err <= tol).all()), float((err / tol.clamp_min(1e-30)).max())
    for b, n in enumerate(lens):
        if n == 0:
            assert not got[b].any()
    assert torch.equal(paged_attention(*args, window=window), got)  # the same bits, whoever takes a segment


@pytest.mark.gpu
def test_asked_for_segments_on_two_streams_and_replayed(cuda_status_clean):
    dev, lens = torch.device("cuda"), _ragged(64, 10500)
    sets = [_inputs(s, lens[s:] + lens[:s], 8, 2, 128, 16, BF, dev) for s in (1, 2)]
    want = [paged_attention(*s).clone() for s in sets]
    streams, got = [torch.cuda.Stream() for _ in sets], [None, None]
    torch.cuda.synchronize()
    for _ in range(3):
        for i, (st, s) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(st):
                got[i] = paged_attention(*s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(paged_attention(*s))
    for s in sets:  # fewer tokens: all segments dealt, then as many as before
        s[4].copy_(s[4] // 2)
    half = [paged_attention(*s) for s in sets]
    torch.cuda.synchronize()
    for want_now in (half, want):
        for st, gr in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want_now))
        for s, n in zip(sets, (lens[1:] + lens[:1], lens[2:] + lens[:2])):
            s[4].copy_(torch.tensor(n, dtype=torch.int32))
        torch.cuda.synchronize()


def test_the_bound_sees_a_lost_tile():
    """A tile left out of the reference (of a row's 600) is off by more than the
    bound at many places, a short segment of eight nearly everywhere."""
    args = _inputs(3, [9600], 8, 2, 128, 16, BF, "cpu")
    whole = _reference(*args, 0, 128**-0.5)
    tol = _bound(*whole, BF, 128, 40, 30, 9600)
    for tiles, share in ((1, 0.3), (8, 0.8)):
        lost = _reference(*args, 0, 128**-0.5, drop=(16 * 200, 16 * tiles))[0]
        assert float(((lost - whole[0]).abs() > tol).double().mean()) > share
