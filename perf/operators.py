"""Measured cases of the decode-step operators: appending rotated keys and
values to a paged cache, attention of one new token over that cache, and the
per-row rules (penalties, biases, masks) on its logits.

``run`` computes them in elementary torch operations while ``own`` is false,
and through the framework's entry points while it is true; ``exact`` computes
them in 64 bits from their definitions.

Sizes are the Llama-3-8B shapes of the benchmark (32 query and 8 key-value
heads of 128, 256 decode rows, 64 x 1024 prompts, positions to 8192 and
beyond, 128256 tokens of vocabulary) and generic odd ones.
"""

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one request decoding alone: the smallest call, all latency
        _append("append_one", 1, 1, 32, 8, 128, 16, "bf16", past=700),
        # the decode step of the Llama-3-8B batch: 256 rows, one new token each
        _append("append_decode", 256, 1, 32, 8, 128, 16, "bf16", past=2000),
        # a right-padded batch of prompts, whose rotated keys the prompt's own attention reads too
        _append("append_prompts", 64, 1024, 32, 8, 128, 16, "bf16", k_out=True),
        # odd sizes: partial rotation of interleaved pairs, pages that are no power of two, a chunk of a long prompt
        _append("append_odd", 5, 77, 6, 2, 80, 12, "fp32", past=100000, rotary=32, interleaved=True),
        # one request early in its answer: the smallest attention call
        _attend("attend_one_short", 1, 200, 32, 8, 128, 16, "bf16"),
        # one request with a long document: work split over the length only
        _attend("attend_one_long", 1, 131072, 32, 8, 128, 64, "fp16"),
        # the decode batch with ragged histories up to the model's 8192 positions
        _attend("attend_decode", 256, 4096, 32, 8, 128, 16, "bf16"),
        # one shared head of 256, a sliding window, rows that have no history yet
        _attend("attend_window", 48, 9000, 16, 1, 256, 32, "bf16", window=1024),
        # 32-bit cache of odd head sizes: a small model held in full precision
        _attend("attend_odd", 7, 1500, 15, 5, 80, 12, "fp32"),
        # one row's rules: short history, a grammar's mask
        _rules("rules_one", 1, 128256, 300, 8, True, "bf16"),
        # the decode batch: every row with its own history, biases and mask
        _rules("rules_decode", 256, 128256, 4096, 64, True, "bf16"),
        # a vocabulary of odd size (rows that start at any alignment), 32-bit logits, no masks
        _rules("rules_odd", 33, 50257, 1000, 300, False, "fp32", wide=False),
    ]


def _append(name, rows, new, heads, kv_heads, dim, page, dtype, past=0, rotary=0, interleaved=False, k_out=False):
    return {"name": name, "op": "append", "rows": rows, "new": new, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "dtype": dtype, "past": past, "rotary": rotary or dim, "interleaved": interleaved,
            "k_out": k_out}


def _attend(name, rows, longest, heads, kv_heads, dim, page, dtype, window=0):
    return {"name": name, "op": "attend", "rows": rows, "longest": longest, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "dtype": dtype, "window": window}


def _rules(name, rows, vocab, history, biases, mask, dtype, wide=True):
    return {"name": name, "op": "rules", "rows": rows, "vocab": vocab, "history": history, "biases": biases,
            "mask": mask, "dtype": dtype, "wide": wide}


def draw(rng):
    def spread(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["append", "attend", "attend", "rules"])
    rows = spread(1, 256)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    page = rng.choice([1, 8, 12, 16, 16, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 7, 8, 16])
    if op == "append":
        most = 6.0e8 / ((2 * heads + 4 * kv_heads) * dim * _BYTES[dtype])
        new = rng.choice([1, spread(1, 1024)])
        new = max(1, min(new, int(most / rows)))
        far = 1.0e9 / (rows * 2 * kv_heads * dim * _BYTES[dtype])  # the cache of the tokens before fits beside the rest
        past = min(spread(1, 130000), max(1, int(far))) if rng.random() < 0.7 else 0
        case = _append("", rows, new, heads, kv_heads, dim, page, dtype, past=past,
                       rotary=rng.choice([dim, dim, dim // 2]), interleaved=rng.random() < 0.3, k_out=rng.random() < 0.3)
    elif op == "attend":
        most = 1.2e9 / (2 * rows * kv_heads * dim * _BYTES[dtype])
        longest = max(1, min(spread(1, 131072), int(most)))
        case = _attend("", rows, longest, heads, kv_heads, dim, page, dtype,
                       window=rng.choice([0, 0, spread(1, longest)]))
    else:
        case = _rules("", rows, spread(500, 200000), spread(1, 8192) - 1, spread(1, 301) - 1, rng.random() < 0.5, dtype,
                      wide=rng.random() < 0.5)
    del case["name"]
    return case


def _spread_lengths(rows, longest, zeros):
    """Lengths of a ragged batch, the same multiset for every seed: a few rows
    without any, the others evenly spread up to the longest."""
    none = rows // 16 if zeros else 0
    some = rows - none
    return [0] * none + [max(1, (longest * (i + 1)) // some) for i in range(some)]


def _new_lengths(c):
    """Valid new tokens of each row of a right-padded batch: a half to all of its width."""
    return [max(1, c["new"] - (i * (c["new"] // 2)) // max(c["rows"] - 1, 1)) for i in range(c["rows"])]


def _seen(c):
    """Tokens that each row of an attention case attends to."""
    lens = _spread_lengths(c["rows"], c["longest"], True)
    return [min(n, c["window"]) if c["window"] else n for n in lens]


def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] == "append":
        rows, dim, heads, kv = case["rows"], case["dim"], case["heads"], case["kv_heads"]
        valid = sum(_new_lengths(case))
        read = valid * (heads + 2 * kv) * dim * e
        wrote = rows * case["new"] * heads * dim * e + valid * 2 * kv * dim * e
        wrote += rows * case["new"] * kv * dim * e if case["k_out"] else 0
        return {"bytes": read + wrote + rows * 8 + valid * 4 // case["page"],
                "flops": valid * (heads + kv) * case["rotary"] * 3}
    if case["op"] == "attend":
        seen = sum(_seen(case))
        ends = 2 * case["rows"] * case["heads"] * case["dim"] * e
        return {"bytes": seen * 2 * case["kv_heads"] * case["dim"] * e + ends + seen * 4 // case["page"] + case["rows"] * 4,
                "flops": seen * case["heads"] * case["dim"] * 4}
    rows, vocab = case["rows"], case["vocab"]
    lists = sum(_spread_lengths(rows, case["history"], False)) if case["history"] else 0
    return {"bytes": 2 * rows * vocab * e + (rows * ((vocab + 31) // 32) * 4 if case["mask"] else 0)
            + lists * (8 if case["wide"] else 4) + rows * case["biases"] * 8, "flops": rows * vocab * 4}


# ------------------------------------------------------------------ the inputs
def _generators(seed):
    host, dev = torch.Generator(), torch.Generator(device="cuda")
    host.manual_seed(seed)
    dev.manual_seed(seed)
    return host, dev


def _normal(shape, dtype, gen):
    return torch.randn(shape, device="cuda", dtype=torch.float32 if dtype == torch.float32 else dtype, generator=gen)


def _shuffled(values, gen):
    order = torch.randperm(len(values), generator=gen).tolist()
    return [values[i] for i in order]


def _pages(lens, page, gen):
    """A page table over pages in random order; unused entries are -1."""
    need = [-(-n // page) for n in lens]
    total = -(-sum(lens) // page) + len(lens) + 3  # the same pool for every order of the rows
    order = torch.randperm(total, generator=gen)
    table = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].to(torch.int32)
        at += n
    return table.cuda(), total


def _frequencies(rotary):
    """The frequencies of the rotation at the Llama-3 base, in 32 bits as models keep them."""
    steps = torch.arange(0, rotary, 2, dtype=torch.float64) / rotary
    return (500000.0 ** -steps).to(torch.float32)


def prepare(case, seed):
    host, dev = _generators(seed)
    dtype = _TYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "append":
        rows, new, dim = case["rows"], case["new"], case["dim"]
        new_lens = _shuffled(_new_lengths(case), host)
        past = _shuffled(_spread_lengths(rows, case["past"], False), host) if case["past"] else [0] * rows
        s["table"], pages = _pages([p + n for p, n in zip(past, new_lens)], case["page"], host)
        s["q"] = _normal((rows, new, case["heads"], dim), dtype, dev)
        s["k"] = _normal((rows, new, case["kv_heads"], dim), dtype, dev)
        s["v"] = _normal((rows, new, case["kv_heads"], dim), dtype, dev)
        # pages that other tokens fill already
        s["k_cache"] = _normal((pages, case["kv_heads"], case["page"], dim), dtype, dev)
        s["v_cache"] = _normal((pages, case["kv_heads"], case["page"], dim), dtype, dev)
        s["past"] = torch.tensor(past, dtype=torch.int32).cuda()
        s["new"] = torch.tensor(new_lens, dtype=torch.int32).cuda()
        s["frequencies"] = _frequencies(case["rotary"]).cuda()
        if own:
            from polylora_b200.paged import rotary_phases

            s["phases"] = rotary_phases(s["frequencies"])  # once for a model, like its frequencies
    elif case["op"] == "attend":
        rows, dim = case["rows"], case["dim"]
        s["lens_host"] = _shuffled(_spread_lengths(rows, case["longest"], True), host)  # the page allocator's own count
        s["table"], pages = _pages(s["lens_host"], case["page"], host)
        # queries as long as those of trained heads, whose softmax has a few large terms
        s["q"] = _normal((rows, case["heads"], dim), dtype, dev) * 2
        s["k_cache"] = _normal((pages, case["kv_heads"], case["page"], dim), dtype, dev)
        s["v_cache"] = _normal((pages, case["kv_heads"], case["page"], dim), dtype, dev)
        s["lens"] = torch.tensor(s["lens_host"], dtype=torch.int32).cuda()
    else:
        rows, vocab, history = case["rows"], case["vocab"], case["history"]
        tokens = torch.int64 if case["wide"] else torch.int32
        s["logits"] = _normal((rows, vocab), dtype, dev) * 4
        lens = _shuffled(_spread_lengths(rows, history, False), host) if history else [0] * rows
        s["lens"] = torch.tensor(lens, dtype=torch.int32).cuda()
        s["prompt"] = torch.tensor([n // 3 for n in lens], dtype=torch.int32).cuda()
        # text repeats its frequent tokens: ids fall off like a power of their rank
        u = torch.rand((rows, history), device="cuda", generator=dev, dtype=torch.float64)
        s["tokens"] = (vocab ** u - 1).to(torch.int64).clamp_(0, vocab - 1).to(tokens)
        s["repetition"] = 1 + torch.rand(rows, device="cuda", generator=dev)
        s["presence"] = torch.rand(rows, device="cuda", generator=dev)
        s["frequency"] = torch.rand(rows, device="cuda", generator=dev) / 4
        s["bias_tokens"] = torch.randint(-1, vocab, (rows, case["biases"]), device="cuda", generator=dev).to(tokens)
        s["bias_values"] = torch.randn((rows, case["biases"]), device="cuda", generator=dev) * 5
        words = (vocab + 31) // 32
        s["allowed"] = torch.randint(-2**31, 2**31, (rows, words), device="cuda", generator=dev,
                                     dtype=torch.int64).to(torch.int32) if case["mask"] else None
        if own:
            from polylora_b200.logits import LogitRules

            s["rules"] = LogitRules(tokens=s["tokens"], token_lens=s["lens"], prompt_lens=s["prompt"],
                                    repetition_penalty=s["repetition"], presence_penalty=s["presence"],
                                    frequency_penalty=s["frequency"], bias_tokens=s["bias_tokens"],
                                    bias_values=s["bias_values"], allowed=s["allowed"])
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    case = s["case"]
    if case["op"] == "append":
        from polylora_b200.paged import paged_append

        q, k = paged_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["past"], s["new"],
                            phases=s["phases"], interleaved=case["interleaved"], return_keys=case["k_out"])
        return {"q": q, "k": k, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if case["op"] == "attend":
        from polylora_b200.paged import paged_attention

        return paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], window=case["window"])
    from polylora_b200.logits import apply_logit_rules

    return apply_logit_rules(s["logits"], s["rules"])


def _rotate_plain(x, cos, sin, interleaved):
    """x (rows, new, heads, dim) in 32 bits; cos and sin (rows, new, 1, pairs)."""
    pairs = cos.shape[-1]
    out = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
        out[..., 0:2 * pairs:2], out[..., 1:2 * pairs:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :pairs], x[..., pairs:2 * pairs]
        out[..., :pairs], out[..., pairs:2 * pairs] = a * cos - b * sin, b * cos + a * sin
    return out


def _run_plain(s):
    return {"append": _append_plain, "attend": _attend_plain, "rules": _rules_plain}[s["case"]["op"]](s)


def _append_plain(s):
    case, dtype = s["case"], s["q"].dtype
    rows, new = case["rows"], case["new"]
    at = s["past"].long()[:, None] + torch.arange(new, device="cuda")[None, :]
    angle = at[:, :, None].double() * s["frequencies"].double()  # far positions need 64 bits
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    live = torch.arange(new, device="cuda")[None, :] < s["new"][:, None]
    zero = torch.zeros((), device="cuda")
    q = torch.where(live[:, :, None, None], _rotate_plain(s["q"].float(), cos, sin, case["interleaved"]), zero).to(dtype)
    k = torch.where(live[:, :, None, None], _rotate_plain(s["k"].float(), cos, sin, case["interleaved"]), zero).to(dtype)
    row, col = live.nonzero(as_tuple=True)
    where = at[row, col]
    page, slot = s["table"][row, where // case["page"]].long(), where % case["page"]
    s["k_cache"][page, :, slot] = k[row, col]
    s["v_cache"][page, :, slot] = s["v"][row, col]
    return {"q": q, "k": k if case["k_out"] else None, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attend_plain(s):
    case = s["case"]
    kv, dim, page = case["kv_heads"], case["dim"], case["page"]
    group = case["heads"] // kv
    out = torch.zeros_like(s["q"])
    for b, n in enumerate(s["lens_host"]):
        if n == 0:
            continue
        first = max(0, n - case["window"]) if case["window"] else 0
        pages = s["table"][b, first // page:-(-n // page)].long()
        skip = first - first // page * page
        k = s["k_cache"][pages].transpose(0, 1).reshape(kv, -1, dim)[:, skip:skip + n - first].float()
        v = s["v_cache"][pages].transpose(0, 1).reshape(kv, -1, dim)[:, skip:skip + n - first].float()
        q = s["q"][b].view(kv, group, dim).float()
        score = torch.matmul(q, k.transpose(1, 2)) / math.sqrt(dim)
        p = torch.exp(score - score.amax(dim=-1, keepdim=True))
        out[b] = (torch.matmul(p, v) / p.sum(dim=-1, keepdim=True)).view(-1, dim).to(out.dtype)
    return out


def _rules_plain(s):
    logits, vocab = s["logits"], s["case"]["vocab"]
    x = logits.float()
    place = torch.arange(s["tokens"].shape[1], device="cuda")[None, :]
    held = place < s["lens"][:, None]
    answer = held & (place >= s["prompt"][:, None])
    ids = s["tokens"].long()
    count = torch.zeros_like(x).scatter_add_(1, ids, answer.float())
    seen = torch.zeros_like(x).scatter_add_(1, ids, held.float()) > 0
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    ids = s["bias_tokens"].long()
    good = ids >= 0
    x.scatter_add_(1, ids.clamp(min=0), s["bias_values"] * good)
    if s["allowed"] is not None:
        token = torch.arange(vocab, device="cuda")
        bit = (s["allowed"][:, token // 32] >> (token % 32)) & 1
        x = torch.where(bit == 0, torch.full((), -math.inf, device="cuda"), x)
    return x.to(logits.dtype)


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _append_exact, "attend": _attend_exact, "rules": _rules_exact}[case["op"]](case, s)


def _append_exact(case, s):
    """The rotation as a product of complex numbers, one row of the batch at a time."""
    pairs, dim, page = case["rotary"] // 2, case["dim"], case["page"]
    caches = {"k": s["k_cache"].double(), "v": s["v_cache"].double()}
    turned = {}
    for name in ("q", "k"):
        x = s[name].double()
        done = torch.zeros_like(x)
        for b in range(case["rows"]):
            n, past = int(s["new"][b]), int(s["past"][b])
            position = torch.arange(past, past + n, device="cuda", dtype=torch.float64)
            unit = torch.polar(torch.ones(1, device="cuda", dtype=torch.float64), torch.outer(position, s["frequencies"].double()))
            head = x[b, :n, :, :2 * pairs]
            if case["interleaved"]:
                z = torch.view_as_complex(head.reshape(n, -1, pairs, 2).contiguous()) * unit[:, None]
                head = torch.view_as_real(z).flatten(-2)
            else:
                z = torch.complex(head[..., :pairs], head[..., pairs:]) * unit[:, None]
                head = torch.cat([z.real, z.imag], dim=-1)
            done[b, :n] = torch.cat([head, x[b, :n, :, 2 * pairs:]], dim=-1)
        turned[name] = done
    table = s["table"].tolist()
    values = s["v"].double()
    for b in range(case["rows"]):
        past, n = int(s["past"][b]), int(s["new"][b])
        at = past
        while at < past + n:  # page by page
            stop = min(past + n, (at // page + 1) * page)
            here = slice(at % page, at % page + stop - at)
            caches["k"][table[b][at // page], :, here] = turned["k"][b, at - past:stop - past].transpose(0, 1)
            caches["v"][table[b][at // page], :, here] = values[b, at - past:stop - past].transpose(0, 1)
            at = stop
    return {"q": turned["q"], "k": turned["k"] if case["k_out"] else None, "k_cache": caches["k"], "v_cache": caches["v"]}


def _attend_exact(case, s):
    """One head of one row at a time."""
    rows, heads, kv, dim, page = (case[x] for x in ("rows", "heads", "kv_heads", "dim", "page"))
    out = torch.zeros((rows, heads, dim), device="cuda", dtype=torch.float64)
    for b in range(rows):
        n = s["lens_host"][b]
        if n == 0:
            continue
        position = torch.arange(n, device="cuda")
        if case["window"]:
            position = position[-case["window"]:]
        page_of, slot_of = s["table"][b].long()[position // page], position % page
        for g in range(kv):
            k, v = s["k_cache"][page_of, g, slot_of].double(), s["v_cache"][page_of, g, slot_of].double()
            q = s["q"][b, g * (heads // kv):(g + 1) * (heads // kv)].double()
            out[b, g * (heads // kv):(g + 1) * (heads // kv)] = torch.softmax(q @ k.t() / dim**0.5, dim=-1) @ v
    return out


def _rules_exact(case, s):
    """Row by row, touching the tokens that its lists name."""
    out = s["logits"].double()
    for b in range(case["rows"]):
        n, p = int(s["lens"][b]), int(s["prompt"][b])
        x, history = out[b], s["tokens"][b, :n].long()
        named = torch.unique(history)
        x[named] *= torch.where(x[named] > 0, 1 / s["repetition"][b].double(), s["repetition"][b].double())
        answered, times = torch.unique(history[p:], return_counts=True)
        x[answered] -= s["frequency"][b].double() * times + s["presence"][b].double()
        good = s["bias_tokens"][b] >= 0
        x.index_add_(0, s["bias_tokens"][b][good].long(), s["bias_values"][b][good].double())
        if s["allowed"] is not None:
            words = s["allowed"][b].long() & 0xFFFFFFFF
            bits = (words[:, None] >> torch.arange(32, device="cuda")) & 1
            x[bits.flatten()[:case["vocab"]] == 0] = -math.inf
    return out
