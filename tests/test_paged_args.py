"""Refusals of the paged-cache and logit operators, and the rotation phases,
on a machine without a GPU."""

import math

import pytest
import torch

from polylora_b200.logits import LogitRules, apply_logit_rules
from polylora_b200.paged import _heads, paged_append, paged_attention, rotary_phases

D = 0x1000  # stands for a device pointer; never dereferenced on the host


def _append(lib, native, **kw):
    a = dict(q=D, qs=(2048, 1024, 64), k=D, ks=(512, 256, 64), v=D, vs=(512, 256, 64), q_out=D, k_out=None, kc=D, vc=D,
             kp=4096, vp=4096, table=D, ts=4, past=D, news=None, phases=D, pairs=32, inter=0, scale=1.0, rows=2, new=2,
             heads=16, kv=4, dim=64, page=16, pages=8, width=4, dtype=native.DTYPE_BF16)
    a.update(kw)
    return lib.plora_paged_append(native.PAGED_APPEND_ARGS.pack(
        a["kc"] or 0, a["vc"] or 0, a["kp"], a["vp"], a["table"] or 0, a["ts"], a["rows"], a["heads"], a["kv"], a["dim"],
        a["page"], a["pages"], a["width"], a["dtype"], a["q"] or 0, *a["qs"], a["k"] or 0, *a["ks"], a["v"] or 0, *a["vs"],
        a["q_out"] or 0, a["k_out"] or 0, a["past"] or 0, a["news"] or 0, a["phases"] or 0, a["pairs"], a["inter"], a["new"],
        a["scale"]), None)


def _attend(lib, native, **kw):
    a = dict(q=D, qs=(1024, 64), kc=D, vc=D, kp=4096, vp=4096, table=D, ts=4, lens=D, out=D, scale=0.125, window=0,
             rows=2, heads=16, kv=4, dim=64, page=16, pages=8, width=4, dtype=native.DTYPE_BF16, ws=D, wb=1 << 30)
    a.update(kw)
    return lib.plora_paged_attention(native.PAGED_ATTENTION_ARGS.pack(
        a["kc"] or 0, a["vc"] or 0, a["kp"], a["vp"], a["table"] or 0, a["ts"], a["rows"], a["heads"], a["kv"], a["dim"],
        a["page"], a["pages"], a["width"], a["dtype"], a["q"] or 0, *a["qs"], a["lens"] or 0, a["out"] or 0, a["scale"],
        a["window"], a["ws"] or 0, a["wb"]), None)


SHARED = [
    (dict(dtype=9), "INVALID"), (dict(rows=-1), "INVALID"), (dict(kv=0), "INVALID"), (dict(heads=10), "INVALID"),
    (dict(dim=60), "UNSUPPORTED"), (dict(dim=264), "UNSUPPORTED"), (dict(page=0), "INVALID"), (dict(pages=0), "INVALID"),
    (dict(width=0), "INVALID"), (dict(rows=1 << 21), "UNSUPPORTED"), (dict(pages=1 << 32), "UNSUPPORTED"),
    (dict(width=1 << 28, ts=1 << 28), "UNSUPPORTED"), (dict(kp=4095), "INVALID"), (dict(vp=4100), "INVALID"),
    (dict(ts=3), "INVALID"), (dict(kc=D + 8), "INVALID"), (dict(kc=None), "INVALID"), (dict(table=None), "INVALID"),
    (dict(q=D + 2), "INVALID"), (dict(kv=60000, heads=60000, page=1 << 20), "UNSUPPORTED"),
    (dict(pages=1 << 30, kp=1 << 40, vp=1 << 40), "INVALID"), (dict(dtype=1 << 32), "INVALID"),
    (dict(heads=1 << 40), "UNSUPPORTED"), (dict(page=1 << 33), "UNSUPPORTED"), (dict(dim=(1 << 32) + 64), "UNSUPPORTED"),
]


@pytest.mark.parametrize("kw,status", SHARED)
@pytest.mark.parametrize("call", [_append, _attend])
def test_cache_arguments_rejected_before_cuda(native, call, kw, status):
    want = {"INVALID": native.ERR_INVALID_ARGUMENT, "UNSUPPORTED": native.ERR_UNSUPPORTED}[status]
    assert call(native.load(), native, **kw) == want, native.last_error()
    assert native.last_error()


def test_append_arguments_rejected_before_cuda(native):
    lib = native.load()
    for kw in (dict(pairs=33), dict(pairs=-1), dict(new=-1), dict(k=None), dict(v=None), dict(past=None), dict(q_out=None),
               dict(phases=None), dict(qs=(2048, 1024, 63)), dict(ks=(-512, 256, 64)), dict(vs=(512, 4, 64)),
               dict(k_out=D + 4)):
        assert _append(lib, native, **kw) == native.ERR_INVALID_ARGUMENT, kw
    assert _append(lib, native, rows=1 << 16, new=1 << 16) == native.ERR_UNSUPPORTED
    assert _append(lib, native, rows=0) == native.OK
    assert _append(lib, native, new=0) == native.OK


def test_attention_arguments_rejected_before_cuda(native):
    lib = native.load()
    for kw in (dict(heads=0), dict(window=-1), dict(q=None), dict(lens=None), dict(out=None), dict(out=D + 8),
               dict(qs=(1024, 4)), dict(ws=D + 16)):
        assert _attend(lib, native, **kw) == native.ERR_INVALID_ARGUMENT, kw
    assert lib.plora_paged_attention_workspace(2, 16, 4, 64, 16, 4, 0, native.DTYPE_BF16) == 0  # 64 tokens
    need = lib.plora_paged_attention_workspace(2, 16, 4, 64, 16, 4000, 0, native.DTYPE_BF16)
    assert need > 0 and lib.plora_paged_attention_workspace(2, 16, 4, 64, 16, 4000, 100, native.DTYPE_BF16) == 0
    assert _attend(lib, native, width=4000, ts=4000, wb=need - 1) == native.ERR_WORKSPACE
    assert _attend(lib, native, width=4000, ts=4000, ws=None, wb=need) == native.ERR_WORKSPACE
    assert _attend(lib, native, rows=0) == native.OK
    for bad in ((2, 16, 5, 64, 16, 4000, 0, 2), (2, 0, 4, 64, 16, 4000, 0, 2), (2, 16, 4, 65, 16, 4000, 0, 2),
                (2, 16, 4, 512, 16, 4000, 0, 2), (2, 16, 4, 64, 16, 4000, 0, 7), (-1, 16, 4, 64, 16, 4000, 0, 2),
                (2, 16, 4, 64, 0, 4000, 0, 2), (2, 16, 4, 64, 16, 4000, -1, 2), (2, 16, 4, 64, 1 << 20, 4000, 0, 2)):
        assert lib.plora_paged_attention_workspace(*bad) == 0


def test_rules_arguments_rejected_before_cuda(native):
    lib = native.load()

    def rules(**kw):
        a = dict(x=D, xs=100, y=D, ys=100, rows=2, vocab=100, dtype=native.DTYPE_BF16, tok=D, tr=8, hist=8, bt=D, br=4,
                 bv=D, vr=4, k=4, mask=None, mr=0, tb=8, ws=D, wb=1 << 30)
        a.update(kw)
        return lib.plora_logit_rules(native.LOGIT_RULES_ARGS.pack(
            a["x"] or 0, a["xs"], a["y"] or 0, a["ys"], a["rows"], a["vocab"], a["dtype"], a["tok"] or 0, a["tr"], a["hist"],
            0, 0, 0, 0, 0, a["bt"] or 0, a["br"], a["bv"] or 0, a["vr"], a["k"], a["mask"] or 0, a["mr"], a["tb"],
            a["ws"] or 0, a["wb"]), None)

    for kw in (dict(dtype=3), dict(rows=-1), dict(vocab=-1), dict(hist=-1), dict(k=-1), dict(tb=2), dict(x=None),
               dict(y=None), dict(tok=None), dict(bt=None), dict(bv=None), dict(xs=99), dict(ys=99), dict(tr=-1),
               dict(br=-1), dict(mask=D, mr=-1), dict(x=D + 1)):
        assert rules(**kw) == native.ERR_INVALID_ARGUMENT, kw
    for kw in (dict(rows=70000), dict(vocab=1 << 31, xs=1 << 31, ys=1 << 31), dict(hist=1 << 30), dict(k=4097)):
        assert rules(**kw) == native.ERR_UNSUPPORTED, kw
    assert rules(rows=0) == native.OK and rules(vocab=0) == native.OK
    assert rules(ws=D + 64) == native.ERR_INVALID_ARGUMENT
    need = lib.plora_logit_rules_workspace(1000, 100, 8, 4)
    assert need > 0 and lib.plora_logit_rules_workspace(2, 100, 8, 4) == 0
    # the lists are for a copy, which a call in place without a mask does not make
    assert rules(rows=1000, y=2 * D, wb=need - 1) == native.ERR_WORKSPACE
    assert rules(rows=1000, y=2 * D, ws=None, wb=need) == native.ERR_WORKSPACE
    for bad in ((-1, 100, 8, 4), (1000, 1 << 31, 8, 4), (1000, 100, -1, 4), (1000, 100, 8, 5000)):
        assert lib.plora_logit_rules_workspace(*bad) == 0


def test_outputs_that_share_a_part_of_their_input_are_refused(native):
    """The ranges are worked out on the host; a call that is taken fails here
    for want of a GPU, with another status."""
    lib = native.load()

    def rules(rows, vocab, x, xs, y, ys):
        return lib.plora_logit_rules(native.LOGIT_RULES_ARGS.pack(
            x, xs, y, ys, rows, vocab, native.DTYPE_BF16, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, D, 4, 8, 0, 0), None)

    for bad in ((2, 100, D, 100, D + 2, 100), (2, 100, D + 198, 100, D, 100), (2, 100, D, 100, D, 104),
                (2, 100, D, 250, D + 2 * 151, 250), (3, 100, D, 250, D + 2 * (250 + 99), 250), (1, 100, D, 100, D + 16, 100)):
        assert rules(*bad) == native.ERR_INVALID_ARGUMENT, bad
        assert "shares" in native.last_error()
    for bad in ((2, 100, D, 1 << 62, 2 * D, 100), (2, 100, D, 100, 2 * D, 1 << 62)):
        assert rules(*bad) == native.ERR_INVALID_ARGUMENT, bad
    for kw in (dict(out=D + 16), dict(q=D + 2 * 2 * 16 * 64 - 16), dict(qs=(2048, 64)), dict(qs=(1024, 128)),
               dict(qs=(0, 64)), dict(qs=(1 << 61, 64), out=2 * D)):
        assert _attend(lib, native, **kw) == native.ERR_INVALID_ARGUMENT, kw
    if torch.cuda.is_available():
        return
    for good in ((2, 100, D, 100, D, 100), (2, 100, D, 100, D + 400, 100), (1, 100, D, 100, D + 200, 100),
                 (2, 100, D, 250, D + 2 * 150, 250), (3, 100, D, 250, D + 2 * (250 + 100), 250)):
        assert rules(*good) not in (native.OK, native.ERR_INVALID_ARGUMENT), good
    for kw in (dict(), dict(out=D + 2 * 2 * 16 * 64), dict(rows=1, qs=(0, 64))):
        assert _attend(lib, native, **kw) not in (native.OK, native.ERR_INVALID_ARGUMENT), kw


def test_cpu_tensors_are_refused():
    kc, table, lens = torch.zeros(1, 1, 4, 8), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        paged_attention(torch.zeros(1, 1, 8), kc, kc, table, lens)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        paged_append(None, torch.zeros(1, 1, 1, 8), torch.zeros(1, 1, 1, 8), kc, kc, table, lens)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        apply_logit_rules(torch.zeros(1, 5), LogitRules())


def test_rotary_phases_are_exact_fractions():
    """Position * phase mod 2^64 is the angle's fraction of a turn to 2^-36 of a
    turn at positions of millions; a phase is off by half a unit of 2^-64 and by
    64-bit division, 2^-52 of a fraction below one."""
    freq = torch.cat([500000.0 ** -(torch.arange(0, 128, 2) / 128), torch.tensor([0.0, 3.0, 6.5, -0.25, 1e-9])])
    for f, p in zip(freq.tolist(), rotary_phases(freq).tolist()):
        for pos in (0, 1, 8191, 131071, 5_000_000):
            turn = ((pos * p) % (1 << 64)) / 2.0**64
            want = math.fmod(pos * math.fmod(f, 2 * math.pi), 2 * math.pi) / (2 * math.pi)
            off = (turn - want) % 1.0
            assert min(off, 1 - off) < (pos + 1) * 2.0**-50, (f, pos)
    assert rotary_phases(torch.zeros(0)).shape == (0,)
    for bad in (torch.zeros(2, 2), torch.zeros(2, dtype=torch.int64), torch.tensor([math.inf])):
        with pytest.raises(ValueError):
            rotary_phases(bad)


def test_heads_copies_only_what_it_must():
    t = torch.zeros(2, 3, 4, 16, dtype=torch.bfloat16)
    for same in (t, t.transpose(0, 1), t[:, :, 1:3], t[:, :, :1].expand(2, 3, 4, 16)):
        assert _heads(same)[0].data_ptr() == same.data_ptr()
    for other in (t.transpose(-1, -2), t[..., 1:9], torch.zeros(2, 3, 4, 12, dtype=torch.bfloat16)[..., :8]):
        got, st, ptr = _heads(other)
        assert got.is_contiguous() and got.data_ptr() == ptr and ptr % 16 == 0
        assert other.shape[-1] % 8 or all(s % 8 == 0 for s in st[:-1])  # heads that the operators take
    assert _heads(torch.zeros(1, 2, 4, 16, dtype=torch.bfloat16).as_strided((1, 2, 4, 16), (7, 64, 16, 1)))[1][0] % 8 == 0


def test_argument_structs_match_the_header(native, tmp_path):
    """The packed layouts are the C structs' (sizes and the offset of every
    section, from a compiled program), and null arguments are refused."""
    import shutil
    import subprocess
    from pathlib import Path

    lib = native.load()
    for fn in (lib.plora_paged_append, lib.plora_paged_attention, lib.plora_logit_rules):
        assert fn(None, None) == native.ERR_INVALID_ARGUMENT
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    src = tmp_path / "sizes.c"
    src.write_text('#include "polylora_b200.h"\n#include <stdio.h>\n#define P(x) printf("%d\\n", (int)(x))\n'
                   "int main(void) { P(sizeof(plora_paged_append_args)); P(sizeof(plora_paged_attention_args));"
                   "P(sizeof(plora_logit_rules_args)); P(offsetof(plora_paged_append_args, q));"
                   "P(offsetof(plora_paged_append_args, q_out)); P(offsetof(plora_paged_append_args, rotary_scale));"
                   "P(offsetof(plora_paged_attention_args, q)); P(offsetof(plora_paged_attention_args, scale));"
                   "P(offsetof(plora_paged_attention_args, workspace)); P(offsetof(plora_logit_rules_args, allowed));"
                   "return 0; }\n")
    include = Path(__file__).resolve().parents[1] / "include"
    subprocess.run([cc, "-std=c11", f"-I{include}", str(src), "-o", str(tmp_path / "sizes")], check=True)
    got = subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout.split()
    want = [native.PAGED_APPEND_ARGS.size, native.PAGED_ATTENTION_ARGS.size, native.LOGIT_RULES_ARGS.size, 14 * 8, 26 * 8,
            34 * 8, 14 * 8, 19 * 8, 21 * 8, 20 * 8]
    assert [int(x) for x in got] == want
