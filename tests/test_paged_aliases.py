"""Caches that share memory, worked out on the host; a call that is taken fails
here for want of a GPU, with another status."""

import pytest
import torch

from test_paged_args import D, _append

PAGE = 4 * 16 * 64  # elements of _append's pages; 8 pages of bf16


@pytest.mark.parametrize("kw", [
    dict(), dict(vc=D + 16), dict(vc=D + 2 * PAGE), dict(vc=D + 2 * (8 * PAGE) - 16), dict(kc=D + 2 * PAGE, vc=D),
    dict(vc=D + 2 * PAGE, kp=2 * PAGE, vp=PAGE), dict(vc=D + 2 * PAGE - 16, kp=2 * PAGE, vp=2 * PAGE),
    dict(vc=D, pages=1), dict(vc=D + 16, pages=1),
])
def test_an_append_whose_caches_share_memory_is_refused(native, kw):
    assert _append(native.load(), native, **{"kp": PAGE, "vp": PAGE, **kw}) == native.ERR_INVALID_ARGUMENT
    assert "share memory" in native.last_error()


@pytest.mark.parametrize("kw", [
    dict(vc=D + 2 * (8 * PAGE)), dict(vc=D + 2 * PAGE, kp=2 * PAGE, vp=2 * PAGE), dict(kc=D + 2 * PAGE, vc=D, kp=2 * PAGE, vp=2 * PAGE),
    dict(vc=D + 2 * PAGE, pages=1),
])
def test_caches_apart_or_page_by_page_are_taken(native, kw):
    if torch.cuda.is_available():
        pytest.skip("the addresses are made up")
    assert _append(native.load(), native, **{"kp": PAGE, "vp": PAGE, **kw}) not in (native.OK, native.ERR_INVALID_ARGUMENT)
