"""What callers of a bounded cache ask once: workspaces for the longest call over its capacity, used by every smaller one, and
whether the library has windows at all."""
import ctypes
import os
import random
import re

import pytest

from hyprstream_amd import bindings as hb

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

P, CROOKED = ctypes.c_void_p(0x100000), ctypes.c_void_p(0x100040)


def accepted(nbytes, B, S, Hq, Hkv, D, T):
    """Is a workspace of `nbytes` large enough for the call?  (Asked with one of a wrong alignment, which is refused once
    its size has passed: nothing is launched.)"""
    lay = hb.contiguous_layout(Hkv, T, D)
    rc = hb.lib().hs_attn_weights(0, P, P, P, ctypes.byref(lay), None, 0, None, P, ctypes.c_int64((T + 3) // 4 * 4), CROOKED,
                                  ctypes.c_size_t(nbytes), B, S, Hq, Hkv, D, T, ctypes.c_float(0.1), None)
    assert rc in (hb.HS_ERR_WORKSPACE, hb.HS_ERR_INVALID_ARGUMENT), rc
    if rc == hb.HS_ERR_INVALID_ARGUMENT:
        assert b"256-byte" in hb.lib().hs_attn_last_error()
    return rc == hb.HS_ERR_INVALID_ARGUMENT


def test_a_workspace_for_the_capacity_serves_every_prefix():
    B, S, Hq, Hkv, D, T = 1, 512, 32, 8, 128, 32768
    n = hb.attn_weights_workspace_bytes(B, S, Hq, Hkv, D, T)
    assert all(accepted(n, B, S, Hq, Hkv, D, t) for t in range(S, T + 1, 64))
    assert not accepted(16, B, S, Hq, Hkv, D, T)


@pytest.mark.parametrize("seed", range(20))
def test_a_workspace_serves_fewer_queries_and_tokens(seed):
    r = random.Random(seed)
    log = lambda lo, hi: int(round(lo * (hi / lo) ** r.random()))
    for _ in range(40):
        B, Hkv, D = log(1, 64), r.choice([1, 2, 3, 8]), r.choice([64, 128, 256])
        Hq, T = Hkv * r.choice([1, 2, 3, 4, 8, 40]), log(1, 1 << 20)
        S = log(1, T)
        n = hb.attn_weights_workspace_bytes(B, S, Hq, Hkv, D, T)
        for _ in range(40):
            t = r.choice([T, log(1, T), max(1, T - r.randrange(3000))])
            s = min(t, r.choice([S, log(1, S), max(1, S - r.randrange(40))]))
            assert accepted(n, B, s, Hq, Hkv, D, t), (B, S, Hq, Hkv, D, T, s, t)
            assert hb.attn_weights_workspace_bytes(B, s, Hq, Hkv, D, t) <= n


@pytest.mark.parametrize("D", [64, 128, 256])
def test_the_bound_stays_near_what_calls_take(D):
    """Room for what a call of exactly this size takes (the statistics: 4 bytes per column) and 16 MB at most."""
    for B, S, G, Hkv, T in ((1, 1, 4, 8, 1 << 20), (1, 32, 4, 8, 32768), (4, 4096, 4, 8, 4096), (64, 1, 4, 8, 8192), (1, 32768, 8, 8, 32768), (64, 512, 1, 8, 8192)):
        n = hb.attn_weights_workspace_bytes(B, S, Hkv * G, Hkv, D, T)
        assert 4 * B * Hkv * S * G <= n <= 4 * B * Hkv * (S * G + 127) + (16 << 20)


def test_revision_tells_libraries_with_windows_from_those_before():
    """Windows took the place of reserved fields within one ABI version: the revision is what a caller of theirs asks for,
    and a library from before does not have it."""
    L, text = hb.lib(), open(os.path.join(ROOT, "include", "hs_attn.h")).read()
    assert L.hs_attn_abi_revision() == int(re.search(r"#define HS_ATTN_ABI_REVISION (\d+)", text).group(1)) >= 1
    rust = open(os.path.join(ROOT, "hs-attn-sys", "src", "bindings.rs")).read()
    assert "pub const HS_ATTN_ABI_REVISION: c_int = %d;" % L.hs_attn_abi_revision() in rust
    check = re.search(r"pub fn check_abi\(\).*?\n}", open(os.path.join(ROOT, "hs-attn-sys", "src", "lib.rs")).read(), flags=re.S).group(0)
    assert "hs_attn_abi_revision()" in check and "HS_ATTN_ABI_REVISION" in check
