"""Windows set on a layout and windows named in a call: the call's own where it names them, else the layout's, which stays as
its owner set it up.  Every call here is refused before it could launch anything; which refusal it is tells what the library
was handed."""
import pytest
import torch

from hyprstream_amd import bindings as hb

B, S, Hq, Hkv, D, T = 1, 2, 4, 2, 64, 64


def _args():
    codes, scales = torch.zeros(B, Hkv, T, D, dtype=torch.int8), torch.zeros(B, Hkv, T)
    return [codes, codes, scales, scales]


def _decode(lay, **kw):
    q = torch.zeros(B, Hq, D, dtype=torch.bfloat16)
    hb.decode_attn(q, *_args(), lay, torch.zeros(B, dtype=torch.int32), q, None, Hkv, T, 0.1, **kw)


def _static(lay, **kw):
    q = torch.zeros(B, Hq, D, dtype=torch.bfloat16)
    hb.decode_attn_static(q, *_args(), lay, torch.zeros(B, dtype=torch.int32), q, Hkv, T + 1, 0.1, **kw)  # more than the cache holds


def _step(lay, fn=hb.decode_step, extra=(), **kw):
    q, n = torch.zeros(B, Hq, D, dtype=torch.bfloat16), torch.zeros(B, 1, Hkv, D, dtype=torch.bfloat16)
    fn(q, n, n, *extra, *_args(), lay, torch.zeros(B, dtype=torch.int32), q, torch.zeros(16, dtype=torch.uint8), Hkv, T, 0.1, **kw)


def _rope(lay, **kw):
    table = torch.zeros(T, D // 2, dtype=torch.bfloat16)
    _step(lay, hb.decode_step_rope, (table, table), **kw)


def _prologue(lay, **kw):
    _step(lay, hb.decode_step_prologue, (hb.QkPrologue(),), **kw)


def _step_weights(lay, **kw):
    q, w = torch.zeros(B, Hq, D, dtype=torch.bfloat16), torch.zeros(B, Hkv, T)
    hb.decode_step_weights(q, None, None, *_args(), lay, torch.zeros(B, dtype=torch.int32), q, None, w, torch.zeros(16, dtype=torch.uint8), Hkv, T,
                           0.1, **kw)


def _weights(lay, **kw):
    q, w = torch.zeros(B, S, Hq, D, dtype=torch.bfloat16), torch.zeros(B, Hkv, T)
    hb.attn_weights(q, *_args()[::2], lay, None, w, torch.zeros(16, dtype=torch.uint8), Hkv, T, 0.1, start_pos=-1, **kw)


def _prefill(lay, **kw):
    q, n = torch.zeros(B, S, 3, D, dtype=torch.bfloat16), torch.zeros(B, S, Hkv, D, dtype=torch.bfloat16)
    hb.prefill_attn(q, n, n, *_args(), lay, 8, q, 0.1, **kw)


CALLS = [("decode_window", f) for f in (_decode, _static, _step, _rope, _prologue, _step_weights)] + [("prefill_window", f) for f in (_weights, _prefill)]


@pytest.fixture(autouse=True)
def _no_gpu(monkeypatch):
    monkeypatch.setattr(hb, "_stream", lambda: None)


@pytest.mark.parametrize("field,call", CALLS, ids=lambda x: x if isinstance(x, str) else x.__name__[1:])
def test_a_call_without_a_window_takes_the_layouts(field, call):
    for name in (field, "attn_sinks"):
        lay = hb.contiguous_layout(Hkv, T, D)
        with pytest.raises(hb.HsError) as e:
            call(lay)  # nothing negative: refused for the other reason
        assert "negative %s" % field not in str(e.value) and "attn_sinks" not in str(e.value)
        setattr(lay, name, -7)
        with pytest.raises(hb.HsError, match="negative (decode_window|prefill_window)"):
            call(lay)
        assert getattr(lay, name) == -7


@pytest.mark.parametrize("field,call", CALLS, ids=lambda x: x if isinstance(x, str) else x.__name__[1:])
def test_a_call_with_a_window_leaves_the_layout(field, call):
    lay = hb.contiguous_layout(Hkv, T, D)
    for kw in (dict(window=-7), dict(sinks=-7), dict(window=5, sinks=-7)):
        with pytest.raises(hb.HsError, match="negative (decode_window|prefill_window)"):
            call(lay, **kw)
    setattr(lay, field, -7)
    lay.attn_sinks = -9
    with pytest.raises(hb.HsError) as e:
        call(lay, window=0, sinks=0)
    assert "attn_sinks" not in str(e.value)
    assert getattr(lay, field) == -7 and lay.attn_sinks == -9 and lay.prefill_window + lay.decode_window == -7
