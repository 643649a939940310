"""Entry points of the 8-bit cache refuse arrays that do not lie on a whole element: a kernel's loads from them would fault."""
import ctypes as C

import pytest

from test_kv8_host import BASE, _batch, _cache


@pytest.mark.parametrize("off", (1, 2, 3))
@pytest.mark.parametrize("which", ("k_scale", "v_scale", "seq_start", "kv_len", "table", "sinks"))
def test_cache_calls_refuse_arrays_off_their_elements(which, off):
    from macseek_b200 import _lib
    c, b = _cache(_lib, **({which: BASE + off} if which.endswith("scale") else {})), _batch(_lib, **({which: BASE + off} if which in ("seq_start", "kv_len", "table") else {}))
    sinks = BASE + off if which == "sinks" else None
    calls = [_lib.lib.msb_kv8_attn(C.byref(c), C.byref(b), 0, BASE, 256, 4, 0.1, 0, sinks, BASE, 256, BASE, 1 << 20, None)]
    if which != "sinks":
        calls += [call(C.byref(c), C.byref(b), 0, BASE, BASE, 128, 128, None) for call in (_lib.lib.msb_kv8_write, _lib.lib.msb_kv8_read)]
        assert _lib.lib.msb_kv8_attn_scratch_bytes(C.byref(c), C.byref(b), 4) == 0
    assert calls == [-1] * len(calls) and b"aligned" in _lib.lib.msb_last_error()


@pytest.mark.parametrize("off", (1, 2, 3))
@pytest.mark.parametrize("at", range(4))
def test_head_norm_rope_refuses_arrays_off_their_elements(at, off):
    from macseek_b200 import _lib
    q_w, k_w, cs, pos = (BASE + (off if at == i else 0) for i in range(4))
    assert _lib.lib.msb_head_norm_rope(0, BASE, 4, 256, q_w, BASE, 2, 128, k_w, 3, 64, 1e-6, cs, pos, 9, 64, 0, 0, BASE, 256, BASE, 128, None) == -1
    assert b"aligned" in _lib.lib.msb_last_error()
