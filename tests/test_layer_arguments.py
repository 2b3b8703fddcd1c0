"""CPU: the entry points of rotary, windowed and 4-bit layers check their arguments before any device call."""
import ctypes as C

import numpy as np
import pytest
import torch


def _buf(n):
    a = np.zeros(n + 16, np.uint8)
    return a, a.ctypes.data + (-a.ctypes.data) % 16


def _rope(**kw):
    import rag_hip
    keep, p = _buf(4096)
    a = dict(qkv=p, stride=96, pos=p, gq=None, gk=None, eps=1e-6, inv=p, rot=32, inter=0, t=1, hq=1, hkv=1, d=32, dt=0, q=p, qs=32, k=p, krs=32, khs=32,
             v=None, vrs=0, vhs=0, row=None, rows=1, stream=None)
    a.update(kw)
    return rag_hip.load_library().rag_enc_qk_norm_rope_dev(*a.values()), rag_hip.last_error()


@pytest.mark.parametrize('kw,code', [
    (dict(dt=7), -1), (dict(d=48), -5), (dict(d=256), -5), (dict(t=-1), -1), (dict(hq=0), -1), (dict(hkv=0), -1), (dict(rot=12), -5), (dict(rot=40), -5),
    (dict(rot=-8), -5), (dict(rows=0), -1), (dict(qkv=None), -1), (dict(q=None), -1), (dict(k=None), -1), (dict(pos=None), -1), (dict(inv=None), -1),
    (dict(stride=95), -1), (dict(stride=92), -1), (dict(qs=28), -1), (dict(krs=33), -1), (dict(khs=2), -1), (dict(t=1 << 41, rows=1 << 41), -5)])
def test_rope_arguments(kw, code):
    rc, text = _rope(**kw)
    assert rc == code and 'rag_enc_qk_norm_rope' in text


def _window(**kw):
    import rag_hip
    keep, p = _buf(4096)
    a = dict(q=p, qs=32, k=p, krs=32, khs=32, v=p, vrs=32, vhs=32, cu=p, tq=1, ks=None, kl=None, tk=1, n=1, mq=1, mk=1, hq=1, hkv=1, d=32, scale=1.0,
             left=-1, right=-1, sinks=0, dt=1, out=p, os=32, work=None, bytes=0, stream=None)
    a.update(kw)
    return rag_hip.load_library().rag_enc_attention_window_dev(*a.values()), rag_hip.last_error()


@pytest.mark.parametrize('kw,code', [
    (dict(dt=3), -1), (dict(d=48), -5), (dict(n=-1), -1), (dict(mq=-1), -1), (dict(tq=-1), -1), (dict(tk=-1), -1), (dict(tq=1 << 31), -5), (dict(mk=1 << 30), -5),
    (dict(hq=3, hkv=2), -1), (dict(hkv=0), -1), (dict(left=-2), -1), (dict(right=-2), -1), (dict(sinks=-1), -1), (dict(scale=float('inf')), -1), (dict(scale=3e38), -1),
    (dict(q=None), -1), (dict(k=None), -1), (dict(out=None), -1), (dict(cu=None), -1), (dict(qs=24), -1), (dict(qs=33), -1), (dict(os=16), -1), (dict(krs=4), -1), (dict(bytes=-1), -1)])
def test_window_arguments(kw, code):
    rc, text = _window(**kw)
    assert rc == code and 'rag_enc_attention_window' in text


def test_window_starts_and_lengths_come_together():
    keep, p = _buf(64)
    assert _window(ks=p)[0] == -1 and _window(kl=p)[0] == -1


def test_workspace_goes_by_the_sizes_and_never_overflows():
    import rag_hip
    f = rag_hip.load_library().rag_enc_attention_window_workspace
    one = f(1, 1, 1, 32768, 32, 8, 128, -1, 0, 0, 1)
    assert one > 0 and one % (32 * 130 * 4 + 8 * 8) == 0       # spans of one token's 32 heads: 128 sums, a maximum and a total; a mark of each key head
    assert f(1 << 30, 1, 1, 32768, 32, 8, 128, -1, 0, 0, 1) == one       # rows of no sequence take no room
    assert f(16384, 1, 16384, 16384, 16, 8, 128, 4096, 0, 4, 1) == 0 and f(0, 0, 0, 0, 1, 1, 64, -1, -1, 0, 0) == 0
    big = (1 << 31) - 1
    for dtype in (0, 1, 2):
        for args in ((big, big, 1, (1 << 30) - 1, 4096, 1, 128), (big, 1, (1 << 30) - 1, (1 << 30) - 1, 4096, 1, 32), (big, 1, 1, (1 << 30) - 1, 4096, 4096, 128)):
            for window in ((-1, -1, 0), (big, big, big), (0, 0, big)):
                assert 0 <= f(*args, *window, dtype) < 1 << 50


def test_a_workspace_too_small_is_refused():
    # refused before any launch: 32768 keys in spans need room for their partial results
    assert _window(hq=32, hkv=8, d=128, qs=4096, os=4096, tq=1, mk=32768, tk=32768, ks=_buf(64)[1], kl=_buf(64)[1])[0] == -1


def test_nothing_to_do_is_no_error():
    assert _rope(t=0, rows=0)[0] == 0 and _window(n=0)[0] == 0 and _window(tq=0, mq=0)[0] == 0 and _linear(m=0)[0] == 0


def _linear(**kw):
    import rag_hip
    keep, p = _buf(4096)
    a = dict(x=p, xs=64, codes=p, scales=p, off=None, bias=None, m=1, n=8, k=64, group=32, dt=1, y=p, ys=8, stream=None)
    a.update(kw)
    return rag_hip.load_library().rag_enc_linear4_dev(*a.values()), rag_hip.last_error()


@pytest.mark.parametrize('kw,code', [
    (dict(dt=9), -1), (dict(m=-1), -1), (dict(n=0), -1), (dict(k=0), -1), (dict(group=16), -5), (dict(group=64, k=96), -5), (dict(k=48), -5), (dict(m=1 << 31), -5),
    (dict(x=None), -1), (dict(codes=None), -1), (dict(scales=None), -1), (dict(y=None), -1), (dict(xs=65), -1), (dict(m=2, xs=56), -1), (dict(m=2, ys=7), -1)])
def test_linear4_arguments(kw, code):
    rc, text = _linear(**kw)
    assert rc == code and 'rag_enc_linear4' in text


@pytest.mark.parametrize('kw', [
    dict(n=1 << 28), dict(k=1 << 26), dict(m=2, xs=(1 << 24) + 8), dict(m=2, xs=1 << 62), dict(m=2, dt=0, xs=(1 << 23) + 4)])
def test_linear4_limits(kw):
    rc, text = _linear(**kw)
    assert rc == -5 and 'rag_enc_linear4' in text


@pytest.mark.parametrize('kw', [dict(krs=(1 << 24) + 8), dict(vrs=(1 << 24) + 8), dict(krs=-32), dict(vrs=1 << 61), dict(dt=0, krs=(1 << 23) + 4)])
def test_window_rows_far_apart_are_refused(kw):
    rc, text = _window(**kw)
    assert rc == -5 and 'rag_enc_attention_window' in text


@pytest.mark.parametrize('symmetric', [False, True])
def test_quantize4_on_the_cpu(symmetric):
    import rag_hip
    w = torch.randn((9, 128), generator=torch.Generator().manual_seed(1))
    codes, scales, off = rag_hip.quantize4(w, 32, symmetric=symmetric)
    c = torch.stack([codes & 15, codes >> 4], dim=2).reshape(9, 128).double()
    s = scales.double().repeat_interleave(32, dim=1)
    o = -8 * s if off is None else off.double().repeat_interleave(32, dim=1)
    # half a step, and the 32-bit roundings of the step and the quotient (16 steps of 2^-23)
    assert bool(((c * s + o - w.double()).abs() <= s * (0.5 + 64 * 2.0 ** -23)).all())
    with pytest.raises(ValueError):
        rag_hip.quantize4(w, 48)
    with pytest.raises(ValueError):
        rag_hip.quantize4(w[:, :96], 64)
    with pytest.raises(ValueError):
        rag_hip.quantize4(w, 32, dtype=torch.float64)


def test_rope_inv_freq():
    import rag_hip
    f = rag_hip.rope_inv_freq(8, 10000.0, device='cpu')
    assert f.dtype == torch.float64 and np.allclose(f.numpy(), [1, 0.1, 0.01, 0.001], rtol=1e-15)


@pytest.mark.parametrize('at', range(1, 10))
def test_sizes_beyond_the_interface_are_refused(at):
    # ctypes would pass 2^32 as 0: a window of one key instead of one beyond every length
    import rag_hip
    sizes = [4, 1, 4, 4, 2, 2, 64, -1, 0, 0, 1]
    assert rag_hip._window_workspace(*sizes) == 0
    sizes[at] = 1 << 32
    with pytest.raises(ValueError, match='2\\^31'):
        rag_hip._window_workspace(*sizes)


def test_calls_of_more_workgroups_than_a_launch_takes_are_refused():
    n = 1 << 28                                               # 2^26 workgroups of 256 threads
    assert _rope(t=n, rows=n)[0] == -5
    assert _window(tq=n, tk=n, n=n)[0] == -5


def test_workspace_of_many_sequences_and_heads_does_not_overflow():
    import rag_hip
    f = rag_hip.load_library().rag_enc_attention_window_workspace
    big, most = (1 << 31) - 1, (1 << 30) - 1
    for hq, hkv in ((4096, 4096), (4096, 2048), (4096, 1), (1, 1)):
        for max_q in (1, 5, 100, 1 << 20, most):
            for max_k in (0, 1, 70000, most):
                for dtype in (0, 1):
                    for window in ((-1, -1, 0), (0, 0, 0), (big, big, big)):
                        assert f(big, big, max_q, max_k, hq, hkv, 128, *window, dtype) == 0       # they fill the chip: nothing is cut


@pytest.mark.parametrize('kw', [dict(krs=0), dict(krs=-28), dict(khs=16), dict(khs=0), dict(v=True, vrs=0), dict(v=True, vhs=-16)])
def test_rope_keys_and_values_that_overlap_are_refused(kw):
    # an expanded tensor: all tokens, or all heads, would be written to the same place
    keep, p = _buf(4096)
    a = dict(t=2, rows=2, hq=1, hkv=2, stride=160, krs=64, khs=32, vrs=64, vhs=32)
    a.update(kw)
    if kw.get('v'):
        a['v'] = p
    rc, text = _rope(**a)
    assert rc == -1 and 'overlap' in text
    assert _rope(**{**a, 't': 0})[0] == 0


@pytest.mark.parametrize('symmetric', [False, True])
def test_quantize4_refuses_what_four_bits_cannot_hold(symmetric):
    import rag_hip
    w = torch.randn((4, 64), generator=torch.Generator().manual_seed(3))
    for bad in (float('nan'), float('inf'), -float('inf')):
        x = w.clone()
        x[2, 40] = bad
        with pytest.raises(ValueError, match='infinities or NaN'):
            rag_hip.quantize4(x, 32, symmetric=symmetric)
    with pytest.raises(ValueError, match='beyond torch.float16'):
        rag_hip.quantize4(w * 1e6, 32, dtype=torch.float16, symmetric=symmetric)
    x = w.clone()
    x[1, 1], x[1, 2] = 3e38, -3e38                            # their difference, or 8 scales of 3e38 / 7, is beyond the type
    with pytest.raises(ValueError, match='beyond torch.float32'):
        rag_hip.quantize4(x, 32, symmetric=symmetric)
    assert bool(torch.isfinite(rag_hip.quantize4(w * 1e4, 32, dtype=torch.float16, symmetric=symmetric)[1]).all())
