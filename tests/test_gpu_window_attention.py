"""GPU: attention with a sliding window and sinks (rag_enc_attention_window_dev) against the formula in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}


def _dev():
    return torch.device('cuda:0')


def _gen(seed):
    return torch.Generator(device=_dev()).manual_seed(seed)


def _cu(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device=_dev())


def _reference(q, k, v, left, right, sinks, scale):
    """One sequence in 64 bits: (result, softmax @ |v|, largest sum of |q k| scale of a row).  Keys that a query does not
    see are taken out before the product with the values."""
    nq, hq, d = q.shape
    nk, hkv, _ = k.shape
    p = torch.arange(nk - nq, nk, device=q.device)[:, None]
    c = torch.arange(nk, device=q.device)[None, :]
    seen = torch.ones((nq, nk), dtype=torch.bool, device=q.device)
    if right >= 0:
        seen &= c - p <= right
    if left >= 0:
        seen &= (p - c <= left) | (c < sinks)
    out = torch.zeros((nq, hq, d), dtype=torch.float64, device=q.device)
    mag, top = torch.zeros_like(out), torch.zeros((nq, hq, 1), dtype=torch.float64, device=q.device)
    for h in range(hq):
        qq, kk, vv = q[:, h].double(), k[:, h // (hq // hkv)].double(), v[:, h // (hq // hkv)].double()
        s = torch.where(seen, qq @ kk.t() * scale, torch.full((), -math.inf, dtype=torch.float64, device=q.device))
        w = torch.where(seen.any(dim=1, keepdim=True), torch.softmax(s, dim=1), torch.zeros_like(s))
        vz = torch.where(torch.isfinite(vv), vv, torch.zeros_like(vv))
        out[:, h], mag[:, h] = w @ vz, w @ vz.abs()
        if nk:
            top[:, h] = (qq.abs() @ torch.nan_to_num(kk, 0, 0, 0).abs().t() * abs(scale)).amax(dim=1, keepdim=True)
    return out, mag, top, seen


def _tolerance(dt, out, mag, top, nk, d):
    # scores: d + 4 roundings of a sum of magnitude top, an exponential of 2 ulp and a sum over nk, in the numerator and in the
    # denominator; 16-bit types: the weights are rounded once (numerator), and the result once
    work = 2 * ((d + 4) * 2.0 ** -24 * top + 2.0 ** -22 + (nk + 8) * 2.0 ** -24)
    info = torch.finfo(dt)
    if dt == torch.float32:
        return work * mag + info.smallest_normal
    # fp16: a weight below the smallest normal (2^-14 of the largest) is rounded to half of 2^-24
    small = nk * 2.0 ** -25 if dt == torch.float16 else 0.0
    inner = (work + info.eps / 2) * mag + small * (mag + mag.amax(dim=-1, keepdim=True))
    return inner + info.eps / 2 * (out.abs() + inner) + info.smallest_normal * info.eps / 2


def _check(got, q, k, v, q_lens, k_rows, left, right, sinks, scale):
    """k_rows: (first row, rows) of every sequence's keys."""
    at, (_, hq, d) = 0, q.shape
    for n, (k0, nk) in zip(q_lens, k_rows):
        out, mag, top, _ = _reference(q[at:at + n], k[k0:k0 + nk], v[k0:k0 + nk], left, right, sinks, scale)
        err = (got[at:at + n].view(n, hq, d).double() - out).abs()
        tol = _tolerance(q.dtype, out, mag, top, nk, d)
        assert bool((err <= tol).all()), (n, nk, float((err - tol).max()), float(err.max()))
        at += n


def _packed(lens, hq, hkv, d, dt, seed, gain=1.0):
    qkv = torch.randn((sum(lens), hq + 2 * hkv, d), generator=_gen(seed), device=_dev())
    qkv[:, :hq] *= gain
    qkv = qkv.to(dt)
    return qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]


WINDOWS = [(-1, -1, 0), (-1, 0, 0), (0, 0, 0), (5, 0, 3), (40, 40, 1), (100, 0, 70), (0, -1, 2), (-1, 7, 5), (63, 64, 0), (500, 0, 4)]


@pytest.mark.parametrize('kind', list(TYPES))
@pytest.mark.parametrize('hq,hkv,d', [(2, 2, 32), (6, 2, 64), (4, 1, 128)])
@pytest.mark.parametrize('left,right,sinks', WINDOWS)
def test_packed_sequences(kind, hq, hkv, d, left, right, sinks):
    import rag_hip
    lens = [1, 0, 33, 128, 2, 300, 64, 0, 31, 129, 65]
    q, k, v = _packed(lens, hq, hkv, d, TYPES[kind], 7 * d + left + right)
    got = rag_hip.enc_attention_window_dev(q, k, v, _cu(lens), max(lens), window_left=left, window_right=right, n_sinks=sinks)
    starts = _cu(lens).tolist()
    _check(got, q, k, v, lens, list(zip(starts, lens)), left, right, sinks, d ** -0.5)


@pytest.mark.parametrize('kind', list(TYPES))
@pytest.mark.parametrize('left,right,sinks', [(-1, -1, 0), (-1, 0, 0), (700, 0, 4), (256, 256, 1), (1023, 0, 0)])
def test_long_sequences(kind, left, right, sinks):
    import rag_hip
    lens = [1500, 2049, 40]
    q, k, v = _packed(lens, 2, 1, 64, TYPES[kind], 11, gain=2.0)
    got = rag_hip.enc_attention_window_dev(q, k, v, _cu(lens), max(lens), window_left=left, window_right=right, n_sinks=sinks)
    _check(got, q, k, v, lens, list(zip(_cu(lens).tolist(), lens)), left, right, sinks, 0.125)


KEPT = [([1], [1]), ([1, 1, 1], [700, 0, 1]), ([1, 1], [5000, 31]), ([3, 1, 5, 0], [64, 900, 3, 10]), ([17, 2], [1000, 257]),
        ([40, 1, 64], [2000, 65, 64]), ([4, 9], [2, 0]), ([130], [1111]), ([1] * 40, list(range(40)))]


@pytest.mark.parametrize('kind', list(TYPES))
@pytest.mark.parametrize('hq,hkv,d', [(1, 1, 32), (8, 2, 64), (16, 1, 128), (12, 3, 128), (40, 2, 64)])
@pytest.mark.parametrize('case', range(len(KEPT)))
def test_queries_behind_kept_keys(kind, hq, hkv, d, case):
    import rag_hip
    q_lens, k_lens = KEPT[case]
    dt, g = TYPES[kind], _gen(case * 10 + d)
    room = max(k_lens) + 3
    q = torch.randn((sum(q_lens), hq, d), generator=g, device=_dev()).to(dt)
    k = torch.randn((len(k_lens) * room, hkv, d), generator=g, device=_dev()).to(dt)
    v = torch.randn((len(k_lens) * room, hkv, d), generator=g, device=_dev()).to(dt)
    order = torch.randperm(len(k_lens), generator=g, device=_dev())
    k_start, k_len = order * room, torch.tensor(k_lens, dtype=torch.int32, device=_dev())
    rows = list(zip(k_start.tolist(), k_lens))
    used = torch.zeros(k.shape[0], dtype=torch.bool, device=_dev())
    for k0, nk in rows:
        used[k0:k0 + nk] = True
    k[~used] = float('nan')                                    # what no sequence owns
    v[~used] = float('inf')
    for left, right, sinks in [(-1, 0, 0), (63, 0, 4), (300, 0, 40), (-1, -1, 0), (10, 3, 1)]:
        got = rag_hip.enc_attention_window_dev(q, k, v, _cu(q_lens), max(q_lens), k_start=k_start, k_len=k_len, max_k_len=max(k_lens),
                                               window_left=left, window_right=right, n_sinks=sinks)
        _check(got, q, k, v, q_lens, rows, left, right, sinks, d ** -0.5)


@pytest.mark.parametrize('kind', list(TYPES))
def test_one_token_over_a_long_text(kind):
    import rag_hip
    dt, g, n = TYPES[kind], _gen(1), 40000
    q = torch.randn((2, 8, 128), generator=g, device=_dev()).to(dt)
    k, v = (torch.randn((2 * n, 2, 128), generator=g, device=_dev()).to(dt) for _ in range(2))
    k_start = torch.tensor([0, n], device=_dev())
    k_len = torch.tensor([n, n - 12345], dtype=torch.int32, device=_dev())
    for left, sinks in ((-1, 0), (8191, 4), (20000, 100)):
        got = rag_hip.enc_attention_window_dev(q, k, v, _cu([1, 1]), 1, k_start=k_start, k_len=k_len, max_k_len=n, window_left=left, window_right=0, n_sinks=sinks)
        _check(got, q, k, v, [1, 1], [(0, n), (n, n - 12345)], left, 0, sinks, 128 ** -0.5)


def test_heads_outside_rows_and_a_shared_prefix():
    """Keys laid out [sequence][head][row], and two sequences that read the same kept rows."""
    import rag_hip
    g, hq, hkv, d, room = _gen(2), 6, 3, 64, 200
    store = torch.randn((2, hkv, room, d), generator=g, device=_dev()).to(torch.bfloat16)
    vals = torch.randn((2, hkv, room, d), generator=g, device=_dev()).to(torch.bfloat16)
    rows = (2 - 1) * hkv * room + room                          # rows of d elements from the first head's point of view
    view = lambda x: x.as_strided((rows, hkv, d), (d, room * d, 1))
    q = torch.randn((5, hq, d), generator=g, device=_dev()).to(torch.bfloat16)
    q_lens, owner, k_lens = [2, 1, 2], [1, 0, 1], [150, 200, 150]
    got = rag_hip.enc_attention_window_dev(q, view(store), view(vals), _cu(q_lens), 2, k_start=torch.tensor([hkv * room, 0, hkv * room], device=_dev()),
                                           k_len=torch.tensor(k_lens, dtype=torch.int32, device=_dev()), max_k_len=200, window_left=90,
                                           window_right=0, n_sinks=2)
    at = 0
    for n, o, nk in zip(q_lens, owner, k_lens):
        kk, vv = store[o].transpose(0, 1)[:nk], vals[o].transpose(0, 1)[:nk]
        _check(got[at:at + n], q[at:at + n], kk, vv, [n], [(0, nk)], 90, 0, 2, d ** -0.5)
        at += n


@pytest.mark.parametrize('kind', list(TYPES))
@pytest.mark.parametrize('d', [32, 128])
def test_what_is_not_seen_does_not_enter(kind, d):
    """NaN and infinities in keys and values that some queries see and others do not."""
    import rag_hip
    lens, hq, hkv = [150, 70], 4, 2
    q, k, v = _packed(lens, hq, hkv, d, TYPES[kind], 5)
    k[100, 0], v[20, 0, 3], v[101, 1], v[160] = float('nan'), float('inf'), float('nan'), float('-inf')
    for left, right, sinks in ((30, 0, 0), (16, 16, 21), (-1, 0, 0)):
        got = rag_hip.enc_attention_window_dev(q, k, v, _cu(lens), max(lens), window_left=left, window_right=right, n_sinks=sinks).view(sum(lens), hq, d)
        for a, n in ((0, lens[0]), (lens[0], lens[1])):
            for h in range(hq):
                kv = h // (hq // hkv)
                out, mag, top, seen = _reference(q[a:a + n, h:h + 1], k[a:a + n, kv:kv + 1], v[a:a + n, kv:kv + 1], left, right, sinks, d ** -0.5)
                bad_k = ~torch.isfinite(k[a:a + n, kv]).all(dim=1)
                bad_v = ~torch.isfinite(v[a:a + n, kv])
                spoiled = (seen & bad_k[None]).any(dim=1)[:, None] | ((seen.float() @ bad_v.float()) > 0)
                mine = got[a:a + n, h].double()
                assert not bool(torch.isfinite(mine[spoiled]).any())
                ok = ~spoiled
                tol = _tolerance(q.dtype, out, mag, top, n, d)[:, 0]
                assert bool(((mine - out[:, 0]).abs()[ok] <= tol[ok]).all()), (left, right, sinks, a, h)


def test_extreme_scores():
    """Scores of some thousands, and of minus some thousands, whose exponentials leave the 32-bit range without their maximum."""
    import rag_hip
    lens = [200]
    q, k, v = _packed(lens, 2, 2, 64, torch.float32, 3, gain=500.0)
    got = rag_hip.enc_attention_window_dev(q, k, v, _cu(lens), 200, window_left=50, window_right=0, n_sinks=2)
    _check(got, q, k, v, lens, [(0, 200)], 50, 0, 2, 0.125)
    qb, kb, vb = (x.to(torch.bfloat16) for x in (q, k, v))
    got = rag_hip.enc_attention_window_dev(qb, kb, vb, _cu(lens), 200, window_left=50, window_right=0, n_sinks=2, scale=-0.25)
    _check(got, qb, kb, vb, lens, [(0, 200)], 50, 0, 2, -0.25)


@pytest.mark.parametrize('kind', list(TYPES))
@pytest.mark.parametrize('nq,nk', [(1, 3000), (200, 200)])
def test_other_scales(kind, nq, nk):
    """A scale of zero (the mean of what is seen), tiny, large and negative ones, in both kernels."""
    import rag_hip
    g, dt = _gen(12), TYPES[kind]
    q = torch.randn((nq, 4, 64), generator=g, device=_dev()).to(dt)
    k, v = (torch.randn((nk, 2, 64), generator=g, device=_dev()).to(dt) for _ in range(2))
    for scale in (0.0, 1e-30, 1e-3, 2.0, -0.125):
        got = rag_hip.enc_attention_window_dev(q, k, v, _cu([nq]), nq, k_start=torch.zeros(1, dtype=torch.int64, device=_dev()),
                                               k_len=torch.tensor([nk], dtype=torch.int32, device=_dev()), max_k_len=nk, window_left=150, window_right=0,
                                               n_sinks=3, scale=scale)
        _check(got, q, k, v, [nq], [(0, nk)], 150, 0, 3, scale)


@pytest.mark.parametrize('hq,hkv', [(8, 8), (8, 1), (40, 1)])
def test_sequences_among_rows_of_none(hq, hkv):
    """Two short sequences somewhere in a long array of queries, over many keys (partial results are kept by sequence)."""
    import rag_hip
    g, rows = _gen(13), 5000
    q = torch.randn((rows, hq, 64), generator=g, device=_dev()).to(torch.bfloat16)
    k, v = (torch.randn((6000, hkv, 64), generator=g, device=_dev()).to(torch.bfloat16) for _ in range(2))
    out = torch.full((rows, hq * 64), 7.0, dtype=torch.bfloat16, device=_dev())
    cu = torch.tensor([4000, 4003, 4005], dtype=torch.int32, device=_dev())
    rag_hip.enc_attention_window_dev(q, k, v, cu, 3, k_start=torch.tensor([0, 500], device=_dev()), k_len=torch.tensor([6000, 5500], dtype=torch.int32, device=_dev()),
                                     max_k_len=6000, window_right=0, out=out)
    _check(out[4000:4005], q[4000:4005], k, v, [3, 2], [(0, 6000), (500, 5500)], -1, 0, 0, 0.125)
    assert bool((out[:4000] == 7).all()) and bool((out[4005:] == 7).all())


@pytest.mark.parametrize('kind', list(TYPES))
@pytest.mark.parametrize('max_q', [4, 80])
def test_bad_sequences_are_flagged_and_rows_of_none_stay(kind, max_q):
    import rag_hip
    rag_hip.fault_flags()
    dt, d = TYPES[kind], 64
    q, k, v = _packed([90], 2, 1, d, dt, 1)
    out = torch.full((90, 2 * d), 7.0, dtype=dt, device=_dev())
    cu = torch.tensor([0, 4, 88, 6, 10, 93, 95], dtype=torch.int32, device=_dev())     # good, too long, negative, good, too long, beyond the rows
    rag_hip.enc_attention_window_dev(q, k, v, cu, max_q, window_right=0, out=out)
    assert rag_hip.fault_flags() == 128
    assert bool((out[4:6] == 7).all()) and bool((out[10:] == 7).all())
    for a in (0, 6):
        _check(out[a:a + 4], q[a:a + 4], k[a:a + 4], v[a:a + 4], [4], [(0, 4)], -1, 0, 0, 0.125)
    out.fill_(7)
    # kept keys: a negative start, a length beyond max_k_len, a range beyond the rows; one good
    cu = torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32, device=_dev())
    ks = torch.tensor([-1, 0, 60, 10], device=_dev())
    kl = torch.tensor([5, 41, 31, 20], dtype=torch.int32, device=_dev())
    rag_hip.enc_attention_window_dev(q, k, v, cu, max_q, k_start=ks, k_len=kl, max_k_len=40, window_right=0, out=out)
    assert rag_hip.fault_flags() == 512
    assert bool((out[:3] == 7).all()) and bool((out[4:] == 7).all())
    _check(out[3:4], q[3:4], k, v, [1], [(10, 20)], -1, 0, 0, 0.125)


def test_offsets_beyond_32_bits():
    """The last rows of an array of more than 2^32 elements."""
    import rag_hip
    d, hkv = 128, 2
    rows = (1 << 32) // (hkv * d) + 5000
    k = torch.zeros((rows, hkv, d), dtype=torch.bfloat16, device=_dev())
    v = torch.zeros((rows, hkv, d), dtype=torch.bfloat16, device=_dev())
    g = _gen(4)
    n = 900
    k[-n:] = torch.randn((n, hkv, d), generator=g, device=_dev()).to(torch.bfloat16)
    v[-n:] = torch.randn((n, hkv, d), generator=g, device=_dev()).to(torch.bfloat16)
    for nq in (1, 200):
        q = torch.randn((nq, 4, d), generator=g, device=_dev()).to(torch.bfloat16)
        got = rag_hip.enc_attention_window_dev(q, k, v, _cu([nq]), nq, k_start=torch.tensor([rows - n], device=_dev()),
                                               k_len=torch.tensor([n], dtype=torch.int32, device=_dev()), max_k_len=n, window_right=0)
        _check(got, q, k[-n:], v[-n:], [nq], [(0, n)], -1, 0, 0, d ** -0.5)
    # and written there by the pass in front of it
    qkv = torch.randn((2, 8 * d), generator=g, device=_dev()).to(torch.bfloat16)
    rag_hip.enc_qk_norm_rope_dev(qkv, torch.zeros(2, dtype=torch.int32, device=_dev()), rag_hip.rope_inv_freq(d), 4, 2, k_out=k, v_out=v,
                                 kv_row=torch.tensor([rows - 1, 0], device=_dev()))
    x = qkv.view(2, 8, d)
    assert torch.equal(k[-1], x[0, 4:6]) and torch.equal(v[-1], x[0, 6:]) and torch.equal(k[0], x[1, 4:6])


def test_no_rows_and_refusals():
    import rag_hip
    dev = _dev()
    q, k, v = _packed([6], 4, 2, 32, torch.bfloat16, 1)
    cu = _cu([6])
    assert rag_hip.enc_attention_window_dev(q[:0], k[:0], v[:0], _cu([]), 0).shape == (0, 128)
    assert rag_hip.enc_attention_window_dev(q[:0], k[:0], v[:0], _cu([0, 0]), 0).shape == (0, 128)
    one = torch.zeros(1, dtype=torch.int64, device=dev)
    no_keys = rag_hip.enc_attention_window_dev(q, k[:0], v[:0], cu, 6, k_start=one, k_len=one.int(), max_k_len=0)
    assert float(no_keys.abs().max()) == 0.0
    for bad in (dict(q=q.double()), dict(k=k.float()), dict(v=v[:, :1]), dict(k=k[:5], v=v[:5]), dict(k_start=one), dict(cu_q=cu.long()),
                dict(k_start=one, k_len=one.int()), dict(k_start=one, k_len=one, max_k_len=1), dict(q=q.cpu()), dict(cu_q=cu.cpu()),
                dict(q=q[:, :3]), dict(out=torch.zeros((6, 128), device=dev)), dict(q=q.transpose(0, 1).contiguous().transpose(0, 1)),
                dict(q=q[..., ::2], k=k[..., ::2], v=v[..., ::2]), dict(k_start=torch.zeros(2, dtype=torch.int64, device=dev), k_len=torch.zeros(2, dtype=torch.int32, device=dev), max_k_len=1)):
        kw = dict(q=q, k=k, v=v, cu_q=cu, max_q_len=6)
        kw.update(bad)
        with pytest.raises(ValueError):
            rag_hip.enc_attention_window_dev(**kw)
    for bad in (dict(window_left=-2), dict(window_right=-5), dict(n_sinks=-1), dict(scale=float('nan')), dict(max_q_len=-1)):
        kw = dict(q=q, k=k, v=v, cu_q=cu, max_q_len=6)
        kw.update(bad)
        with pytest.raises(rag_hip.RagHipError):
            rag_hip.enc_attention_window_dev(**kw)
    with pytest.raises(rag_hip.RagHipError):                   # head size 48
        x = torch.zeros((6, 2, 48), dtype=torch.bfloat16, device=dev)
        rag_hip.enc_attention_window_dev(x, x, x, cu, 6)
    with pytest.raises(rag_hip.RagHipError):                   # misaligned rows
        x = torch.zeros(6 * 65, dtype=torch.bfloat16, device=dev).as_strided((6, 1, 64), (65, 64, 1), 1)
        rag_hip.enc_attention_window_dev(x, x, x, cu, 6)


@pytest.mark.parametrize('kept', [False, True])
def test_another_stream_and_graphs_replayed_in_turn(kept):
    """Two captured calls of other sizes, replayed in turn with eager calls between: no buffer is shared between them."""
    import rag_hip
    g, hq, hkv, d = _gen(6), 8, 2, 64

    def make(nq, nk):
        q = torch.randn((nq, hq, d), generator=g, device=_dev()).to(torch.bfloat16)
        k, v = (torch.randn((nk, hkv, d), generator=g, device=_dev()).to(torch.bfloat16) for _ in range(2))
        kw = dict(window_left=3000, window_right=0, n_sinks=4)
        if kept:
            kw.update(k_start=torch.zeros(1, dtype=torch.int64, device=_dev()), k_len=torch.tensor([nk], dtype=torch.int32, device=_dev()), max_k_len=nk)
        return lambda: rag_hip.enc_attention_window_dev(q, k, v, _cu_kept[nq], nq, **kw), q
    _cu_kept = {n: _cu([n]) for n in (1, 2, 700, 300)}
    (f1, q1), (f2, q2) = (make(1, 9000), make(2, 5000)) if kept else (make(700, 700), make(300, 300))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = f1()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, f1())
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        y1 = f1()
    with torch.cuda.graph(g2):
        y2 = f2()
    for i in range(4):
        q1.mul_(0.9)
        q2.mul_(1.1)
        g1.replay()
        g2.replay()
        a, b = f1(), f2()
        torch.cuda.synchronize()
        assert torch.equal(y1, a) and torch.equal(y2, b), i


def test_a_layer_of_all_three_token_by_token_and_at_once():
    """4-bit q|k|v projection, norm + rotation into the kept keys, windowed attention, 4-bit output projection: a text fed
    at once, in pieces behind its kept prefix and token by token gives the same rows, and those of the layer in 64 bits."""
    import rag_hip
    g, hq, hkv, d, hidden, n = _gen(9), 8, 2, 64, 256, 150
    dt = torch.bfloat16
    w_in = rag_hip.quantize4((torch.randn(((hq + 2 * hkv) * d, hidden), generator=g, device=_dev()) / 16).to(dt), 64)
    w_out = rag_hip.quantize4((torch.randn((hidden, hq * d), generator=g, device=_dev()) / 23).to(dt), 32, symmetric=True)
    gamma = (1 + 0.2 * torch.randn(d, generator=g, device=_dev())).to(dt)
    inv = rag_hip.rope_inv_freq(d)
    x = torch.randn((n, hidden), generator=g, device=_dev()).to(dt)
    first = 40                                                  # where the text lies among the kept rows

    def layer(cuts):
        k_keep, v_keep = (torch.full((250, hkv, d), float('nan'), dtype=dt, device=_dev()) for _ in range(2))
        rows = []
        for a, b in zip(cuts, cuts[1:]):
            at = torch.arange(a, b, device=_dev())
            qkv = rag_hip.enc_linear4_dev(x[a:b], *w_in)
            q, _, _ = rag_hip.enc_qk_norm_rope_dev(qkv, at.int(), inv, hq, hkv, gamma_q=gamma, gamma_k=gamma, k_out=k_keep, v_out=v_keep, kv_row=at + first)
            ctx = rag_hip.enc_attention_window_dev(q, k_keep, v_keep, _cu([b - a]), b - a, k_start=torch.tensor([first], device=_dev()),
                                                   k_len=torch.tensor([b], dtype=torch.int32, device=_dev()), max_k_len=b, window_left=50,
                                                   window_right=0, n_sinks=2)
            rows.append(rag_hip.enc_linear4_dev(ctx, *w_out))
        return torch.cat(rows).double()

    def wide(w):
        codes, scales, off = w
        c = torch.stack([codes & 15, codes >> 4], dim=2).reshape(codes.shape[0], -1).double()
        s = scales.double().repeat_interleave(c.shape[1] // scales.shape[1], dim=1)
        return c * s + (off.double().repeat_interleave(c.shape[1] // scales.shape[1], dim=1) if off is not None else -8 * s)
    qkv = (x.double() @ wide(w_in).t()).view(n, hq + 2 * hkv, d)
    qk = qkv[:, :hq + hkv]
    qk = qk / torch.sqrt((qk * qk).mean(dim=-1, keepdim=True) + 1e-6) * gamma.double()
    t = torch.arange(n, device=_dev()).double()[:, None] * inv[None, :]
    c, s = torch.cos(t)[:, None], torch.sin(t)[:, None]
    lo, hi = qk[..., :d // 2], qk[..., d // 2:]
    qk = torch.cat([lo * c - hi * s, hi * c + lo * s], dim=-1)
    ctx, mag, top, _ = _reference(qk[:, :hq], qk[:, hq:], qkv[:, hq + hkv:], 50, 0, 2, d ** -0.5)
    want = ctx.reshape(n, -1) @ wide(w_out).t()
    # Roundings to bf16 on the way (u = 2^-8 each): q|k|v once, normed and rotated q and k once more: a score is off by at
    # most 4 u of its sum of magnitudes (top), which moves softmax weights by e^(2 * 4 u top) - 1; values u, weights u, ctx u,
    # result u.  top is below 64 * scale * (max |gamma|)^2-ish, so the worst case is wide; the errors are
    # independent, so the root-mean-square is held to a tenth of it.
    u = 2.0 ** -8
    worst = torch.expm1(8 * u * top) + 3 * u
    tol = ((worst * mag).reshape(n, -1) @ wide(w_out).abs().t()) + u * want.abs()
    runs = [layer([0, n]), layer([0, 3, 90, 91, 130, n]), layer(list(range(n + 1)))]
    for got in runs:
        assert bool(((got - want).abs() <= tol).all())
        assert float((got - want).pow(2).mean().sqrt()) <= 0.1 * float(tol.pow(2).mean().sqrt())


@pytest.mark.parametrize('kind', list(TYPES))
def test_a_workspace_may_hold_anything(kind):
    # Spans' results are put together by the workgroups of the call itself, which mark what they have written in the workspace.
    # Whatever the memory holds, the same call gives the same bits: zeros, ones, what another call of other sizes
    # left there, what this call left there, and a captured call that finds its own leavings when it is replayed.
    import rag_hip
    dt, dev, hq, hkv, d = TYPES[kind], _dev(), 4, 2, 64
    code = {'f32': 0, 'bf16': 1, 'f16': 2}[kind]
    lens = [1500, 0, 3, 2600, 40, 700, 2599]
    g = _gen(91)
    k = torch.randn((sum(lens), hkv, d), generator=g, device=dev).to(dt)
    v = torch.randn((sum(lens), hkv, d), generator=g, device=dev).to(dt)
    q = torch.randn((len(lens), hq, d), generator=g, device=dev).to(dt)
    ks = [sum(lens[:i]) for i in range(len(lens))]
    cu, k_start = _cu([1] * len(lens)), torch.tensor(ks, dtype=torch.int64, device=dev)
    k_len = torch.tensor(lens, dtype=torch.int32, device=dev)
    lib = rag_hip.load_library()
    work = torch.zeros((1 << 20,), dtype=torch.uint8, device=dev)

    def call(left, out):
        need = lib.rag_enc_attention_window_workspace(len(lens), len(lens), 1, 2600, hq, hkv, d, left, 0, 2, code)
        assert 0 < need <= work.numel()
        rc = lib.rag_enc_attention_window_dev(q.data_ptr(), hq * d, k.data_ptr(), hkv * d, d, v.data_ptr(), hkv * d, d, cu.data_ptr(), len(lens),
                                              k_start.data_ptr(), k_len.data_ptr(), sum(lens), len(lens), 1, 2600, hq, hkv, d, d ** -0.5, left, 0, 2,
                                              code, out.data_ptr(), hq * d, work.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        return out

    def fresh():
        return torch.full((len(lens), hq * d), 7.0, dtype=dt, device=dev)

    want = {left: call(left, fresh()) for left in (-1, 1400)}
    for left in (-1, 1400):
        _check(want[left], q, k, v, [1] * len(lens), list(zip(ks, lens)), left, 0, 2, d ** -0.5)
    for fill in (0, 0xff, None):
        for left in (-1, 1400, -1):
            if fill is not None:
                work.fill_(fill)
            assert torch.equal(call(left, fresh()), want[left])
    out = fresh()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        call(-1, out)
    for i in range(6):
        out.fill_(3.0)
        graph.replay()
        assert torch.equal(out, want[-1]), i
        assert torch.equal(call(1400, fresh()), want[1400])
        torch.cuda.synchronize()


@pytest.mark.parametrize('kind', list(TYPES))
@pytest.mark.parametrize('hq,hkv', [(4, 1), (16, 1)])
def test_many_spans(kind, hq, hkv):
    # one token whose keys are cut into few spans and into many, a length that ends inside a tile and a span, and one key
    import rag_hip
    dt, dev, d = TYPES[kind], _dev(), 64
    for nk, max_k in ((1, 20000), (33, 20000), (1029, 1029), (5003, 20000), (20000, 20000), (30011, 30011)):
        g = _gen(nk)
        k, v = (torch.randn((nk, hkv, d), generator=g, device=dev).to(dt) for _ in range(2))
        q = torch.randn((1, hq, d), generator=g, device=dev).to(dt)
        got = rag_hip.enc_attention_window_dev(q, k, v, _cu([1]), 1, k_start=torch.zeros(1, dtype=torch.int64, device=dev),
                                               k_len=torch.full((1,), nk, dtype=torch.int32, device=dev), max_k_len=max_k, window_right=0)
        _check(got, q, k, v, [1], [(0, nk)], -1, 0, 0, d ** -0.5)


def test_two_streams_at_once():
    # two calls whose spans are on the chip together, each with its own workspace
    import rag_hip
    dt, dev, hq, hkv, d, nk = torch.bfloat16, _dev(), 4, 1, 128, 6000
    g = _gen(17)
    k, v = (torch.randn((2 * nk, hkv, d), generator=g, device=dev).to(dt) for _ in range(2))
    q = torch.randn((2, hq, d), generator=g, device=dev).to(dt)
    one, cu = torch.full((1,), nk, dtype=torch.int32, device=dev), _cu([1])
    starts = [torch.full((1,), i * nk, dtype=torch.int64, device=dev) for i in range(2)]

    def call(i):
        return rag_hip.enc_attention_window_dev(q[i:i + 1], k, v, cu, 1, k_start=starts[i], k_len=one, max_k_len=nk, window_right=0)

    want = [call(i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(call(i))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


@pytest.mark.parametrize('kind', list(TYPES))
@pytest.mark.parametrize('hq,hkv,d', [(6, 2, 64), (8, 1, 32), (4, 4, 128), (12, 1, 128)])
@pytest.mark.parametrize('left,right,sinks', [(-1, -1, 0), (-1, 0, 0), (900, 0, 5), (300, 200, 1)])
def test_pieces_of_a_text_behind_kept_keys(kind, hq, hkv, d, left, right, sinks):
    # some tens or hundreds of queries on long keys: the rows of a key/value head in tiles, the keys in spans
    import rag_hip
    dt, dev = TYPES[kind], _dev()
    q_lens, lens = [1, 0, 37, 210, 70], [3000, 10, 37, 2100, 40]
    g = _gen(hq * 7 + d)
    q = torch.randn((sum(q_lens) + 3, hq, d), generator=g, device=dev).to(dt)
    k, v = (torch.randn((sum(lens), hkv, d), generator=g, device=dev).to(dt) for _ in range(2))
    k0 = [sum(lens[:i]) for i in range(len(lens))]
    out = torch.full((q.shape[0], hq * d), 5.0, dtype=dt, device=dev)
    kw = dict(k_start=torch.tensor(k0, dtype=torch.int64, device=dev), k_len=torch.tensor(lens, dtype=torch.int32, device=dev), max_k_len=3000,
              window_left=left, window_right=right, n_sinks=sinks)
    rag_hip.enc_attention_window_dev(q, k, v, _cu(q_lens), 210, out=out, **kw)
    assert bool((out[sum(q_lens):] == 5.0).all())
    _check(out, q, k, v, q_lens, list(zip(k0, lens)), left, right, sinks, d ** -0.5)
    if right == 0:
        # keys and values behind the first 150 queries of the fourth sequence hold what must not reach them, key by key
        # (rows that meet them are computed again in another order: as near the formula, but not the same bits)
        kn, vn = k.clone(), v.clone()
        hidden = k0[3] + 2100 - 60
        kn[hidden::2], vn[hidden::3] = math.nan, math.inf
        again = rag_hip.enc_attention_window_dev(q, kn, vn, _cu(q_lens), 210, **kw)
        _check(again[38:188], q[38:188], k, v, [150], [(k0[3], 2100 - 60)], left, right, sinks, d ** -0.5)


def test_pieces_of_a_text_in_a_captured_graph():
    import rag_hip
    dt, dev, hq, hkv, d, nq, nk = torch.bfloat16, _dev(), 8, 2, 64, 90, 7000
    g = _gen(5)
    q = torch.randn((nq, hq, d), generator=g, device=dev).to(dt)
    k, v = (torch.randn((nk, hkv, d), generator=g, device=dev).to(dt) for _ in range(2))
    cu, k_start, k_len = _cu([nq]), torch.zeros(1, dtype=torch.int64, device=dev), torch.full((1,), nk, dtype=torch.int32, device=dev)

    def call():
        return rag_hip.enc_attention_window_dev(q, k, v, cu, nq, k_start=k_start, k_len=k_len, max_k_len=nk, window_right=0)
    graph = torch.cuda.CUDAGraph()
    call()
    with torch.cuda.graph(graph):
        out = call()
    for n in (7000, 300, 90, 7000, 2501):
        k_len.fill_(n)
        q.mul_(0.95)
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(out, want), n
        _check(want, q, k, v, [nq], [(0, n)], -1, 0, 0, d ** -0.5)


@pytest.mark.parametrize('hq,hkv,d', [(2, 2, 32), (4, 2, 64), (2, 1, 128)])
@pytest.mark.parametrize('q_lens,k_lens,right', [([300, 600], None, -1), ([300, 600], None, 0), ([64, 64, 60], [2049, 700, 2000], 0), ([1, 3, 2], [4000, 300, 2500], 0)])
def test_float32_keeps_24_bits(hq, hkv, d, q_lens, k_lens, right):
    # The worst-case tolerance above is too wide to tell products of all 24 bits from less, so the root-mean-square error is held to
    # the root of the summed squares of what is added up (weight times value).  In half steps of that, 2^-24: a score of
    # magnitude 1 is at most d / 16 * 6 * 4 = 192 roundings, each uniform (1 / sqrt(3)), 8; its exponential with the
    # multiply-add in front of it 5; the sums of weights and of weighted values grow over nk / 16 * 6 roundings, at most 0.9
    # sqrt(nk) together.  One of the six products of parts left out gives 250 to 380 (computed with the parts in 64 bits).
    import rag_hip
    g = _gen(d + sum(q_lens))
    k_rows = sum(q_lens if k_lens is None else k_lens)
    q = torch.randn((sum(q_lens), hq, d), generator=g, device=_dev())
    k, v = (torch.randn((k_rows, hkv, d), generator=g, device=_dev()) for _ in range(2))
    kw = {}
    if k_lens is not None:
        kw = dict(k_start=_cu(k_lens)[:-1].long(), k_len=torch.tensor(k_lens, dtype=torch.int32, device=_dev()), max_k_len=max(k_lens))
    got = rag_hip.enc_attention_window_dev(q, k, v, _cu(q_lens), max(q_lens), window_right=right, **kw).view(-1, hq, d).double()
    at = k0 = 0
    for nq, nk in zip(q_lens, q_lens if k_lens is None else k_lens):
        hidden = torch.arange(nk, device=_dev())[None, :] > torch.arange(nk - nq, nk, device=_dev())[:, None]
        for h in range(hq):
            kk, vv = k[k0:k0 + nk, h // (hq // hkv)].double(), v[k0:k0 + nk, h // (hq // hkv)].double()
            s = q[at:at + nq, h].double() @ kk.t() * d ** -0.5
            w = torch.softmax(s.masked_fill(hidden, -math.inf) if right == 0 else s, dim=1)
            err, square = got[at:at + nq, h] - w @ vv, w ** 2 @ vv ** 2
            assert float(err.pow(2).mean().sqrt()) <= (16 + nk ** 0.5) * 2.0 ** -24 * float(square.mean().sqrt()), (nq, nk, h)
        at, k0 = at + nq, k0 + nk


@pytest.mark.parametrize('kind', ['bf16', 'f32'])
@pytest.mark.parametrize('hq,hkv,d', [(2, 2, 32), (8, 2, 64), (4, 1, 128)])
@pytest.mark.parametrize('q_lens,k_lens,left,right', [([1, 200, 77], None, -1, 0), ([300], None, 60, 60), ([1], [40], -1, 0), ([1], [2000], -1, 0),
                                                      ([9, 3], [700, 2000], -1, 0), ([64, 50], [3000, 1800], -1, 0)])
def test_values_near_the_end_of_the_range(kind, hq, hkv, d, q_lens, k_lens, left, right):
    # values of 1e37 to 1e38: their weighted mean is as large, their sum with weights of up to 2^8, or of many keys, is beyond fp32
    import rag_hip
    dt, g = TYPES[kind], _gen(d + sum(q_lens))
    k_rows = q_lens if k_lens is None else k_lens
    q = (2 * torch.randn((sum(q_lens), hq, d), generator=g, device=_dev())).to(dt)
    k = torch.randn((sum(k_rows), hkv, d), generator=g, device=_dev()).to(dt)
    v = ((1 + 0.2 * torch.randn((sum(k_rows), hkv, d), generator=g, device=_dev())) * 4e37).to(dt)
    v[:, :, ::3] *= -1
    kw = {}
    if k_lens is not None:
        kw = dict(k_start=_cu(k_lens)[:-1].long(), k_len=torch.tensor(k_lens, dtype=torch.int32, device=_dev()), max_k_len=max(k_lens))
    got = rag_hip.enc_attention_window_dev(q, k, v, _cu(q_lens), max(q_lens), window_left=left, window_right=right, **kw)
    assert bool(torch.isfinite(got).all())
    _check(got, q, k, v, q_lens, list(zip(_cu(k_rows).tolist(), k_rows)), left, right, 0, d ** -0.5)


@pytest.mark.parametrize('nq,nk', [(3, 900), (1, 20000), (300, 400), (60, 3000)])
def test_queries_beyond_32_bits(nq, nk):
    """The last rows of queries of more than 2^32 elements; the rows in front of them belong to no sequence."""
    import rag_hip
    hq, hkv, d, g = 32, 8, 128, _gen(nq)
    rows = (1 << 32) // (hq * d) + 1000
    q = torch.zeros((rows, hq, d), dtype=torch.bfloat16, device=_dev())
    q[-nq:] = torch.randn((nq, hq, d), generator=g, device=_dev()).to(torch.bfloat16)
    k, v = (torch.randn((nk, hkv, d), generator=g, device=_dev()).to(torch.bfloat16) for _ in range(2))
    out = torch.full((rows, hq * d), 7.0, dtype=torch.bfloat16, device=_dev())
    rag_hip.enc_attention_window_dev(q, k, v, torch.tensor([rows - nq, rows], dtype=torch.int32, device=_dev()), nq, k_start=torch.zeros(1, dtype=torch.int64, device=_dev()),
                                     k_len=torch.tensor([nk], dtype=torch.int32, device=_dev()), max_k_len=nk, window_right=0, out=out)
    _check(out[-nq:], q[-nq:], k, v, [nq], [(0, nk)], -1, 0, 0, d ** -0.5)
    assert bool((out[:-nq] == 7).all())


@pytest.mark.parametrize('nq,nk', [(1, 5000), (200, 200), (60, 3000)])
def test_windows_beyond_every_length_are_no_windows(nq, nk):
    import rag_hip
    g, far = _gen(8), (1 << 31) - 1
    q = torch.randn((nq, 4, 64), generator=g, device=_dev()).to(torch.float16)
    k, v = (torch.randn((nk, 2, 64), generator=g, device=_dev()).to(torch.float16) for _ in range(2))
    kw = dict(k_start=torch.zeros(1, dtype=torch.int64, device=_dev()), k_len=torch.tensor([nk], dtype=torch.int32, device=_dev()), max_k_len=nk)
    want = rag_hip.enc_attention_window_dev(q, k, v, _cu([nq]), nq, **kw)
    for left, right, sinks in ((far, far, 0), (far, -1, far), (-1, 1 << 30, 5), (1 << 30, far, 0)):
        assert torch.equal(want, rag_hip.enc_attention_window_dev(q, k, v, _cu([nq]), nq, window_left=left, window_right=right, n_sinks=sinks, **kw))
    near = (1 << 30) - 1                                        # the longest that is one: every key in it, by another path perhaps
    got = rag_hip.enc_attention_window_dev(q, k, v, _cu([nq]), nq, window_left=near, window_right=near, n_sinks=far, **kw)
    _check(got, q, k, v, [nq], [(0, nk)], -1, -1, 0, 0.125)


@pytest.mark.parametrize('kind', list(TYPES))
@pytest.mark.parametrize('nq,nk', [(3, 40), (4, 5000), (200, 200), (60, 3000)])
def test_a_query_that_is_not_finite_spoils_its_own_row_only(kind, nq, nk):
    import rag_hip
    dt, g = TYPES[kind], _gen(nq)
    q = torch.randn((nq, 4, 64), generator=g, device=_dev()).to(dt)
    k, v = (torch.randn((nk, 2, 64), generator=g, device=_dev()).to(dt) for _ in range(2))
    bad = q.clone()
    bad[1, 2, 5], bad[2, 0, 7], bad[0, 3, 63] = float('nan'), float('inf'), -float('inf')
    got = rag_hip.enc_attention_window_dev(bad, k, v, _cu([nq]), nq, k_start=torch.zeros(1, dtype=torch.int64, device=_dev()),
                                           k_len=torch.tensor([nk], dtype=torch.int32, device=_dev()), max_k_len=nk, window_right=0).view(nq, 4, 64)
    assert bool(torch.isnan(got[1, 2]).all())
    ref = rag_hip.enc_attention_window_dev(q, k, v, _cu([nq]), nq, k_start=torch.zeros(1, dtype=torch.int64, device=_dev()),
                                           k_len=torch.tensor([nk], dtype=torch.int32, device=_dev()), max_k_len=nk, window_right=0).view(nq, 4, 64).clone()
    rest = torch.ones((nq, 4), dtype=torch.bool, device=_dev())
    rest[1, 2] = rest[2, 0] = rest[0, 3] = False
    mixed = torch.where(rest[:, :, None], got, ref)
    _check(mixed.reshape(nq, -1), q, k, v, [nq], [(0, nk)], -1, 0, 0, 0.125)


@pytest.mark.parametrize('kind', ['bf16', 'f16'])
@pytest.mark.parametrize('nq,hq,hkv,d,nk', [(1, 16, 8, 128, 2000), (1, 64, 4, 64, 300), (4, 16, 4, 32, 9000), (1, 8, 8, 128, 30000)])
def test_few_rows_are_rounded_once(kind, nq, hq, hkv, d, nk):
    # up to 16 rows of a key/value head: the result's own rounding is all that is lost, so the root-mean-square error is that
    # rounding's (with weights rounded to the type as well it would be 1.2 to 1.4 times as large; the fp32 work adds 2^-17 of it)
    import rag_hip
    dt, g = TYPES[kind], _gen(nk)
    q = torch.randn((nq * 16, hq, d), generator=g, device=_dev()).to(dt)
    k, v = (torch.randn((nk, hkv, d), generator=g, device=_dev()).to(dt) for _ in range(2))
    n = torch.full((16,), nk, dtype=torch.int32, device=_dev())
    got = rag_hip.enc_attention_window_dev(q, k, v, _cu([nq] * 16), nq, k_start=torch.zeros(16, dtype=torch.int64, device=_dev()), k_len=n, max_k_len=nk)
    want = torch.cat([_reference(x, k, v, -1, -1, 0, d ** -0.5)[0] for x in q.split(nq)]).reshape(nq * 16, -1)
    rounding = (want.to(dt).double() - want).pow(2).mean().sqrt()
    assert float((got.double() - want).pow(2).mean().sqrt()) <= 1.02 * float(rounding)
