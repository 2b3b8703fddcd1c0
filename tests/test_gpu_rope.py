"""GPU: norms of queries and keys + rotation by position in one pass (rag_enc_qk_norm_rope_dev) against the formula in 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}


def _dev():
    return torch.device('cuda:0')


def _gen(seed):
    return torch.Generator(device=_dev()).manual_seed(seed)


def _ref(x, pos, inv_freq, gamma, eps, interleaved):
    """x [T, heads, D] -> (result, |a| + |b| of the pair each value was made of), 64 bits."""
    n = x.double()
    if gamma is not None:
        n = n / torch.sqrt((n * n).mean(dim=-1, keepdim=True) + eps) * gamma.double()
    rot = 2 * (inv_freq.shape[0] if inv_freq is not None else 0)
    out, mag = n.clone(), n.abs()
    if rot:
        t = pos.double()[:, None] * inv_freq[None, :]
        c, s = torch.cos(t)[:, None], torch.sin(t)[:, None]
        i = torch.arange(rot // 2, device=x.device)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        na, nb = n[..., a], n[..., b]
        out[..., a], out[..., b] = na * c - nb * s, nb * c + na * s
        mag[..., a] = mag[..., b] = na.abs() + nb.abs()
    return out, mag


def _close(got, ref, mag):
    # the 32-bit work: norm (13 roundings of the sum of squares count half after the root, then root, quotient and two
    # products), sine and cosine (2 ulp), two products and a sum: below 24 half steps of the pair's magnitude; then one
    # rounding to the result's type, and half of its smallest step where the type runs out of exponent
    info = torch.finfo(got.dtype)
    err = (got.double() - ref).abs()
    work = 24 * 2.0 ** -24 * mag
    step = 0.0 if got.dtype == torch.float32 else info.eps / 2
    tol = work + step * (ref.abs() + work) + info.smallest_normal * info.eps / 2
    assert bool((err <= tol).all()), float((err - tol).max())


def _call(qkv, pos, inv, hq, hkv, gq, gk, inter, **kw):
    import rag_hip
    return rag_hip.enc_qk_norm_rope_dev(qkv, pos, inv, hq, hkv, gamma_q=gq, gamma_k=gk, eps=1e-6, interleaved=inter, **kw)


@pytest.mark.parametrize('kind', list(TYPES))
@pytest.mark.parametrize('t,hq,hkv,d,rot,inter,norm', [
    (1, 1, 1, 32, 32, False, True), (1, 16, 8, 128, 128, False, True), (2, 12, 12, 64, 64, True, True),
    (7, 5, 5, 32, 8, False, True), (33, 12, 4, 64, 24, True, False), (129, 32, 8, 128, 64, False, True),
    (257, 3, 1, 128, 120, False, True), (65, 7, 7, 64, 0, False, True), (3, 17, 1, 32, 16, True, True)])
def test_matches_the_formula(kind, t, hq, hkv, d, rot, inter, norm):
    import rag_hip
    g, dt = _gen(t * 100 + d + rot), TYPES[kind]
    qkv = (torch.randn((t, (hq + 2 * hkv) * d), generator=g, device=_dev()) * 2).to(dt)
    pos = torch.randint(-5, 1 << 20, (t,), generator=g, device=_dev(), dtype=torch.int32)
    inv = rag_hip.rope_inv_freq(rot) if rot else None
    gq = (1 + 0.3 * torch.randn(d, generator=g, device=_dev())).to(dt) if norm else None
    gk = (1 + 0.3 * torch.randn(d, generator=g, device=_dev())).to(dt) if norm else None
    before = qkv.clone()
    q, k, v = _call(qkv, pos, inv, hq, hkv, gq, gk, inter)
    x = qkv.view(t, hq + 2 * hkv, d)
    _close(q, *_ref(x[:, :hq], pos, inv, gq, 1e-6, inter))
    _close(k, *_ref(x[:, hq:hq + hkv], pos, inv, gk, 1e-6, inter))
    assert torch.equal(v, x[:, hq + hkv:])
    assert torch.equal(qkv, before)


def test_one_norm_without_the_other_and_zero_rows():
    import rag_hip
    g = _gen(3)
    qkv = torch.randn((5, 4 * 32), generator=g, device=_dev())
    qkv[2] = 0
    pos = torch.arange(5, dtype=torch.int32, device=_dev())
    inv, gk = rag_hip.rope_inv_freq(32), torch.randn(32, generator=g, device=_dev())
    q, k, _ = _call(qkv, pos, inv, 2, 1, None, gk, False)
    x = qkv.view(5, 4, 32)
    _close(q, *_ref(x[:, :2], pos, inv, None, 1e-6, False))
    _close(k, *_ref(x[:, 2:3], pos, inv, gk, 1e-6, False))
    assert float(q[2].abs().max()) == 0.0 and float(k[2].abs().max()) == 0.0


@pytest.mark.parametrize('kind', ['bf16', 'f32'])
def test_keys_and_values_go_to_the_rows_named(kind):
    import rag_hip
    g, dt = _gen(8), TYPES[kind]
    t, hq, hkv, d, rows = 37, 8, 2, 64, 300
    wide = (torch.randn((t, (hq + 2 * hkv) * d + 32), generator=g, device=_dev())).to(dt)
    qkv = wide[:, :(hq + 2 * hkv) * d]                          # rows with a stride
    pos = torch.randint(0, 5000, (t,), generator=g, device=_dev(), dtype=torch.int32)
    inv, gq = rag_hip.rope_inv_freq(d, 1e6), torch.randn(d, generator=g, device=_dev()).to(dt)
    # one array [rows][head][D], one [head][rows][D]
    k_out = torch.full((rows, hkv, d), 7.0, dtype=dt, device=_dev())
    v_out = torch.full((hkv, rows, d), 7.0, dtype=dt, device=_dev()).transpose(0, 1)
    row = torch.randperm(rows, generator=g, device=_dev())[:t].contiguous()
    row[5], row[20] = -1, -9
    q_out = torch.full((t + 3, hq, d), 7.0, dtype=dt, device=_dev())
    q, k, v = _call(qkv, pos, inv, hq, hkv, gq, gq, False, q_out=q_out[:t], k_out=k_out, v_out=v_out, kv_row=row)
    assert k is k_out and v is v_out and q.data_ptr() == q_out.data_ptr()
    x = qkv.unflatten(1, (hq + 2 * hkv, d))
    _close(q, *_ref(x[:, :hq], pos, inv, gq, 1e-6, False))
    here = row >= 0
    kr, km = _ref(x[:, hq:hq + hkv], pos, inv, gq, 1e-6, False)
    _close(k_out[row[here]], kr[here], km[here])
    assert torch.equal(v_out[row[here]], x[here][:, hq + hkv:])
    rest = torch.ones(rows, dtype=torch.bool, device=_dev())
    rest[row[here]] = False
    assert bool((k_out[rest] == 7).all()) and bool((v_out[rest] == 7).all()) and bool((q_out[t:] == 7).all())


def test_a_row_beyond_the_array_is_flagged_and_not_written():
    import rag_hip
    rag_hip.fault_flags()
    store = torch.full((12, 1, 32), 7.0, device=_dev())
    k_out = store[:10]
    qkv = torch.ones((3, 3 * 32), device=_dev())
    pos = torch.zeros(3, dtype=torch.int32, device=_dev())
    row = torch.tensor([0, 10, 1 << 40], device=_dev())
    _call(qkv, pos, rag_hip.rope_inv_freq(32), 1, 1, None, None, False, k_out=k_out, kv_row=row)
    assert rag_hip.fault_flags() == 512
    assert bool((store[0] == 1).all()) and bool((store[1:] == 7).all())


@pytest.mark.parametrize('kind', list(TYPES))
@pytest.mark.parametrize('inter', [False, True])
def test_in_place(kind, inter):
    import rag_hip
    g, dt = _gen(21), TYPES[kind]
    t, hq, hkv, d = 70, 6, 3, 64
    qkv = torch.randn((t, (hq + 2 * hkv) * d), generator=g, device=_dev()).to(dt)
    pos = torch.arange(t, dtype=torch.int32, device=_dev())
    inv, gq = rag_hip.rope_inv_freq(48), torch.randn(d, generator=g, device=_dev()).to(dt)
    want_q, want_k, want_v = _call(qkv, pos, inv, hq, hkv, gq, gq, inter)
    want_v = want_v.clone()
    x = qkv.view(t, hq + 2 * hkv, d)
    _call(qkv, pos, inv, hq, hkv, gq, gq, inter, q_out=x[:, :hq], k_out=x[:, hq:hq + hkv], v_out=x[:, hq + hkv:])
    assert torch.equal(x[:, :hq], want_q) and torch.equal(x[:, hq:hq + hkv], want_k) and torch.equal(x[:, hq + hkv:], want_v)


def test_far_positions_keep_the_angle():
    """Position 2^30: a 32-bit angle would be off by tens of radians."""
    import rag_hip
    qkv = torch.ones((4, 3 * 32), device=_dev())
    pos = torch.tensor([1 << 30, (1 << 30) + 1, -(1 << 30), 2147483647], dtype=torch.int32, device=_dev())
    inv = rag_hip.rope_inv_freq(32)
    q, _, _ = _call(qkv, pos, inv, 1, 1, None, None, False)
    t = (pos.cpu().numpy().astype(np.longdouble)[:, None] * inv.cpu().numpy().astype(np.longdouble)[None, :])
    # the angle in 64 bits is off by 2^-53 of itself (2.4e-7 at 2^31), in turns by as much again
    want = torch.from_numpy(np.concatenate([np.cos(t) - np.sin(t), np.cos(t) + np.sin(t)], axis=1).astype(np.float64))
    assert float((q[:, 0].cpu().double() - want).abs().max()) < 2 * 3 * 2.0 ** 31 * 2.0 ** -53 + 24 * 2.0 ** -24 * 2


def test_no_tokens_and_refusals():
    import rag_hip
    dev = _dev()
    inv = rag_hip.rope_inv_freq(32)
    q, k, v = _call(torch.zeros((0, 96), device=dev), torch.zeros(0, dtype=torch.int32, device=dev), inv, 1, 1, None, None, False)
    assert q.shape == (0, 1, 32) and k.shape == (0, 1, 32) and v.shape == (0, 1, 32)
    qkv, pos = torch.zeros((4, 96), device=dev), torch.zeros(4, dtype=torch.int32, device=dev)
    for bad in (dict(pos=pos.long()), dict(pos=pos[:3]), dict(inv_freq=inv.float()), dict(qkv=qkv.double()), dict(qkv=qkv.t()),
                dict(n_kv_heads=0), dict(n_q_heads=3), dict(gamma_q=torch.ones(31, device=dev)), dict(v_out=qkv.view(4, 3, 32)[:, :1]),
                dict(k_out=torch.zeros((3, 1, 32), device=dev)), dict(qkv=qkv.cpu()), dict(pos=pos.cpu()),
                dict(kv_row=torch.zeros(4, dtype=torch.int64, device=dev)), dict(gamma_q=torch.ones(32, device=dev).half())):
        kw = dict(qkv=qkv, pos=pos, inv_freq=inv, n_q_heads=1, n_kv_heads=1)
        kw.update(bad)
        with pytest.raises(ValueError):
            rag_hip.enc_qk_norm_rope_dev(**kw)
    with pytest.raises(rag_hip.RagHipError):                   # head size 48
        rag_hip.enc_qk_norm_rope_dev(torch.zeros((4, 144), device=dev), pos, inv, 1, 1)
    with pytest.raises(rag_hip.RagHipError):                   # rotation over 12 dimensions
        rag_hip.enc_qk_norm_rope_dev(qkv, pos, rag_hip.rope_inv_freq(12), 1, 1)
    with pytest.raises(rag_hip.RagHipError):                   # rotation wider than the head
        rag_hip.enc_qk_norm_rope_dev(qkv, pos, rag_hip.rope_inv_freq(64), 1, 1)
    with pytest.raises(rag_hip.RagHipError):                   # misaligned rows
        rag_hip.enc_qk_norm_rope_dev(torch.zeros((4, 97), device=dev)[:, 1:], pos, inv, 1, 1)


def test_another_stream_and_a_replayed_graph():
    import rag_hip
    g = _gen(5)
    t, hq, hkv, d = 50, 8, 2, 128
    qkv = torch.randn((t, (hq + 2 * hkv) * d), generator=g, device=_dev()).to(torch.bfloat16)
    pos = torch.arange(t, dtype=torch.int32, device=_dev())
    inv, gq = rag_hip.rope_inv_freq(d), torch.ones(d, dtype=torch.bfloat16, device=_dev())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q1, k1, _ = _call(qkv, pos, inv, hq, hkv, gq, gq, False)
    torch.cuda.current_stream().wait_stream(side)
    q0, k0, _ = _call(qkv, pos, inv, hq, hkv, gq, gq, False)
    assert torch.equal(q0, q1) and torch.equal(k0, k1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q2, k2, _ = _call(qkv, pos, inv, hq, hkv, gq, gq, False)
    for i in range(4):
        qkv.copy_(torch.randn(qkv.shape, generator=g, device=_dev()))
        pos.add_(1000)
        graph.replay()
        torch.cuda.synchronize()
        q0, k0, _ = _call(qkv, pos, inv, hq, hkv, gq, gq, False)
        assert torch.equal(q0, q2) and torch.equal(k0, k2), i


@pytest.mark.parametrize('kind', list(TYPES))
@pytest.mark.parametrize('t,hq,hkv,d,rot,inter,norm', [
    (5000, 13, 4, 128, 128, False, True), (4999, 5, 3, 64, 40, True, True), (4400, 17, 16, 32, 32, False, False), (4097, 1, 1, 32, 16, True, True),
    (4096, 1, 1, 32, 16, False, True),
    (8192, 1, 1, 32, 24, False, True), (8193, 1, 1, 32, 24, False, True)])
def test_many_tokens(kind, t, hq, hkv, d, rot, inter, norm):
    # more waves than a lane with one head each would have on the chip: four heads a lane, heads that end inside its four
    import rag_hip
    g, dt = _gen(t + d), TYPES[kind]
    qkv = torch.randn((t, (hq + 2 * hkv) * d), generator=g, device=_dev()).to(dt)
    pos = torch.randint(0, 1 << 17, (t,), generator=g, device=_dev(), dtype=torch.int32)
    inv = rag_hip.rope_inv_freq(rot)
    gq, gk = ((1 + 0.3 * torch.randn(d, generator=g, device=_dev())).to(dt) if norm else None for _ in range(2))
    x = qkv.clone().view(t, hq + 2 * hkv, d)
    rows = torch.randperm(t + 9, generator=g, device=_dev())[:t].to(torch.int64)
    rows[5::7] = -1
    k_out, v_out = (torch.full((t + 9, hkv, d), 3.0, dtype=dt, device=_dev()) for _ in range(2))
    q, _, _ = _call(qkv, pos, inv, hq, hkv, gq, gk, inter, k_out=k_out, v_out=v_out, kv_row=rows)
    kept = rows >= 0
    k_ref, k_mag = _ref(x[:, hq:hq + hkv], pos, inv, gk, 1e-6, inter)
    _close(q, *_ref(x[:, :hq], pos, inv, gq, 1e-6, inter))
    _close(k_out[rows[kept]], k_ref[kept], k_mag[kept])
    assert torch.equal(v_out[rows[kept]], x[:, hq + hkv:][kept])
    other = torch.ones(t + 9, dtype=torch.bool, device=_dev())
    other[rows[kept]] = False
    assert bool((k_out[other] == 3.0).all()) and bool((v_out[other] == 3.0).all())
    # in place
    heads = qkv.view(t, hq + 2 * hkv, d)
    _call(qkv, pos, inv, hq, hkv, gq, gk, inter, q_out=heads[:, :hq], k_out=heads[:, hq:hq + hkv])
    assert torch.equal(heads[:, :hq], q) and torch.equal(heads[:, hq:hq + hkv][kept], k_out[rows[kept]])
    assert torch.equal(heads[:, hq + hkv:], x[:, hq + hkv:])


@pytest.mark.parametrize('kind', list(TYPES))
@pytest.mark.parametrize('inter', [False, True])
@pytest.mark.parametrize('t,d,rot', [(3, 32, 0), (3, 64, 24), (9000, 128, 64), (9000, 32, 8), (2, 128, 0)])
def test_an_infinity_outside_the_rotation_stays_where_it_is(kind, inter, t, d, rot):
    # without a norm, dimensions from rot_dim on are copied: what one of them holds does not reach another
    import rag_hip
    dt, hq, hkv = TYPES[kind], 3, 2
    qkv = torch.randn((t, (hq + 2 * hkv) * d), generator=_gen(d + rot), device=_dev()).to(dt)
    pos = torch.arange(t, dtype=torch.int32, device=_dev())
    inv = rag_hip.rope_inv_freq(rot) if rot else None
    want_q, want_k, _ = _call(qkv, pos, inv, hq, hkv, None, None, inter)
    bad = qkv.clone().view(t, hq + 2 * hkv, d)
    for i, x in enumerate((float('inf'), float('nan'), -float('inf'))):
        bad[i % t, i % hq, rot + (5 + 3 * i) % (d - rot)] = x          # one dimension of a query head each,
        bad[(i + 1) % t, hq + i % hkv, rot + 2 * i] = x                 # of a key head,
        bad[t - 1, :hq + hkv, d - 1 - i] = x                            # and the last ones of all
    q, k, _ = _call(bad.view(t, -1), pos, inv, hq, hkv, None, None, inter)
    for got, want, x in ((q, want_q, bad[:, :hq]), (k, want_k, bad[:, hq:hq + hkv])):
        assert torch.equal(got[..., :rot], want[..., :rot])
        torch.testing.assert_close(got[..., rot:], x[..., rot:], rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize('kind', list(TYPES))
@pytest.mark.parametrize('inter', [False, True])
def test_an_infinity_under_the_norm(kind, inter):
    # x / inf: the head's finite dimensions become 0, the infinite one infinity / infinity; rotated, it takes its pair with it
    import rag_hip
    dt, t, d, rot = TYPES[kind], 2, 64, 16
    qkv = torch.randn((t, 3 * d), generator=_gen(1), device=_dev()).to(dt)
    qkv[0, 40] = float('inf')
    qkv[1, 3] = -float('inf')
    ones = torch.ones(d, dtype=dt, device=_dev())
    q, _, _ = _call(qkv, torch.arange(1, 3, dtype=torch.int32, device=_dev()), rag_hip.rope_inv_freq(rot), 1, 1, ones, ones, inter)
    nan = torch.zeros((t, d), dtype=torch.bool, device=_dev())
    nan[0, 40] = nan[1, 3] = nan[1, 2 if inter else 3 + rot // 2] = True
    assert torch.equal(torch.isnan(q[:, 0]), nan) and float(q[:, 0][~nan].abs().max()) == 0.0


def test_rows_beyond_32_bits():
    """The first and last tokens of a projection of more than 2^32 elements."""
    import rag_hip
    t, d, n = (1 << 32) // 96 + 2000, 32, 1000
    qkv = torch.zeros((t, 3 * d), dtype=torch.bfloat16, device=_dev())
    for part in (slice(0, n), slice(t - n, t)):
        qkv[part] = torch.randn((n, 3 * d), generator=_gen(4), device=_dev()).to(torch.bfloat16)
    pos = torch.arange(t, dtype=torch.int32, device=_dev())
    inv = rag_hip.rope_inv_freq(d)
    q, k, v = _call(qkv, pos, inv, 1, 1, None, None, False)
    for part in (slice(0, n), slice(t - n, t)):
        x = qkv[part].view(n, 3, d)
        _close(q[part], *_ref(x[:, :1], pos[part], inv, None, 1e-6, False))
        _close(k[part], *_ref(x[:, 1:2], pos[part], inv, None, 1e-6, False))
        assert torch.equal(v[part], x[:, 2:])
    assert float(q[n:t - n].abs().max()) == 0.0
