"""GPU: products with 4-bit weights (rag_enc_linear4_dev) against the same product in 64 bits, and the quantiser's codes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}


def _dev():
    return torch.device('cuda:0')


def _operands(m, n, k, group, offsets, dt, seed):
    g = torch.Generator(device=_dev()).manual_seed(seed)
    x = torch.randn((m, k), generator=g, device=_dev()).to(dt)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device=_dev(), dtype=torch.uint8)
    scales = (0.05 * (0.2 + torch.rand((n, k // group), generator=g, device=_dev()))).to(dt)
    off = (0.3 * torch.randn((n, k // group), generator=g, device=_dev())).to(dt) if offsets else None
    bias = torch.randn((n,), generator=g, device=_dev()).to(dt)
    return x, codes, scales, off, bias


def _weights(codes, scales, off):
    n, k = codes.shape[0], codes.shape[1] * 2
    c = torch.stack([codes & 15, codes >> 4], dim=2).reshape(n, k).double()
    s = scales.double().repeat_interleave(k // scales.shape[1], dim=1)
    o = off.double().repeat_interleave(k // scales.shape[1], dim=1) if off is not None else -8 * s
    return c, s, o


def _check(y, x, codes, scales, off, bias):
    c, s, o = _weights(codes, scales, off)
    ref = x.double() @ (c * s + o).t()
    if bias is not None:
        ref = ref + bias.double()
    # 32-bit sums of the codes' and the offsets' products (a code may be summed with 16 added to it and taken off again
    # with the offset): at most k + 16 roundings of the magnitudes added up; then one rounding to the result's type
    mag = x.double().abs() @ ((c + 16) * s + (o - 16 * s).abs()).t() + (bias.double().abs() if bias is not None else 0)
    work = (x.shape[1] + 16) * 2.0 ** -24 * mag
    info = torch.finfo(y.dtype)
    step = 0.0 if y.dtype == torch.float32 else info.eps / 2
    tol = work + step * (ref.abs() + work) + info.smallest_normal * info.eps / 2
    err = (y.double() - ref).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


SIZES = [(1, 1, 32, 32), (1, 16, 128, 128), (1, 1152, 384, 64), (2, 17, 96, 32), (5, 383, 416, 32), (15, 100, 64, 64), (16, 64, 640, 128),
         (17, 65, 192, 64), (33, 31, 1024, 32), (48, 200, 256, 32), (63, 129, 384, 128), (64, 384, 1536, 64), (65, 50, 160, 32), (200, 33, 128, 32), (1, 4096, 4096, 128),
         (3, 77, 8192, 32), (9, 4111, 2048, 64)]


@pytest.mark.parametrize('kind', list(TYPES))
@pytest.mark.parametrize('m,n,k,group', SIZES)
def test_matches_64_bits(kind, m, n, k, group):
    import rag_hip
    x, codes, scales, off, bias = _operands(m, n, k, group, True, TYPES[kind], m + n + k)
    _check(rag_hip.enc_linear4_dev(x, codes, scales, off, bias), x, codes, scales, off, bias)
    _check(rag_hip.enc_linear4_dev(x, codes, scales), x, codes, scales, None, None)


def test_rows_of_x_do_not_mix_and_strides():
    import rag_hip
    x, codes, scales, off, bias = _operands(20, 50, 256, 64, True, torch.bfloat16, 4)
    want = rag_hip.enc_linear4_dev(x, codes, scales, off, bias)
    wide = torch.full((20, 512), float('nan'), dtype=torch.bfloat16, device=_dev())
    wide[:, 128:384] = x
    out = torch.full((22, 70), 7.0, dtype=torch.bfloat16, device=_dev())
    got = rag_hip.enc_linear4_dev(wide[:, 128:384], codes, scales, off, bias, out=out[:20, 3:53])
    assert torch.equal(got, want)
    assert bool((out[20:] == 7).all()) and bool((out[:, :3] == 7).all()) and bool((out[:, 53:] == 7).all())
    bad = x.clone()
    bad[3] = float('nan')
    bad[17, 5] = float('inf')
    got = rag_hip.enc_linear4_dev(bad, codes, scales, off, bias)
    keep = [i for i in range(20) if i not in (3, 17)]
    assert torch.equal(got[keep], want[keep])
    assert bool(torch.isnan(got[3]).all()) and not bool(torch.isfinite(got[17]).any())


def test_large_and_small_activations():
    import rag_hip
    x, codes, scales, off, bias = _operands(4, 40, 512, 32, True, torch.float32, 9)
    x[0] *= 1e20
    x[1] *= 1e-20
    x[2, ::2] *= 1e4
    _check(rag_hip.enc_linear4_dev(x, codes, scales, off), x, codes, scales, off, None)


@pytest.mark.parametrize('symmetric', [False, True])
@pytest.mark.parametrize('kind', list(TYPES))
def test_quantised_weights(kind, symmetric):
    import rag_hip
    dt = TYPES[kind]
    g = torch.Generator(device=_dev()).manual_seed(2)
    w = (torch.randn((70, 256), generator=g, device=_dev()) / 16).to(dt)
    w[5, 64:128] = 0.25                                         # a constant group: scale 0 without `symmetric`
    w[6] = 0
    codes, scales, off = rag_hip.quantize4(w, 64, symmetric=symmetric)
    assert (off is None) == symmetric and scales.dtype == dt
    c, s, o = _weights(codes, scales, off)
    # half a step inside the range; the ends may lie outside it by the rounding of the scale (15 steps) and the offset
    eps = torch.finfo(dt).eps / 2
    tol = s * (0.5 + 16 * 2 * eps) + o.abs() * eps * 2 + 1e-6 * w.double().abs() + torch.finfo(dt).smallest_normal
    assert bool(((c * s + o - w.double()).abs() <= tol).all())
    x = torch.randn((3, 256), generator=g, device=_dev()).to(dt)
    _check(rag_hip.enc_linear4_dev(x, codes, scales, off), x, codes, scales, off, None)


def test_refusals_and_no_rows():
    import rag_hip
    x, codes, scales, off, bias = _operands(2, 8, 128, 64, True, torch.bfloat16, 1)
    assert rag_hip.enc_linear4_dev(x[:0], codes, scales, off, bias).shape == (0, 8)
    for bad in (dict(x=x.double()), dict(x=x[:, :64]), dict(x=x.t()), dict(scales=scales.float()), dict(codes=codes.view(torch.int8)), dict(offsets=off[:, :1]),
                dict(bias=bias[:3]), dict(x=x.cpu()), dict(codes=codes.cpu()), dict(scales=scales[:4]), dict(codes=codes.t().contiguous().t()),
                dict(out=torch.zeros((2, 9), dtype=torch.bfloat16, device=_dev())), dict(out=torch.zeros((2, 8), device=_dev()))):
        kw = dict(x=x, codes=codes, scales=scales, offsets=off, bias=bias)
        kw.update(bad)
        with pytest.raises(ValueError):
            rag_hip.enc_linear4_dev(**kw)
    with pytest.raises(rag_hip.RagHipError):                   # group 16
        rag_hip.enc_linear4_dev(x, codes, scales.repeat(1, 4), None, bias)
    with pytest.raises(rag_hip.RagHipError):                   # misaligned rows of x
        rag_hip.enc_linear4_dev(torch.zeros((2, 129), dtype=torch.bfloat16, device=_dev())[:, 1:], codes, scales)


def test_another_stream_and_a_replayed_graph():
    import rag_hip
    x, codes, scales, off, bias = _operands(13, 500, 2048, 128, True, torch.float16, 6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y1 = rag_hip.enc_linear4_dev(x, codes, scales, off, bias)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y1, rag_hip.enc_linear4_dev(x, codes, scales, off, bias))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y2 = rag_hip.enc_linear4_dev(x, codes, scales, off, bias)
    for i in range(4):
        x.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y2, rag_hip.enc_linear4_dev(x, codes, scales, off, bias)), i


def test_weights_beyond_the_interface_are_refused():
    import rag_hip
    x = torch.zeros((1, 32), device='cuda')
    with pytest.raises(ValueError, match='2\\^31'):
        rag_hip.enc_linear4_dev(x, torch.zeros((1, 16), dtype=torch.uint8, device='cuda').expand(1 << 32, 16), torch.zeros((1, 1), device='cuda').expand(1 << 32, 1))


def test_first_calls_of_many_threads():
    # what the wrapper keeps of torch is set once, whichever thread comes first
    import threading
    import rag_hip
    x, codes, scales, off, _ = _operands(3, 64, 128, 32, True, torch.float32, 5)
    want = rag_hip.enc_linear4_dev(x, codes, scales, off)
    torch.cuda.synchronize()
    for _ in range(5):
        rag_hip._current, got, start = None, [None] * 8, threading.Barrier(8)

        def run(i):
            start.wait()
            got[i] = rag_hip.enc_linear4_dev(x, codes, scales, off)
        threads = [threading.Thread(target=run, args=(i,)) for i in range(8)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert all(y is not None and torch.equal(y, want) for y in got)


# every tile of the kernel, x as operands and by rows
LARGE = [(1, 40, 128, 128), (3, 17, 1024, 128), (13, 600, 640, 128), (2, 5000, 256, 64), (13, 5000, 256, 32), (40, 5000, 384, 64), (64, 384, 1536, 128),
         (200, 5000, 256, 128)]


@pytest.mark.parametrize('kind', ['bf16', 'f32'])
@pytest.mark.parametrize('m,n,k,group', LARGE)
@pytest.mark.parametrize('offsets', [False, True])
def test_finite_products_of_large_values(kind, m, n, k, group, offsets):
    # x of 1e37 and weights of some thousandths: the sum of all magnitudes stays below 1e38, while x times a code of 24 does not
    import rag_hip
    x, codes, scales, off, bias = _operands(m, n, k, group, offsets, TYPES[kind], m + k)
    want = rag_hip.enc_linear4_dev(x, codes, scales * 0.01, off * 0.01 if offsets else None, bias)
    large = list(range(0, m, 3))
    x[large] *= 1e37
    scales, off = scales * 0.01, off * 0.01 if offsets else None
    c, s, o = _weights(codes, scales, off)
    assert float((x.double().abs() @ (c * s + o).abs().t()).max()) < 2e38
    y = rag_hip.enc_linear4_dev(x, codes, scales, off, bias)
    assert bool(torch.isfinite(y).all())
    _check(y, x, codes, scales, off, bias)
    rest = [i for i in range(m) if i % 3]
    assert torch.equal(y[rest], want[rest])


@pytest.mark.parametrize('kind', ['bf16', 'f32'])
@pytest.mark.parametrize('offsets', [False, True])
def test_finite_products_of_large_scales(kind, offsets):
    # weights up to 2e38, whose scale times 24, or offset minus 16 scales, is beyond the type
    import rag_hip
    x, codes, scales, off, bias = _operands(5, 70, 256, 64, offsets, TYPES[kind], 3)
    x, scales = x * 1e-4, scales * 2e38 * 2
    if offsets:
        off = off * 0.5e38 - 8 * scales
    c, s, o = _weights(codes, scales, off)
    assert float((c * s + o).abs().max()) < 3e38
    y = rag_hip.enc_linear4_dev(x, codes, scales, off, bias)
    assert bool(torch.isfinite(y).all())
    _check(y, x, codes, scales, off, bias)


@pytest.mark.parametrize('m,n,k,group', [(1, 1152, 384, 64), (16, 300, 256, 32), (40, 5000, 1024, 64), (3, 500, 4096, 128), (200, 129, 640, 128), (9, 4111, 8192, 32)])
@pytest.mark.parametrize('offsets', [False, True])
def test_float32_keeps_24_bits_of_x(m, n, k, group, offsets):
    # The worst-case tolerance above is too wide to tell 24 bits of x from 16, so the root-mean-square error is held to the root
    # of the summed squares of what is added up (x times code + 16, x times the offset less 16 scales).  In half steps of that,
    # 2^-24: a sum over 32 columns is at most some 36 roundings, each uniform (1 / sqrt(3)), 3.5, and again as many of the
    # offsets' part, which is two thirds as large; two multiply-adds into a sum that grows over up to 64 steps: 4.6; together below
    # 6.5.  One part of x less leaves 22 to 79 (computed with the parts in 64 bits at these sizes), two less over 7000.
    import rag_hip
    x, codes, scales, off, _ = _operands(m, n, k, group, offsets, torch.float32, 3 * m + k)
    c, s, o = _weights(codes, scales, off)
    err = rag_hip.enc_linear4_dev(x, codes, scales, off).double() - x.double() @ (c * s + o).t()
    square = x.double() ** 2 @ (((c + 16) * s) ** 2 + (o - 16 * s) ** 2).t()
    assert float(err.pow(2).mean().sqrt()) <= 8 * 2.0 ** -24 * float(square.mean().sqrt())


@pytest.mark.parametrize('m', [1, 13])
def test_weights_beyond_32_bits(m):
    """The first and last rows of weights of more than 2^32 bytes."""
    import rag_hip
    n, k, group, part = (1 << 20) + 77, 8192, 128, 300
    x, some, scales, off, bias = _operands(m, 2 * part, k, group, True, torch.bfloat16, m)
    codes = torch.zeros((n, k // 2), dtype=torch.uint8, device=_dev())
    s, o = (torch.zeros((n, k // group), dtype=torch.bfloat16, device=_dev()) for _ in range(2))
    b = torch.zeros((n,), dtype=torch.bfloat16, device=_dev())
    for to, at in ((slice(0, part), slice(0, part)), (slice(n - part, n), slice(part, 2 * part))):
        codes[to], s[to], o[to], b[to] = some[at], scales[at], off[at], bias[at]
    y = rag_hip.enc_linear4_dev(x, codes, s, o, b)
    _check(torch.cat([y[:, :part], y[:, n - part:]], dim=1), x, some, scales, off, bias)
    assert float(y[:, part:n - part].abs().max()) == 0.0


def test_two_million_rows():
    import rag_hip
    m = 2097120                                                 # the most that a launch takes
    x, codes, scales, off, bias = _operands(m, 3, 32, 32, True, torch.bfloat16, 2)
    y = rag_hip.enc_linear4_dev(x, codes, scales, off, bias)
    for part in (slice(0, 5000), slice(m - 5000, m)):
        _check(y[part], x[part], codes, scales, off, bias)
    with pytest.raises(rag_hip.RagHipError, match='too many rows'):
        rag_hip.enc_linear4_dev(torch.cat([x, x[:1]]), codes, scales, off, bias)
