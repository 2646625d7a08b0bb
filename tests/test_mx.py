"""Microscaled 4-bit floating point (vhap_amd.mx) against its definitions in 64 bits, code by code where numbers become codes.

Tolerances of the products: products of codes with anything are exact (an fp32 operand is exactly three bf16 pieces), so what rounds is the fp32 sum -- an addition in
the matrix instruction may cut off instead of rounding, 2^-23 each -- of K products (times the pieces), in any order: at most (K P + 4) 2^-23 of the sum of their
magnitudes; the split sums of an input gradient add one addition a split; and the result is rounded to its type once."""
import ctypes
import math

import pytest
import torch

from vhap_amd import _lib, mx

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
PIECES = {torch.float32: 3, torch.float16: 2, torch.bfloat16: 1}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
MAGNITUDES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def randn(shape, seed, dtype=torch.float32, device="cuda"):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)


def random_mx(rows, k, seed, device="cuda", lo=118, hi=130, garbage=False):
    """random codes and scales; `garbage`: the codes behind k are anything"""
    g = torch.Generator().manual_seed(seed)
    kb = -(-k // 32)
    codes = torch.randint(0, 256, (rows, 16 * kb), generator=g, dtype=torch.uint8)
    if not garbage:
        at = torch.arange(16 * kb) * 2
        codes &= torch.where(at + 1 < k, 255, torch.where(at < k, 15, 0)).to(torch.uint8)
    return mx.MXTensor(codes.to(device), torch.randint(lo, hi, (rows, kb), generator=g, dtype=torch.uint8).to(device), (rows, k))


def values64(t):
    """the numbers an MXTensor stands for, from the table of codes"""
    codes, scales, k = t.codes.cpu().long(), t.scales.cpu(), t.shape[-1]
    table = torch.tensor(MAGNITUDES + [-v for v in MAGNITUDES], dtype=torch.float64)
    pair = torch.stack([codes % 16, codes // 16], -1).flatten(-2)
    s = torch.tensor([2.0 ** (b - 127) if b < 255 else math.nan for b in range(256)], dtype=torch.float64)[scales.long()]
    return (table[pair] * s.repeat_interleave(32, -1))[..., :k]


def quantize64(x):
    """-> (values, scale bytes) of a [rows, K] matrix by search over the eight magnitudes"""
    x = x.detach().cpu().double()
    rows, k = x.shape
    kb = -(-k // 32)
    x = torch.nn.functional.pad(x, (0, 32 * kb - k)).view(rows, kb, 32)
    most = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    byte = torch.zeros(rows, kb, dtype=torch.long)
    for i in range(rows):
        for j in range(kb):
            m = float(most[i, j])
            byte[i, j] = 255 if bool(bad[i, j]) else max(0, math.frexp(m)[1] - 1 - 2 + 127) if m > 0 else 0
    scale = torch.tensor([2.0 ** (b - 127) for b in range(256)], dtype=torch.float64)[byte][..., None]
    v = (x / scale).abs()
    best, far = torch.zeros_like(v), torch.full_like(v, math.inf)
    for code in (0, 2, 4, 6, 1, 3, 5, 7):                                       # the even codes first: a tie stays theirs
        d = (v - MAGNITUDES[code]).abs()
        best, far = torch.where(d < far, MAGNITUDES[code], best), torch.minimum(d, far)
    out = torch.where(torch.signbit(x), -best, best) * scale
    out[bad] = math.nan
    return out.view(rows, -1)[:, :k], byte


def same(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a, nan=0.0, posinf=math.inf, neginf=-math.inf),
                                                                       torch.nan_to_num(b, nan=0.0, posinf=math.inf, neginf=-math.inf))


def check_sum(got, want, mags, adds, dtype):
    """`want` the exact sums, `mags` the sums of the magnitudes"""
    off = (got.detach().cpu().double() - want).abs()
    limit = (adds + 4) * 2.0 ** -23 * mags
    limit = limit * (1 + HALF[dtype]) + HALF[dtype] * want.abs() + TINY[dtype]
    worst = float((off / limit.clamp(min=1e-300)).max()) if off.numel() else 0.0
    assert bool((off <= limit).all()), (worst, float(off.max()))


# ---- host ----
def test_refusals_on_the_host():
    x = torch.ones(4, 40)
    w = random_mx(4, 40, 1, "cpu")
    for call in (lambda: mx.quantize(x), lambda: mx.linear(x, w), lambda: mx.linear_input_grad(torch.ones(4, 4), w), lambda: mx.matmul(w, w)):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()
    for call in (lambda: mx.quantize(x.double()), lambda: mx.linear(x.int(), w), lambda: mx.linear(x, x), lambda: mx.matmul(w, x), lambda: w.dequantize(torch.float64),
                 lambda: mx.MXTensor(w.codes.int(), w.scales, (4, 40))):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: mx.MXTensor(w.codes, w.scales, (4, 65)), lambda: mx.MXTensor(w.codes, w.scales, (2, 2, 40)), lambda: mx.MXTensor(w.codes, w.scales, (4, 0)),
                 lambda: mx.MXTensor(w.codes, w.scales, ()), lambda: mx.MXTensor(w.codes.t().contiguous().t(), w.scales, (4, 40)),
                 lambda: mx.MXTensor(torch.zeros(129, dtype=torch.uint8)[1:].view(4, 32), w.scales, (4, 40))):
        with pytest.raises(ValueError):
            call()
    assert w.nbytes() == 4 * 34 and w.rows == 4


def test_dequantize_on_the_host_is_the_definition():
    w = random_mx(5, 77, 3, "cpu", 0, 256)
    assert same(w.dequantize(torch.float32).double(), values64(w).float().double())


def test_c_entry_refusals():
    L, P = _lib.lib(), 1 << 30
    assert L.vhap_mx4_quantize(P, 3, 32, 1, 32, P, P, 0) == _lib.E_BADDIM
    assert L.vhap_mx4_quantize(P, 0, 32, -1, 32, P, P, 0) == _lib.E_BADDIM
    assert L.vhap_mx4_quantize(P, 0, 32, 1, 0, P, P, 0) == _lib.E_BADDIM
    assert L.vhap_mx4_quantize(P, 0, 32, 1, (1 << 24) + 1, P, P, 0) == _lib.E_BADDIM
    assert L.vhap_mx4_quantize(0, 0, 32, 1, 32, P, P, 0) == _lib.E_NULLPTR
    assert L.vhap_mx4_quantize(0, 0, 32, 0, 32, 0, 0, 0) == 0
    assert L.vhap_mx4_dequantize(0, P, 1, 32, P, 0, 0) == _lib.E_NULLPTR
    assert L.vhap_mx4_linear(P, 0, -1, 1, P, P, 1, 32, 0, P, 0) == _lib.E_BADDIM
    assert L.vhap_mx4_linear(P, 0, 32, 1, P, P, 1, 32, 0, 0, 0) == _lib.E_NULLPTR
    assert L.vhap_mx4_linear(0, 0, 32, 0, 0, 0, 1, 32, 0, 0, 0) == 0
    assert L.vhap_mx4_linear_input_grad(P, 0, 32, 1, P, P, 32, 32, P, 0, P, 0, 0) == _lib.E_WORKSPACE
    assert L.vhap_mx4_linear_input_grad(P, 0, 32, 1, P, P, 0, 32, P, 0, P, 0, 0) == _lib.E_BADDIM
    assert L.vhap_mx4_linear_input_grad(P, 1, 32, 1, P, P, 32, 32, P, 1 << 30, P, _lib.CALL_MX_ACCUMULATE, 0) == _lib.E_UNSUPPORTED
    assert L.vhap_mx4_linear_input_grad(P, 0, 32, 1, P, P, 32, 32, 0, 1 << 30, P, 0, 0) == _lib.E_NULLPTR
    assert L.vhap_mx4_matmul(P, P, 1, P, P, 1, 32, 0, 0, 0, 0, 0) == _lib.E_NULLPTR
    assert L.vhap_mx4_matmul(P, P, 1 << 40, P, P, 1, 32, 0, P, 0, 0, 0) == _lib.E_BADDIM
    assert L.vhap_mx4_column_sums(P, 0, 1, 1, 1, 0, 0) == _lib.E_NULLPTR


# ---- quantise ----
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (5, 32), (2, 33), (7, 100), (1, 257), (64, 128), (33, 1000)])
def test_quantize(shape, dtype):
    x = (randn(shape, 1, torch.float32, "cpu") * torch.exp(2 * randn((shape[0], 1), 2, device="cpu"))).to(dtype)
    x[-1] = 0
    want, byte = quantize64(x)
    q = mx.quantize(x.cuda())
    assert torch.equal(q.scales.cpu().long(), byte) and q.shape == x.shape
    assert torch.equal(values64(q), want) and torch.equal(torch.signbit(values64(q)), torch.signbit(x.double()))
    pad = torch.stack([q.codes & 15, q.codes >> 4], -1).flatten(-2)[:, shape[1]:]
    assert not bool(pad.any())                                                   # zeros behind the last element
    for dt in (torch.float32, torch.bfloat16):
        assert torch.equal(q.dequantize(dt).cpu().double(), want)
    assert torch.equal(q.dequantize(torch.float16).cpu(), want.to(torch.float16))


@pytest.mark.gpu
def test_quantize_borders_and_extremes():
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0]
    rows = []
    for s in (1.0, 2.0 ** -126, 2.0 ** -130, 2.0 ** -149, 2.0 ** 100, 2.0 ** 125):
        for lift in (-1, 0, 1):                                                  # on the border, a last place below and above
            v = torch.tensor(ties + [4.0] * 8, dtype=torch.float32) * torch.tensor(s, dtype=torch.float32)
            if lift:
                v = torch.nextafter(v, torch.full_like(v, math.inf if lift > 0 else 0.0))
            rows.append(torch.cat([v, -v]))
    x = torch.stack(rows)
    x[x.isinf()] = 3.4028234663852886e38
    x = torch.cat([x, torch.zeros(1, 32), -torch.zeros(1, 32)])
    want, byte = quantize64(x)
    q = mx.quantize(x.cuda())
    assert torch.equal(q.scales.cpu().long(), byte)
    assert torch.equal(values64(q), want)
    assert same(q.dequantize().cpu().double(), want.float().double())
    bad = randn((6, 96), 4, device="cpu")
    for i, v in enumerate((math.nan, math.inf, -math.inf)):
        bad[i, 40 + i] = v
    q = mx.quantize(bad.cuda())
    assert (q.scales[:3, 1] == 255).all() and not (q.scales == 255)[3:].any() and not (q.scales == 255)[:, 0].any()
    assert same(q.dequantize().cpu().double(), quantize64(bad)[0])


@pytest.mark.gpu
def test_quantize_shapes_and_strides():
    x = randn((4, 6, 70), 5)
    q = mx.quantize(x)
    assert q.shape == x.shape and q.codes.shape == (4, 6, 48) and q.scales.shape == (4, 6, 3)
    flat = mx.quantize(x.reshape(-1, 70))
    assert torch.equal(q.codes.view(24, 48), flat.codes)
    for view in (x[:, :, 3:40], x.permute(1, 2, 0), x[::2], x[0, 0], x[0, 0, ::2], x[:, :, :1].expand(4, 6, 64)):
        want = mx.quantize(view.contiguous())
        got = mx.quantize(view)
        assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
    e = mx.quantize(torch.empty(0, 40, device="cuda"))
    assert e.codes.shape == (0, 32) and e.dequantize().shape == (0, 40)
    with pytest.raises(ValueError):
        mx.quantize(torch.empty(3, 0, device="cuda"))
    with pytest.raises(ValueError):
        mx.quantize(torch.tensor(1.0, device="cuda"))


# ---- linear ----
LINEAR = [(1, 1, 1), (1, 5, 33), (1, 1000, 100), (5, 65, 128), (6, 64, 129), (8, 130, 300), (16, 257, 512), (17, 63, 31), (16, 500, 513), (33, 129, 100), (65, 300, 400),
          (1, 500, 1024), (16, 70, 1500), (5, 33, 2049), (3, 4100, 1025), (300, 4000, 130), (17, 100001, 33), (6, 100003, 20),
          (2, 4099, 64), (130, 77, 700), (257, 641, 40), (1, 70001, 100), (3, 20011, 100), (20, 9000, 96)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", LINEAR)
def test_linear_and_gradients(m, n, k, dtype):
    w = random_mx(n, k, m + n + k, garbage=True)
    W = values64(w)
    x = randn((m, k), 1, dtype).requires_grad_()
    bias = randn((n,), 2).requires_grad_()
    g = randn((m, n), 3, dtype)
    y = mx.linear(x, w, bias)
    assert y.dtype == dtype and y.shape == (m, n)
    X, G, P = x.detach().cpu().double(), g.cpu().double(), PIECES[dtype]
    check_sum(y, X @ W.t() + bias.detach().cpu().double(), X.abs() @ W.abs().t() + bias.detach().cpu().double().abs(), k * P + 1, dtype)
    check_sum(mx.linear(x.detach(), w), X @ W.t(), X.abs() @ W.abs().t(), k * P, dtype)
    y.backward(g)
    assert x.grad.dtype == dtype and bias.grad.dtype == torch.float32
    check_sum(x.grad, G @ W, G.abs() @ W.abs(), n * P + 1024, dtype)
    check_sum(bias.grad, G.sum(0), G.abs().sum(0), m, torch.float32)
    assert torch.equal(x.grad, mx.linear_input_grad(g, w))


@pytest.mark.gpu
def test_linear_gradient_against_differences():
    """a linear map's difference quotient is its gradient: L(x + h d) - L(x - h d) = 2 h <grad, d>, in 64-bit sums over fp32 results"""
    w = random_mx(300, 77, 5)
    x, d, g = randn((4, 77), 6), randn((4, 77), 7), randn((4, 300), 8)
    loss = lambda t: float((mx.linear(t, w).double() * g.double()).sum())
    x0 = x.clone().requires_grad_()
    mx.linear(x0, w).backward(g)
    want = float((x0.grad.double() * d.double()).sum())
    got = (loss(x + d) - loss(x - d)) / 2
    scale = float((g.abs().double() @ w.dequantize().double().abs() * (x.abs() + d.abs()).double()).sum())
    assert abs(got - want) <= (77 * 3 + 300 * 3 + 1100) * 2.0 ** -22 * scale


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_shapes_strides_and_empties(dtype):
    w = random_mx(70, 90, 1)
    x = randn((3, 4, 90), 2, dtype)
    want = mx.linear(x.reshape(-1, 90), w)
    assert torch.equal(mx.linear(x, w), want.view(3, 4, 70))
    assert torch.equal(mx.linear(x[1, 2], w), mx.linear(x[1, 2][None], w)[0])
    wide = randn((12, 201), 3, dtype)
    assert torch.equal(mx.linear(wide[:, 7:97], w), mx.linear(wide[:, 7:97].contiguous(), w))
    assert torch.equal(mx.linear(wide.t()[:90].t(), w), mx.linear(wide[:, :90].contiguous(), w))
    assert torch.equal(mx.linear(wide[:1, :90].expand(12, 90), w), mx.linear(wide[:1, :90].repeat(12, 1), w))
    gw = randn((12, 301), 4, dtype)
    for m in (1, 2, 12):
        assert torch.equal(mx.linear_input_grad(gw[:m, 5:75], w), mx.linear_input_grad(gw[:m, 5:75].contiguous(), w))
    x0 = torch.empty(0, 90, dtype=dtype, device="cuda", requires_grad=True)
    y0 = mx.linear(x0, w)
    assert y0.shape == (0, 70)
    y0.sum().backward()
    assert x0.grad.shape == (0, 90)
    none = mx.MXTensor(torch.empty(0, 48, dtype=torch.uint8, device="cuda"), torch.empty(0, 3, dtype=torch.uint8, device="cuda"), (0, 90))
    assert mx.linear(x, none).shape == (3, 4, 0)
    assert not bool(mx.linear_input_grad(torch.empty(5, 0, dtype=dtype, device="cuda"), none).any())
    x1 = x.clone().requires_grad_()
    mx.linear(x1, w).sum().backward()                                            # an expanded gradient
    assert torch.equal(x1.grad, mx.linear_input_grad(torch.ones(3, 4, 70, dtype=dtype, device="cuda"), w))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 4, 20])
def test_linear_with_what_is_not_finite(m):
    w = random_mx(100, 70, 1)
    w.scales[50, 1] = 255                                                        # one block of one row is NaN
    W, x, g = values64(w), randn((m, 70), 2), randn((m, 100), 3)
    y = mx.linear(x, w).cpu()
    assert y[:, 50].isnan().all() and not y[:, :50].isnan().any() and not y[:, 51:].isnan().any()
    dx = mx.linear_input_grad(g, w).cpu()
    assert dx[:, 32:64].isnan().all() and not dx[:, :32].isnan().any() and not dx[:, 64:].isnan().any()
    w = random_mx(100, 70, 4)
    W = values64(w)
    for v in (math.inf, -math.inf, math.nan, 3.4028234663852886e38, 1e-40, -0.0):
        x = randn((m, 70), 5)
        x[0, 9] = v
        want = (x.cpu().double()[:, None, :] * W[None]).sum(-1)
        got = mx.linear(x, w).cpu().double()
        assert torch.equal(got.isnan(), want.isnan()), v
        if abs(v) == math.inf:
            assert torch.equal(got[0].isinf(), want[0].isinf()) and torch.equal(got[0][got[0].isinf()], want[0][want[0].isinf()])
        if m > 1:
            check_sum(got[1:], want[1:], (x[1:].cpu().double()[:, None, :] * W[None]).abs().sum(-1), 70 * 3, torch.float32)
    g = randn((m, 100), 6)
    g[0, 17] = math.inf
    got, want = mx.linear_input_grad(g, w).cpu().double(), (g.cpu().double()[:, :, None] * W[None]).sum(1)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())


@pytest.mark.gpu
def test_linear_refusals():
    w, x = random_mx(70, 90, 1), randn((3, 90), 2)
    for call in (lambda: mx.linear(x[:, :89], w), lambda: mx.linear(x, w, torch.zeros(69, device="cuda")), lambda: mx.linear(x, w, torch.zeros(70, device="cuda").half()),
                 lambda: mx.linear(x, w, torch.zeros(70)), lambda: mx.linear_input_grad(x, w), lambda: mx.linear(x, mx.quantize(x[None]))):
        with pytest.raises(ValueError):
            call()
    x.requires_grad_()
    (d,) = torch.autograd.grad(mx.linear(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()


# ---- matmul ----
MATMUL = [(1, 1, 1), (1, 1, 32), (3, 5, 33), (16, 16, 128), (17, 65, 129), (64, 64, 100), (65, 127, 31), (129, 130, 257), (300, 256, 256), (40, 68, 1000), (2, 513, 64), (1000, 7, 160)]


@pytest.mark.gpu
@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("m,n,k", MATMUL)
def test_matmul(m, n, k, out):
    a, b = random_mx(m, k, 1, garbage=True), random_mx(n, k, 2, garbage=True)
    A, B, bias = values64(a), values64(b), randn((n,), 3)
    mags = A.abs() @ B.abs().t()
    y = mx.matmul(a, b, out_dtype=out)
    assert y.dtype == out and y.shape == (m, n)
    if out != torch.float16 or float(mags.max()) < 6e4:
        check_sum(y, A @ B.t(), mags, k, out)
    want = A @ B.t() + bias.cpu().double()
    mags = mags + bias.abs().cpu().double()
    if out != torch.float16 or float(mags.max()) < 6e4:
        check_sum(mx.matmul(a, b, bias, out_dtype=out), want, mags, k + 1, out)
        check_sum(mx.matmul(a, b, bias, relu=True, out_dtype=out), want.clamp(min=0), mags, k + 1, out)


@pytest.mark.gpu
def test_matmul_extremes_and_refusals():
    a, b = random_mx(40, 100, 1, lo=1, hi=20), random_mx(50, 100, 2, lo=100, hi=120)      # results far below 1
    A, B = values64(a), values64(b)
    check_sum(mx.matmul(a, b), A @ B.t(), A.abs() @ B.abs().t() + 2.0 ** -126, 100, torch.float32)
    a, b = random_mx(40, 100, 3), random_mx(50, 100, 4)
    a.scales[7, 2] = 255
    y = mx.matmul(a, b, relu=True)
    assert y[7].isnan().all() and not y[:7].isnan().any() and not y[8:].isnan().any()
    b.scales[3, 0] = 255
    y = mx.matmul(a, b)
    assert y[:, 3].isnan().all() and not y[:7, 4:].isnan().any()
    none = mx.MXTensor(torch.empty(0, 64, dtype=torch.uint8, device="cuda"), torch.empty(0, 4, dtype=torch.uint8, device="cuda"), (0, 100))
    assert mx.matmul(none, b).shape == (0, 50) and mx.matmul(a, none).shape == (40, 0)
    with pytest.raises(ValueError):
        mx.matmul(a, random_mx(5, 99, 1))
    with pytest.raises(ValueError):
        mx.matmul(a, mx.quantize(randn((2, 5, 100), 1)))
    with pytest.raises(ValueError):
        mx.matmul(a, b, torch.zeros(49, device="cuda"))
    with pytest.raises(TypeError):
        mx.matmul(a, b, out_dtype=torch.float64)


# ---- as they are used ----
@pytest.mark.gpu
def test_streams_and_captures():
    w = random_mx(5000, 100, 1)
    xs = [randn((1, 100), 2), randn((40, 100), 3)]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        y = mx.linear(xs[0], w)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(y, mx.linear(xs[0], w))

    def chain(x):
        q = mx.quantize(x)
        y = mx.linear(x, w)
        return y, mx.linear_input_grad(y, w), q.dequantize(), mx.matmul(q, w)
    for x in xs:
        chain(x)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(chain(x))
        graphs.append(g)
    for k in range(4):
        for i, x in enumerate(xs):
            x.copy_(randn(x.shape, 50 + 2 * k + i))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for x, out in zip(xs, outs):
            for a, b in zip(out, chain(x)):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_a_code_is_fitted_in_a_4_bit_basis():
    """quantised basis -> linear -> loss -> its gradient -> clipped Adam, as a texture code is fitted: every step's numbers against the same step in 64 bits from
    the same state"""
    from vhap_amd.native import HipAdam
    w = mx.quantize(randn((3000, 50), 1) * 10)
    W, mean = values64(w), randn((3000,), 2)
    target = (torch.randn(50, generator=torch.Generator().manual_seed(3), dtype=torch.float64) @ W.t()).float().cuda() + mean
    code = torch.nn.Parameter(torch.zeros(1, 50, device="cuda"))
    opt = HipAdam([code], lr=0.05, max_grad_norm=1.0)
    for _ in range(4):
        c64 = code.detach().cpu().double()
        y = mx.linear(code, w, mean)
        loss = ((y - target) ** 2).mean()
        opt.zero_grad()
        loss.backward()
        r = c64 @ W.t() + mean.cpu().double() - target.cpu().double()
        want = 2 / 3000 * r @ W
        # r: the sums of 50 products and the difference, then 3000 products of it
        slack = (50 * 3 + 10) * 2.0 ** -23 * (c64.abs() @ W.abs().t() + mean.abs().cpu().double() + target.abs().cpu().double()) @ W.abs() + (9000 + 1030) * 2.0 ** -23 * r.abs() @ W.abs()
        assert bool(((code.grad.cpu().double() - want).abs() <= 2 / 3000 * slack).all())
        opt.step()
        n = float(code.grad.double().norm())
        assert abs(float(opt.grad_norm) - n) <= 1.01 * 2.0 ** -24 * n


def test_a_negated_view_is_refused():
    x = torch.randn(4, 40, dtype=torch.complex64).conj().imag
    w = random_mx(4, 40, 1, "cpu")
    for call in (lambda: mx.quantize(x), lambda: mx.linear(x, w), lambda: mx.linear(torch.ones(4, 40), w, x[:, 0])):
        with pytest.raises((TypeError, RuntimeError)):
            call()
    with pytest.raises(TypeError, match="negated"):
        mx.quantize(x)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m", [1, 4, 20])
def test_linear_with_scales_at_the_ends(m, dtype):
    """the smallest scales (elements down to 2^-128, subnormal in bf16 and fp32) against large numbers, the largest finite ones against small numbers"""
    for lo, hi, times in ((0, 4, 2.0 ** 110), (248, 253, 2.0 ** -90)):
        w = random_mx(70, 200, 1, lo=lo, hi=hi)
        W = values64(w)
        x, g = (randn((m, 200), 2) * times).to(dtype), (randn((m, 70), 3) * times).to(dtype)
        X, G, P = x.cpu().double(), g.cpu().double(), PIECES[dtype]
        check_sum(mx.linear(x, w), X @ W.t(), X.abs() @ W.abs().t(), 200 * P, dtype)
        check_sum(mx.linear_input_grad(g, w), G @ W, G.abs() @ W.abs(), 70 * P + 1024, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("lo,hi", [((0, 3), (252, 255)), ((0, 255), (127, 128)), ((0, 1), (0, 1))])
def test_matmul_with_scales_at_the_ends(lo, hi):
    a, b = random_mx(40, 200, 1, lo=lo[0], hi=lo[1]), random_mx(70, 200, 2, lo=hi[0], hi=hi[1])
    A, B = values64(a), values64(b)
    want, mags = A @ B.t(), A.abs() @ B.abs().t()
    got = mx.matmul(a, b).cpu().double()
    fits = mags < 2.0 ** 126
    off = (got - want).abs()
    assert bool((off <= (204 * 2.0 ** -23) * mags + 2.0 ** -126)[fits].all()) and bool(fits.any())       # (a sum below the normal numbers may be cut off)


@pytest.mark.gpu
def test_gradients_over_many_rows():
    """more tiles of rows than a grid's second or third axis holds"""
    m = 64 * 65536 + 1
    w = random_mx(8, 33, 1)
    g = randn((64, 8), 2, torch.bfloat16).repeat(65537, 1)[:m]
    dx = mx.linear_input_grad(g, w)
    for at in (0, 64 * 40000, m - 65):
        assert torch.equal(dx[at:at + 64], mx.linear_input_grad(g[at:at + 64], w))
    L, n = _lib.lib(), 2 ** 29 + 5                                               # and as many columns
    g = torch.arange(n, device="cuda").remainder(251).to(torch.bfloat16)
    out = torch.empty(n, dtype=torch.float32, device="cuda")
    assert L.vhap_mx4_column_sums(g.data_ptr(), 1, 0, 8, n, out.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(out, g.float() * 8)                                       # (the same row eight times)


@pytest.mark.gpu
def test_a_captured_backward():
    """forward and backward in a capture, replayed against the eager ones; and refused while an eager graph of the same leaf is alive"""
    w, bias = random_mx(300, 90, 1), randn((300,), 2).requires_grad_()
    x, g = randn((5, 90), 3).requires_grad_(), randn((5, 300), 4)
    y = mx.linear(x, w, bias)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="alive"):
        with torch.cuda.graph(graph):
            mx.linear(x, w, bias)
    del y
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = mx.linear(x, w, bias)
        dx, db = torch.autograd.grad(y, (x, bias), g)
    for k in range(3):
        with torch.no_grad():
            x.copy_(randn((5, 90), 10 + k))
            g.copy_(randn((5, 300), 20 + k))
        graph.replay()
        torch.cuda.synchronize()
        x1 = x.detach().clone().requires_grad_()
        y1 = mx.linear(x1, w, bias.detach())
        assert torch.equal(y.detach(), y1.detach()) and torch.equal(dx, torch.autograd.grad(y1, x1, g)[0])
        assert torch.equal(db, torch.autograd.grad(mx.linear(x1, w, b1 := bias.detach().clone().requires_grad_()), b1, g)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("n,k", [(270001, 100), (2 ** 20 + 37, 7), (81000, 401)])
def test_one_row_against_a_large_matrix(n, k):
    w = random_mx(n, k, 1)
    g, x = randn((1, n), 2), randn((1, k), 3)
    W, G, X = w.dequantize().double(), g.double(), x.double()                    # (dequantize is tested above)
    check_sum(mx.linear_input_grad(g, w), (G @ W).cpu(), (G.abs() @ W.abs()).cpu(), n + 1024, torch.float32)
    check_sum(mx.linear(x, w), (X @ W.t()).cpu(), (X.abs() @ W.abs().t()).cpu(), k, torch.float32)
    w.scales[n - 1, 0] = 255                                                     # the last row's first block alone
    dx = mx.linear_input_grad(g, w)
    assert dx[:, :32].isnan().all() and not dx[:, 32:].isnan().any()


@pytest.mark.gpu
def test_inference_mode_and_two_backwards():
    w, x, g = random_mx(90, 70, 1), randn((4, 70), 2), randn((4, 90), 3)
    want = mx.linear(x, w)
    with torch.inference_mode():
        assert torch.equal(mx.linear(x, w), want)
        q = mx.quantize(x)
        y = mx.matmul(q, w)
        assert torch.equal(mx.linear(x.clone(), w), want)
    assert torch.equal(y, mx.matmul(mx.quantize(x), w))
    x1 = x.clone().requires_grad_()
    y = mx.linear(x1, w)
    y.backward(g, retain_graph=True)
    first = x1.grad.clone()
    y.backward(g)
    assert torch.equal(x1.grad, first + first)
    with pytest.raises(RuntimeError):
        y.backward(g)
    y = mx.linear(x1, w)                                                         # W changed between forward and backward: refused
    w.codes.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(g)


@pytest.mark.gpu
def test_threads_and_streams_at_once():
    """two host threads, each with its stream, on one matrix"""
    import threading
    w = random_mx(3000, 100, 1)
    xs = [randn((m, 100), m) for m in (1, 7, 40, 1)]
    want = [(mx.linear(x, w), mx.linear_input_grad(mx.linear(x, w), w)) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(k):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(20):
                x1 = xs[k].clone().requires_grad_()
                y = mx.linear(x1, w)
                y.backward(y.detach())
                if not (torch.equal(y, want[k][0]) and torch.equal(x1.grad, want[k][1])):
                    bad.append(k)
    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(4, 100, 1100), (1, 70, 2050), (40, 300, 200), (2, 40000, 200)])
def test_not_finite_stays_where_it_is(m, n, k, dtype):
    """a NaN block (the last of K, the last row), an infinity in x: only the results they enter"""
    w = random_mx(n, k, 1, lo=124, hi=128)
    w.scales[n - 1, -1] = 255
    x = randn((m, k), 2, dtype)
    y = mx.linear(x, w)
    assert y[:, n - 1].isnan().all() and bool(y[:, :n - 1].isfinite().all())
    x[m - 1, k - 1] = math.inf
    y, last = mx.linear(x, w).cpu(), values64(w)[:, -1]
    assert bool(y[:m - 1, :n - 1].isfinite().all())
    row, last = y[m - 1, :n - 1], last[:n - 1]
    assert bool((row.isnan() == (last == 0)).all())                              # infinity times zero
    assert bool((row[last != 0] == (torch.sign(last[last != 0]) * math.inf).to(dtype)).all())
