"""The global gradient norm, clipping to a largest norm (vhap_amd.native.grad_norm / clip_by_global_norm / clip_grad_norm_) and the Adam step on clipped gradients
(HipAdam(max_grad_norm=)) against their definitions in 64 bits.

Tolerances: the norm is summed in 64 bits and rounded to fp32 once (2^-24); a clipped gradient is rounded twice, the factor to fp32 (2^-24) and the product to its
type (2^-24, bf16 2^-8, fp16 2^-11), plus half of the type's smallest step where the product is subnormal."""
import ctypes
import math

import pytest
import torch

from vhap_amd import _lib
from vhap_amd import native as NV

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def norm64(ts, p):
    x = torch.cat([t.detach().reshape(-1).double().cpu() for t in ts]) if ts else torch.zeros(0, dtype=torch.float64)
    if x.numel() == 0:
        return 0.0
    return float(x.abs().max()) if p == math.inf else float((x.abs() ** p).sum() ** (1.0 / p))


def near_norm(got, want):
    if math.isnan(want) or math.isinf(want):
        return math.isnan(got) if math.isnan(want) else got == want
    return abs(got - want) <= 2.0 ** -24 * 1.001 * want


def check_clipped(got, src, c):
    want = src.detach().double().cpu() * c
    off = (got.detach().double().cpu() - want).abs()
    assert bool((off <= want.abs() * (HALF[src.dtype] + 2.0 ** -24) * 1.001 + TINY[src.dtype]).all()), float(off.max())


def coefficient(norm, max_norm):
    return min(1.0, max_norm / (norm + 1e-6))


def randn(shape, seed, dtype=torch.float32, scale=1.0, device="cuda"):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(device)


LISTS = {
    "one": [((1,), torch.float32)],
    "odd": [((511,), torch.float32), ((513,), torch.bfloat16), ((7, 3), torch.float16), ((), torch.float32)],
    "empty_among": [((0,), torch.float32), ((5,), torch.float32), ((3, 0), torch.bfloat16), ((1000,), torch.float32)],
    "tracker": [((300,), torch.float32), ((16, 100), torch.float32), ((16, 3), torch.float32), ((1,), torch.float32), ((1, 5143, 3), torch.float32), ((3, 257, 255), torch.float32)],
    "one_block_border": [((32768,), torch.float32)],
    "past_one_block": [((32769,), torch.float32)],
    "one_block_border_16": [((65536,), torch.bfloat16)],
    "past_one_block_16": [((65535,), torch.float16), ((1,), torch.bfloat16)],
    "large_mixed": [((1 << 20,), torch.float32), ((123457,), torch.float16), ((3, 1025, 333), torch.bfloat16)],
}


# ---- refusals (no device needed) ----
def test_refusals_on_the_host():
    x = torch.ones(3)
    with pytest.raises(RuntimeError, match="HIP device"):
        NV.grad_norm([x])
    with pytest.raises(RuntimeError, match="HIP device"):
        NV.clip_by_global_norm([x], 1.0)
    with pytest.raises(ValueError, match="norm_type"):
        NV.grad_norm([x], 3)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            NV.clip_by_global_norm([x], bad)
        with pytest.raises(ValueError, match="max_norm"):
            NV.clip_grad_norm_([x], bad)
        with pytest.raises(ValueError, match="max_norm"):
            NV.HipAdam([torch.nn.Parameter(x.clone())], max_grad_norm=bad)
    with pytest.raises(TypeError):
        NV.grad_norm([x.double()])
    with pytest.raises(TypeError):
        NV.grad_norm([x.to_sparse()])
    with pytest.raises(TypeError):
        NV.grad_norm(["x"])
    assert float(NV.grad_norm([])) == 0.0
    assert NV.clip_by_global_norm([], 1.0)[0] == []
    assert float(NV.clip_grad_norm_([torch.nn.Parameter(x.clone())], 1.0)) == 0.0            # no gradients
    opt = NV.HipAdam([torch.nn.Parameter(x.clone())], max_grad_norm=1.0)
    with pytest.raises(ValueError, match="pieces"):
        opt.step(only=(opt.param_groups[0]["params"][0],))
    with pytest.raises(ValueError, match="pieces"):
        opt.step(skip=())
    assert opt.fused_update_args(opt.param_groups[0]["params"][0]) is None


def _c_clip(src, dst, numel, dtype=None, kind=2, max_norm=1.0, ws=1 << 40, nbytes=0):
    """vhap_grad_clip on made-up addresses: every call here is refused before anything is launched"""
    n = len(src)
    P = ctypes.c_void_p * n
    d = (ctypes.c_int32 * n)(*(dtype or [0] * n))
    return _lib.lib().vhap_grad_clip(n, P(*src), P(*dst), (ctypes.c_int64 * n)(*numel), d, kind, max_norm, ws, nbytes, 1 << 41, 0)


def test_c_entry_refusals():
    B = 1 << 30
    big = 1 << 20                                                    # (more than one block's work: a workspace is needed)
    assert _c_clip([B], [B], [big]) == _lib.E_WORKSPACE
    assert _c_clip([B], [B], [-1]) == _lib.E_BADDIM
    assert _c_clip([B], [B], [1 << 38]) == _lib.E_BADDIM
    assert _c_clip([B, B], [B, B], [1 << 37, 1 << 37]) == _lib.E_BADDIM
    assert _c_clip([B], [B], [big], dtype=[3]) == _lib.E_BADDIM
    assert _c_clip([B], [B], [big], max_norm=-1.0) == _lib.E_BADDIM
    assert _c_clip([B], [B], [big], max_norm=math.nan) == _lib.E_BADDIM
    assert _c_clip([B], [B], [big], kind=3) == _lib.E_UNSUPPORTED
    assert _c_clip([0], [B], [big]) == _lib.E_NULLPTR
    assert _c_clip([B], [0], [big]) == _lib.E_NULLPTR
    # memory: the same tensor twice, a result inside another, a result over another's source, a result half over its own source
    far = B + 16 * big
    assert _c_clip([B, B], [B, B], [big, big]) == _lib.E_UNSUPPORTED
    assert _c_clip([B, far], [B, B + 4], [big, 4]) == _lib.E_UNSUPPORTED
    assert _c_clip([B, far], [far, 2 * far], [big, big]) == _lib.E_UNSUPPORTED
    assert _c_clip([B], [B + 4], [big]) == _lib.E_UNSUPPORTED
    # and what is not: neighbours, sources that share memory
    assert _c_clip([B, B + 4 * big], [B, B + 4 * big], [big, big]) == _lib.E_WORKSPACE
    assert _c_clip([B, B], [far, 2 * far], [big, big]) == _lib.E_WORKSPACE
    L = _lib.lib()
    one = (ctypes.c_void_p * 1)(B)
    n1, i1 = (ctypes.c_int64 * 1)(big), (ctypes.c_int32 * 1)(0)
    assert L.vhap_adam_step_clipped(17, one, one, one, one, n1, i1, B, B, 0.9, 0.99, 1e-8, 1.0, 0, 0, 0, 0, 0) == _lib.E_BADDIM
    assert L.vhap_adam_step_clipped(1, one, one, one, one, n1, i1, B, B, 0.9, 0.99, 1e-8, -1.0, 0, 0, 0, 0, 0) == _lib.E_BADDIM
    assert L.vhap_adam_step_clipped(1, one, one, one, one, n1, i1, B, B, 0.9, 0.99, 1e-8, 1.0, 0, 0, 0, 0, 0) == _lib.E_WORKSPACE
    assert L.vhap_adam_step_clipped(1, one, one, None, one, n1, i1, B, B, 0.9, 0.99, 1e-8, 1.0, 0, 0, 0, 0, 0) == _lib.E_NULLPTR


# ---- GPU ----
@pytest.mark.gpu
@pytest.mark.parametrize("name", sorted(LISTS))
@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("share", [0.25, 4.0])
def test_norm_and_clip(name, p, share):
    gs = [randn(s, 7 * i + 1, d, 10.0 ** (i % 3 - 1)) for i, (s, d) in enumerate(LISTS[name])]
    want = norm64(gs, p)
    assert near_norm(float(NV.grad_norm(gs, p)), want)
    max_norm = float(torch.tensor(want * share))
    c = coefficient(want, max_norm)
    keep = [g.clone() for g in gs]
    out, n = NV.clip_by_global_norm(gs, max_norm, p)
    assert near_norm(float(n), want) and n.shape == () and n.dtype == torch.float32
    for o, g, k in zip(out, gs, keep):
        assert o.data_ptr() != g.data_ptr() or g.numel() == 0
        assert torch.equal(g, k) and o.shape == g.shape and o.dtype == g.dtype
        check_clipped(o, k, c)
    _, n2 = NV.clip_by_global_norm(gs, max_norm, p, out=gs)                       # in place: the same bits
    assert torch.equal(n, n2)
    for o, g in zip(out, gs):
        assert torch.equal(o, g)


@pytest.mark.gpu
@pytest.mark.parametrize("share", [0.5, 2.0])
def test_some_in_place_some_not(share):
    """one list, a large tensor in place beside one that is not, clipped and within the limit (where the first is left alone and the second copied)"""
    gs = [randn((1 << 21,), 1), randn((1 << 21,), 2), randn((3, 1000, 1001), 3, torch.bfloat16)]
    keep = [g.clone() for g in gs]
    want = norm64(keep, 2.0)
    out = [gs[0], torch.zeros_like(gs[1]), gs[2]]
    n = NV.clip_by_global_norm(gs, want * share, out=out)[1]
    assert near_norm(float(n), want) and torch.equal(gs[1], keep[1])
    for o, k in zip(out, keep):
        check_clipped(o, k, coefficient(want, want * share))


@pytest.mark.gpu
@pytest.mark.parametrize("flat", [False, True])
@pytest.mark.parametrize("count", [127, 128, 129, 500])
def test_many_tensors(flat, count):
    sizes = [(37 * i) % 1301 for i in range(count)]
    if flat:                                                                     # views of one flat buffer, at every alignment; guards on both sides
        buf, at, gs = randn((sum(sizes) + 2,), 3, torch.bfloat16), 1, []
        for s in sizes:
            gs.append(buf[at:at + s])
            at += s
        guard = (buf[0].clone(), buf[-1].clone())
    else:
        gs = [randn((s,), i, torch.float32) for i, s in enumerate(sizes)]
    keep = [g.clone() for g in gs]
    want = norm64(keep, 2.0)
    n = NV.clip_by_global_norm(gs, 0.5, out=gs)[1]
    assert near_norm(float(n), want)
    for g, k in zip(gs, keep):
        check_clipped(g, k, coefficient(want, 0.5))
    if flat:
        assert torch.equal(buf[0], guard[0]) and torch.equal(buf[-1], guard[1])


@pytest.mark.gpu
def test_strides():
    base = randn((6, 40, 30), 5)
    perm, cols, step = base.permute(2, 0, 1), randn((50, 33), 6)[:, 3:20], randn((999,), 7)[::3]
    gs = [perm, cols, step]
    keep = [g.clone() for g in gs]
    want = norm64(gs, 2.0)
    assert near_norm(float(NV.grad_norm(gs)), want)
    out, _ = NV.clip_by_global_norm(gs, 1.0)
    for o, k in zip(out, keep):
        check_clipped(o, k, coefficient(want, 1.0))
    NV.clip_by_global_norm(gs, 1.0, out=gs)
    for g, o in zip(gs, out):
        assert torch.equal(g, o)
    assert near_norm(float(NV.grad_norm([torch.ones(1, device="cuda").expand(100)])), 10.0)
    for bad in ([torch.ones(1, device="cuda").expand(100)], [base, base], [cols, cols]):
        with pytest.raises(ValueError):
            NV.clip_by_global_norm(bad, 1.0, out=bad)
    with pytest.raises(ValueError):
        NV.clip_by_global_norm([base], 1.0, out=[base.view(-1)])
    with pytest.raises(ValueError):
        NV.clip_by_global_norm([base.view(-1)[:100]], 1.0, out=[base.view(-1)[50:150]])


@pytest.mark.gpu
@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("n", [100, 100_000])
def test_values_that_are_not_ordinary(p, n):
    big = randn((n,), 1, scale=1e30)                                             # squares beyond fp32
    want = norm64([big], p)
    if want < 3e38:
        assert near_norm(float(NV.grad_norm([big], p)), want)
    out, _ = NV.clip_by_global_norm([big], 1.0, p)
    check_clipped(out[0], big, 1.0 / (want + 1e-6))
    small = randn((n,), 2, scale=1e-30)                                          # squares below it; never above the limit: left alone
    assert near_norm(float(NV.grad_norm([small], p)), norm64([small], p))
    out, _ = NV.clip_by_global_norm([small], 1.0, p)
    assert torch.equal(out[0], small)
    zero = torch.zeros(n, device="cuda")
    out, z = NV.clip_by_global_norm([zero], 1.0, p)
    assert float(z) == 0.0 and torch.equal(out[0], zero)
    assert torch.equal(NV.clip_by_global_norm([big], 0.0, p)[0][0], torch.zeros_like(big))
    for where in (0, n // 2, n - 1):
        bad = randn((n,), 3)
        bad[where] = math.nan
        out, z = NV.clip_by_global_norm([randn((5,), 4), bad], 1.0, p)
        assert math.isnan(float(z)) and bool(out[0].isnan().all()) and bool(out[1].isnan().all())
        bad[where] = -math.inf
        out, z = NV.clip_by_global_norm([randn((5,), 4), bad], 1.0, p)
        assert float(z) == math.inf and not bool(out[0].any()) and bool(out[1][where].isnan()) and int(out[1].isnan().sum()) == 1


@pytest.mark.gpu
def test_clip_grad_norm_like_torch():
    ps = [torch.nn.Parameter(randn(s, i)) for i, s in enumerate([(300,), (4, 100), (3, 64, 64), (7,)])]
    ref = [torch.nn.Parameter(p.detach().double().cpu()) for p in ps]
    for p, r in list(zip(ps, ref))[:-1]:                                         # the last has no gradient
        p.grad = randn(p.shape, 17)
        r.grad = p.grad.double().cpu()
    want = float(torch.nn.utils.clip_grad_norm_(ref, 2.5))
    assert near_norm(float(NV.clip_grad_norm_(ps, 2.5, error_if_nonfinite=True)), want)
    for p, r in list(zip(ps, ref))[:-1]:
        assert bool(((p.grad.double().cpu() - r.grad).abs() <= r.grad.abs() * 2.0 ** -23 * 1.001).all())
    assert ps[-1].grad is None
    v = ps[0].grad._version
    NV.clip_grad_norm_(ps[0], 1e-3)                                              # a single tensor; autograd sees that the gradient was written
    assert ps[0].grad._version > v
    ps[0].grad[0] = math.inf
    keep = ps[1].grad.clone()
    with pytest.raises(RuntimeError, match="norm"):
        NV.clip_grad_norm_(ps, 1.0, error_if_nonfinite=True)
    assert torch.equal(ps[1].grad, keep)


@pytest.mark.gpu
def test_streams_and_captures():
    """on a stream that is not the current default, two captured calls side by side (own workspaces), several replays with eager work between them"""
    lists = [[randn((70_000 + 13 * j,), 10 * j), randn((999,), 10 * j + 1, torch.bfloat16)] for j in range(2)]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        n = NV.grad_norm(lists[0])
    torch.cuda.current_stream().wait_stream(st)
    assert near_norm(float(n), norm64(lists[0], 2.0))
    graphs, results = [], []
    for gs in lists:
        NV.clip_by_global_norm(gs, 1.0)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(NV.clip_by_global_norm(gs, 1.0))
        graphs.append(g)
    for k in range(4):
        for j, gs in enumerate(lists):
            for i, t in enumerate(gs):
                t.copy_(randn(t.shape, 100 + 10 * k + 3 * j + i, t.dtype))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for gs, (out, n) in zip(lists, results):
            eager, n2 = NV.clip_by_global_norm(gs, 1.0)
            assert torch.equal(n, n2) and all(torch.equal(a, b) for a, b in zip(out, eager))


B1, B2 = 0.9, 0.999


def _adam64(p, m, v, g, t, lr, c):
    g = g * c
    m = B1 * m + (1 - B1) * g
    v = B2 * v + (1 - B2) * g * g
    return p - lr / (1 - B1 ** t) * m / ((v / (1 - B2 ** t)).sqrt() + 1e-8), m, v


@pytest.mark.gpu
@pytest.mark.parametrize("shapes", [[(5,)], [(300,), (16, 100), (0,), (1,)], [(300,), (3, 256, 257), (15429,)], [(1,)] * 16])
@pytest.mark.parametrize("share", [0.2, 5.0])
def test_clipped_adam(shapes, share):
    """three steps against Adam in 64 bits; the norm and the moments' first step bit for bit those of clipping in place"""
    grads = [[randn(s, 50 * t + i, scale=10.0 ** -(i % 4)) for i, s in enumerate(shapes)] for t in range(3)]
    p0 = [randn(s, 900 + i) for i, s in enumerate(shapes)]
    max_norm = float(torch.tensor(norm64(grads[0], 2.0) * share))
    fused = [torch.nn.Parameter(p.clone()) for p in p0]
    a = NV.HipAdam([{"params": fused[:1], "lr": 1e-2}, {"params": fused[1:], "lr": 3e-3}], max_grad_norm=max_norm)
    ref = [(p.double().cpu(), torch.zeros(p.shape, dtype=torch.float64), torch.zeros(p.shape, dtype=torch.float64)) for p in p0]
    for t, gs in enumerate(grads):
        for f, g in zip(fused, gs):
            f.grad = g.clone()
        want = norm64(gs, 2.0)
        a.step()
        assert near_norm(float(a.grad_norm), want)
        assert all(torch.equal(f.grad, g) for f, g in zip(fused, gs))            # the gradients stay as they were
        clipped, n = NV.clip_by_global_norm(gs, max_norm)
        assert torch.equal(n, a.grad_norm)
        if t == 0:
            assert all(torch.equal(a.state[f]["exp_avg"], g * 0.1) for f, g in zip(fused, clipped))
        c = coefficient(want, max_norm)
        ref = [_adam64(*r, g.double().cpu(), t + 1, 1e-2 if i == 0 else 3e-3, c) for i, (r, g) in enumerate(zip(ref, gs))]
    assert int(a.step_count) == 3
    u = 2.0 ** -24
    for i, (f, (p, m, v)) in enumerate(zip(fused, ref)):
        top = max([coefficient(norm64(gs, 2.0), max_norm) * float(gs[i].double().abs().max()) for gs in grads if gs[i].numel()] + [0.0])
        # a step of m: c and g c round (2 u of 0.1 g), 1 - b1 (1 u of 0.1 (g - m)), g - m, its product and the sum: with |m| <= 0.3 top under 1 u top; three steps
        assert bool(((a.state[f]["exp_avg"].double().cpu() - m).abs() <= 3 * u * top + 1e-44).all())
        # a step of v: g c squared (2 x 2 u, 2 u, 1 u of 0.001 g^2), b2 v and the sum (3 u of at most 0.003 top^2): under 0.02 u top^2; three steps
        assert bool(((a.state[f]["exp_avg_sq"].double().cpu() - v).abs() <= 0.06 * u * top * top + 1e-44).all())
        # p: a step's own rounding, and lr x (at most 1.75 = m / sqrt v over three nearly equal weights) x the relative roundings of the corrections, the moments and the
        # quotient: under 60 u
        lr = 1e-2 if i == 0 else 3e-3
        assert bool(((f.detach().double().cpu() - p).abs() <= 3 * (u * (p.abs() + 0.1) + lr * 1.75 * 60 * u)).all())


@pytest.mark.gpu
def test_clipped_adam_counter_flags_and_capture():
    ps = [torch.nn.Parameter(randn((40_000,), 1)), torch.nn.Parameter(randn((7,), 2))]
    for p in ps:
        p.grad = randn(p.shape, 3)
    opt = NV.HipAdam(ps, lr=1e-3, max_grad_norm=0.1)
    opt.step(advance=False)
    assert int(opt.step_count) == 0
    opt.advance()
    opt.step(advanced=True)
    assert int(opt.step_count) == 1
    opt.step()
    assert int(opt.step_count) == 2
    ps[0].grad = None                                                            # now one block's work: the single launch counts as well
    opt.step(advance=False)
    assert int(opt.step_count) == 2
    opt.step()
    assert int(opt.step_count) == 3 and near_norm(float(opt.grad_norm), norm64([ps[1].grad], 2.0))
    empty = torch.nn.Parameter(torch.zeros(0, device="cuda"))
    empty.grad = torch.zeros_like(empty)
    o = NV.HipAdam([empty], max_grad_norm=1.0)
    o.step()
    assert int(o.step_count) == 1 and float(o.grad_norm) == 0.0
    for n in (2000, 200_000):                                                    # captured: replays against an eager twin
        a, b = (torch.nn.Parameter(randn((n,), 9)) for _ in range(2))
        a.grad, b.grad = torch.zeros_like(a), torch.zeros_like(b)
        oa, ob = NV.HipAdam([a], lr=1e-2, max_grad_norm=0.3), NV.HipAdam([b], lr=1e-2, max_grad_norm=0.3)
        oa._build()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            oa.step()
        for k in range(4):
            a.grad.copy_(randn((n,), 20 + k))
            b.grad.copy_(a.grad)
            g.replay()
            ob.step()
            torch.cuda.synchronize()
            assert torch.equal(a.detach(), b.detach()) and torch.equal(oa.grad_norm, ob.grad_norm) and int(oa.step_count) == k + 1


def test_a_negated_view_is_refused():
    """.imag of a conjugated tensor is real, dense and holds the opposite of what its memory does"""
    x = torch.randn(8, dtype=torch.complex64).conj().imag
    assert x.is_neg()
    for call in (lambda: NV.grad_norm([x]), lambda: NV.clip_by_global_norm([x], 1.0), lambda: NV.clip_by_global_norm([torch.ones(8)], 1.0, out=[x])):
        with pytest.raises((TypeError, RuntimeError)):
            call()
    with pytest.raises(TypeError, match="negated"):
        NV.grad_norm([x])


@pytest.mark.gpu
def test_strided_results_side_by_side_and_overlapping():
    buf = randn((40, 60), 1, scale=3.0)
    src = buf.clone()
    views = [buf[:, :25], buf[:, 25:59], buf[:, 59:]]                            # columns of one matrix: the norm is the matrix's
    _, norm = NV.clip_by_global_norm(views, 1.0, out=views)
    want = norm64([src], 2)
    assert near_norm(float(norm), want)
    check_clipped(buf, src, coefficient(want, 1.0))
    g = [randn((40, 30), 2), randn((40, 30), 3)]
    square = torch.empty(30, 40, device="cuda")
    for out in ([buf[:, :30], buf[:, 29:59]], [buf[:, :30], buf[::1, :30]], [buf[:, 30:], buf[:, :31][:, 1:]], [square.t(), square.view(40, 30)],
                [buf[:, :30], buf.view(-1)[45:45 + 1200].view(40, 30)]):
        keep = buf.clone()
        with pytest.raises(ValueError, match="overlap|twice"):
            NV.clip_by_global_norm(g, 1.0, out=out)
        assert torch.equal(buf, keep)
    out = [buf[:, 30:], buf[:, :30]]                                             # in the other order in memory
    _, norm = NV.clip_by_global_norm(g, 1.0, out=out)
    for o, x in zip(out, g):
        check_clipped(o, x, coefficient(norm64(g, 2), 1.0))
