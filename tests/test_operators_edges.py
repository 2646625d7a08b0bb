"""The operators of the parameter update and of 4-bit spaces where a call is allowed but unusual: views that autograd makes by itself, results that interleave in memory,
derivatives these operators do not have, sizes that take a kernel of their own."""
import math

import pytest
import torch

from tests.test_gradnorm import check_clipped, coefficient, near_norm, norm64, randn
from tests.test_mx import PIECES, TYPES, check_sum, random_mx, values64
from vhap_amd import _lib, mx
from vhap_amd import native as NV


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 70])
def test_a_gradient_that_is_a_negated_view(n):
    """autograd hands a node views whose memory holds the opposite of what they say (the imaginary part of a conjugate): dense ones, and for a W of one row strided ones"""
    w, c = random_mx(n, 40, 1), randn((5, n), 2)

    def gradients(of):
        x, b = randn((5, 40), 3).requires_grad_(), randn((n,), 4).requires_grad_()
        y, seen = mx.linear(x, w, b), []
        y.register_hook(lambda g: seen.append(g.is_neg()))
        of(y)
        return x.grad, b.grad, seen
    dx, db, _ = gradients(lambda y: y.backward(c))
    for of in (lambda y: y.backward(torch._neg_view(-c)), lambda y: (torch.complex(c, y).conj() * torch.complex(c, c)).real.sum().backward()):
        dx1, db1, seen = gradients(of)
        assert seen == [True] and torch.equal(dx1, dx) and torch.equal(db1, db)


@pytest.mark.gpu
def test_one_result_given_for_two_gradients():
    """the first gradient goes through a copy, the second straight to the kernel"""
    g = [randn((30, 40), 1).t(), randn((40, 30), 2)]
    o, keep = randn((40, 30), 3), randn((40, 30), 3)
    for grads in (g, g[::-1], [g[0], g[0]]):
        with pytest.raises(ValueError, match="overlap|twice"):
            NV.clip_by_global_norm(grads, 1.0, out=[o, o])
        assert torch.equal(o, keep)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [60, 61])
def test_results_that_interleave(width):
    """no element in common, though each lies between the other's"""
    buf = randn((40, width), 1, scale=3.0)
    square = randn((50, 50), 2, scale=3.0)
    cube = randn((6, 9, 8), 3, scale=3.0)
    for whole, views in ((buf, [buf[:, ::2], buf[:, 1::2]]), (buf, [buf[::2], buf[1::2, ::3], buf[1::2, 1::3], buf[1::2, 2::3]]),
                         (cube, [cube[:, ::3], cube[:, 1::3], cube[:, 2::3, ::2], cube[:, 2::3, 1::2]]), (buf.t(), [buf.t()[::3], buf.t()[1::3], buf.t()[2::3]])):
        src = whole.clone()
        _, norm = NV.clip_by_global_norm(views, 1.0, out=views)
        want = norm64([src], 2)
        assert near_norm(float(norm), want)
        check_clipped(whole, src, coefficient(want, 1.0))
    lines = [torch.diagonal(square), square.view(-1)[1::51]]
    keep, src = square.clone(), [v.clone() for v in lines]
    NV.clip_by_global_norm(lines, 1.0, out=lines)
    for v, s in zip(lines, src):
        check_clipped(v, s, coefficient(norm64(src, 2), 1.0))
    rest = ~(torch.eye(50, dtype=torch.bool) | torch.diag(torch.ones(49, dtype=torch.bool), 1)).cuda()
    assert torch.equal(square[rest], keep[rest])
    for views in ([buf[:, ::2], buf[:, ::3]], [buf[::2], buf[::5, :1]], [square[:, :1], torch.diagonal(square)], [cube[:, :, ::3], cube[:, 8:, 6:7]]):
        keep = [v.clone() for v in views]
        with pytest.raises(ValueError, match="overlap"):
            NV.clip_by_global_norm(views, 1.0, out=views)
        assert all(torch.equal(v, k) for v, k in zip(views, keep))


@pytest.mark.gpu
def test_what_counts_as_overlapping_is_what_shares_memory():
    """random strided pairs of both widths of element, against the sets of bytes"""
    import random
    rng = random.Random(5)
    base = torch.zeros(1200, device="cuda")
    taken = refused = 0
    for _ in range(300):
        views, bytes_of = [], []
        for _ in range(2):
            dt = rng.choice([torch.float32, torch.bfloat16])
            sizes = [rng.randint(1, 4) for _ in range(rng.randint(1, 3))]
            order, step, strides = list(range(len(sizes))), rng.randint(1, 3), [0] * len(sizes)
            rng.shuffle(order)
            for d in order:                                                      # (nested, so that no view overlaps itself)
                strides[d] = step
                step = step * sizes[d] + rng.randint(0, 5)
            at = rng.randint(0, 40)
            v = base.view(dt).as_strided(sizes, strides, at)
            index = torch.arange(4800 // dt.itemsize).as_strided(sizes, strides, at).reshape(-1).tolist()
            views.append(v)
            bytes_of.append({i * dt.itemsize + b for i in index for b in range(dt.itemsize)})
        grads = [torch.full(tuple(v.shape), 2.0, dtype=v.dtype, device="cuda") for v in views]
        base.zero_()
        if bytes_of[0] & bytes_of[1]:
            refused += 1
            with pytest.raises(ValueError, match="overlap"):
                NV.clip_by_global_norm(grads, 1e9, out=views)
        else:
            taken += 1
            NV.clip_by_global_norm(grads, 1e9, out=views)
            assert all(bool((v == 2.0).all()) for v in views)
    assert taken > 50 and refused > 50


@pytest.mark.gpu
def test_a_result_that_overlaps_itself():
    base = randn((64,), 1)
    keep = base.clone()
    for sizes, strides in (((5, 4), (1, 1)), ((4, 6), (5, 1)), ((3, 3, 3), (4, 2, 4)), ((7,), (0,))):
        with pytest.raises(ValueError, match="share memory"):
            NV.clip_by_global_norm([randn(sizes, 2)], 1.0, out=[base.as_strided(sizes, strides)])
        assert torch.equal(base, keep)
    g = randn((2, 3), 3)                                                         # 0, 2, 4, 3, 5, 7: strides that look as if they did
    out = base.as_strided((2, 3), (3, 2))
    NV.clip_by_global_norm([g], 1e9, out=[out])
    assert torch.equal(out, g)


def test_a_forward_mode_tangent_is_refused():
    """dropped, it would count as zero"""
    import torch.autograd.forward_ad as fwAD
    w, x, b, g = random_mx(70, 40, 1, "cpu"), torch.randn(5, 40), torch.randn(70), torch.randn(5, 70)
    with fwAD.dual_level():
        for call in (lambda: mx.linear(fwAD.make_dual(x, torch.ones_like(x)), w), lambda: mx.linear(x, w, fwAD.make_dual(b, torch.ones_like(b))),
                     lambda: mx.linear_input_grad(fwAD.make_dual(g, torch.ones_like(g)), w)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


@pytest.mark.gpu
def test_a_forward_mode_tangent_is_refused_on_the_device():
    import torch.autograd.forward_ad as fwAD
    w, x, g = random_mx(70, 40, 1), randn((5, 40), 2), randn((5, 70), 3)
    with fwAD.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"), torch.no_grad():
            mx.linear(fwAD.make_dual(x, torch.ones_like(x)), w)
        x1 = x.clone().requires_grad_()
        with pytest.raises(RuntimeError, match="forward-mode"):                  # forward over reverse
            torch.autograd.grad(mx.linear(x1, w), x1, fwAD.make_dual(g, torch.ones_like(g)))
        torch.autograd.grad(mx.linear(x1, w), x1, g)


def _collectives(monkeypatch, seen):
    """stand-ins for a group of two equal ranks over gloo: what they are given is noted"""
    from vhap_amd import dist as D
    monkeypatch.setattr(D.dist, "get_rank", lambda group=None: 0)
    monkeypatch.setattr(D.dist, "get_world_size", lambda group=None: 2)
    monkeypatch.setattr(D.dist, "get_backend", lambda group=None: "gloo")

    def all_reduce(t, op=None, group=None, async_op=False):
        seen.append(t)
        t.mul_(2)

    def all_gather_into_tensor(out, src, group=None, async_op=False):
        seen.extend([out, src])
        out.copy_(torch.cat([src, src]).view_as(out))
    monkeypatch.setattr(D.dist, "all_reduce", all_reduce)
    monkeypatch.setattr(D.dist, "all_gather_into_tensor", all_gather_into_tensor)
    return D.FrameShardContext()


def _use_collectives(ctx, make):
    """every collective of the context on tensors from make(values) -> what they leave"""
    v = torch.arange(24, dtype=torch.float32)
    out = []
    t = make(v)
    out += [ctx.all_reduce_sum(t), t]
    t = make(v)
    assert ctx.all_reduce_sum_(t) is t
    out.append(t)
    for a in (False, True):
        t = make(v)
        w = ctx.all_reduce_mean_(t, async_op=a)
        assert w is None
        full, part = make(v), make(torch.zeros(12))
        ctx.reduce_scatter_mean(full, part, async_op=a).wait()
        planes = make(v.view(3, 4, 2))
        for w in ctx.all_gather_rows(planes, 0, 2, async_op=a):
            w.wait()
        out += [t, part, planes]
    p, q = make(v).requires_grad_(), make(v[:5]).requires_grad_()
    p.grad = make(v * 3)
    ctx.average_gradients([p, q])
    return out + [p.grad, q.grad]


def _check_collectives(out):
    v = torch.arange(24, dtype=torch.float32)
    planes = v.view(3, 4, 2)
    gathered = torch.cat([planes[:, :2], planes[:, :2]], 1)
    want = [2 * v, v, 2 * v] + [v, v[:12], gathered] * 2 + [3 * v, torch.zeros(5)]
    assert len(out) == len(want)
    for a, b in zip(out, want):
        assert a.shape == b.shape and torch.equal(a.detach().cpu(), b)


class _Elsewhere(torch.Tensor):
    """a tensor in host memory that says it is on the device"""
    is_cuda = True

    def cpu(self):
        return self.detach().as_subclass(torch.Tensor).clone()


def test_gloo_is_given_host_memory(monkeypatch):
    seen = []
    ctx = _collectives(monkeypatch, seen)
    out = _use_collectives(ctx, lambda v: v.clone().as_subclass(_Elsewhere))
    assert len(seen) > 10 and not any(isinstance(t, _Elsewhere) for t in seen)
    _check_collectives([t.as_subclass(torch.Tensor) for t in out])
    seen.clear()
    _check_collectives(_use_collectives(ctx, lambda v: v.clone()))               # and what is in host memory goes as it is
    assert len(seen) > 10


@pytest.mark.gpu
def test_gloo_is_given_host_memory_of_device_tensors(monkeypatch):
    seen = []
    ctx = _collectives(monkeypatch, seen)
    out = _use_collectives(ctx, lambda v: v.cuda())
    assert len(seen) > 10 and not any(t.is_cuda for t in seen) and all(t.is_cuda for t in out)
    _check_collectives(out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 130, 70), (2, 40000, 150), (1, 40000, 300), (4, 100, 70), (40, 300, 135), (40, 20000, 20), (33, 70000, 33), (3, 40, 1030), (16, 100, 1100)])
def test_codes_behind_the_last_element_are_no_numbers(m, n, k, dtype):
    """the largest scales, at which a code of 4 or 6 (253) or of 2 and more (254) is past float32: elements that are not, codes behind them that are"""
    w = random_mx(n, k, 1, lo=253, hi=255)
    kb = w.scales.shape[1]
    half = torch.randint(0, 2, (n, 32 * kb), generator=torch.Generator().manual_seed(2), dtype=torch.uint8) + 8 * torch.randint(
        0, 2, (n, 32 * kb), generator=torch.Generator().manual_seed(3), dtype=torch.uint8)                      # +-0, +-0.5
    half[:, k:] = 7
    w.codes.copy_((half[:, 0::2] | half[:, 1::2] << 4).cuda())
    W, X = values64(w), (randn((m, k), 4) * 2.0 ** -12).to(dtype)
    X64 = X.cpu().double()
    want, mags = X64 @ W.t(), X64.abs() @ W.abs().t()
    got = mx.linear(X, w)
    if dtype == torch.float16:
        assert not bool(got.isnan().any())                                       # (infinite: past float16)
    else:
        assert float(mags.max()) < 3.4e38
        check_sum(got, want, mags, k * PIECES[dtype], dtype)


@pytest.mark.gpu
def test_matmul_with_codes_behind_the_last_element_at_the_largest_scales():
    for m, n, k in ((40, 50, 70), (6200, 1000, 70)):
        a, b = random_mx(m, k, 1, lo=253, hi=255, garbage=True), random_mx(n, k, 2, lo=60, hi=64, garbage=True)
        A, B = values64(a), values64(b)
        check_sum(mx.matmul(a, b), A @ B.t(), A.abs() @ B.abs().t(), k, torch.float32)
        check_sum(mx.matmul(b, a), B @ A.t(), B.abs() @ A.abs().t(), k, torch.float32)


def test_a_gradient_that_needs_no_partial_sums_asks_for_next_to_no_workspace():
    bytes_of = _lib.lib().vhap_mx4_linear_input_grad_workspace_bytes
    assert 0 < bytes_of(4_200_000, 8, 33) <= 64 and 0 < bytes_of(5, 300, 90) <= 64
    assert bytes_of(1, 786432, 100) >= 4 * 128 * 256 and bytes_of(256, 15429, 400) >= 4 * 2 * 256 * 512
    assert bytes_of(1, 1 << 20, 7) >= 4 * 128 and bytes_of(1, 2, (1 << 24)) >= 4 * (1 << 24)     # one row against many blocks: always by way of partial sums


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_a_gradient_without_partial_sums(dtype):
    L, w, g = _lib.lib(), random_mx(300, 90, 1), randn((5, 300), 2, dtype)
    dx, code, ws = torch.empty(5, 90, dtype=dtype, device="cuda"), TYPES.index(dtype), torch.empty(64, dtype=torch.uint8, device="cuda")
    _lib.check(L.vhap_mx4_linear_input_grad(g.data_ptr(), code, 300, 5, w.codes.data_ptr(), w.scales.data_ptr(), 300, 90, ws.data_ptr(), 64, dx.data_ptr(), 0,
                                            torch.cuda.current_stream().cuda_stream), "vhap_mx4_linear_input_grad")
    W, G = values64(w), g.cpu().double()
    check_sum(dx, G @ W, G.abs() @ W.abs(), 300 * PIECES[dtype], dtype)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    m = 200_000                                                                  # dx alone is 18 MB, partial sums would be 102
    mx.linear_input_grad(torch.zeros(m, 8, dtype=dtype, device="cuda"), random_mx(8, 45, 1))
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < 1.2 * m * (8 + 45) * dtype.itemsize + (4 << 20)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16, torch.float64])
def test_the_texture_space_in_other_types(dtype):
    """the module moved to another floating-point type takes codes of that type, as it does with a basis in that type"""
    from tests.test_texpca import _space
    from vhap_amd.flame import FlameTexPCA
    n, T = 50, 64
    m = FlameTexPCA(n, tex_size=T, tex_space=_space(), basis_format="mxfp4").cuda().to(dtype)
    code = randn((2, n), 1).to(dtype).requires_grad_()
    out = m(code)
    assert out.dtype == dtype and out.shape == (2, 3, T, T)
    W, mean, c = values64(m.mx_basis()), m.texture_mean.reshape(-1).cpu().double(), code.detach().cpu().double()
    S = m.src_size
    want = (mean + c @ W.t()).view(2, S, S, 3).permute(0, 3, 1, 2)
    want = torch.nn.functional.interpolate(want, [T, T])[:, [2, 1, 0]] / 255
    size = (mean.abs() + c.abs() @ W.abs().t()).view(2, S, S, 3).permute(0, 3, 1, 2)
    size = torch.nn.functional.interpolate(size, [T, T])[:, [2, 1, 0]] / 255
    # fp32 sums of at most three pieces a product; three roundings to the type (the sum, 1 / 255 or the quotient); clamping only brings nearer
    u = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float64: 2.0 ** -53}[dtype]
    limit = (n * 3 + 5) * 2.0 ** -23 * size + 4 * u * want.abs() + 4 * u * 2.0 ** -14
    assert bool(((out.detach().cpu().double() - want.clamp(0, 1)).abs() <= limit).all())
    out.sum().backward()
    assert code.grad.dtype == dtype and bool(code.grad.isfinite().all()) and bool(code.grad.any())


def test_a_limit_that_is_no_limit_is_refused_on_the_host(flame_model):
    """torch's clipping takes a negative limit and turns the gradients round"""
    from tests.test_operators_in_use import _tracker
    import numpy as np
    for bad in (-1.0, math.nan):
        tr, _ = _tracker(flame_model, device="cpu", T=64, H=32, W=32, max_grad_norm=bad)
        with pytest.raises(ValueError, match="max_norm"):
            opt = tr.configure_optimizer(tr.get_train_parameters("lmk_init_all"))
            tr.optimize_iter(tr.get_sample(np.arange(2)), opt, "lmk_init_all")


@pytest.mark.gpu
def test_a_capture_beside_an_eager_graph_behind_the_input():
    """x made in the capture from a leaf of which an eager graph is alive, x itself made outside; nothing of either is differentiated here"""
    w = random_mx(70, 40, 1)
    leaf = randn((5, 40), 2).requires_grad_()
    bias = randn((70,), 3).requires_grad_()
    alive = [leaf * 2, bias * 2]
    torch.cuda.synchronize()
    for call in (lambda: mx.linear(leaf * 3, w), lambda: mx.linear(alive[0], w), lambda: mx.linear(torch.ones(5, 40, device="cuda"), w, bias * 3),
                 lambda: mx.linear((leaf * 3).view(5, 40)[:, :40] + 1, w)):
        with pytest.raises(RuntimeError, match="alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    del alive
    torch.cuda.synchronize()
    graph, g = torch.cuda.CUDAGraph(), randn((5, 70), 4)
    with torch.cuda.graph(graph):
        dx, db = torch.autograd.grad(mx.linear(leaf * 3, w, bias * 1), (leaf, bias), g)
    for k in range(3):
        g.copy_(randn((5, 70), 10 + k))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dx, 3 * mx.linear_input_grad(g, w)) and torch.equal(db, torch.autograd.grad(mx.linear(leaf.detach(), w, b1 := bias.detach().clone().requires_grad_()), b1, g)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("m,n,k", [(6200, 1000, 100), (6200, 1000, 128), (6145, 1023, 257), (12289, 513, 384), (70000, 65, 31)])
def test_matmul_over_many_tiles(m, n, k, out):
    """128 x 128 tiles: from 384 of them on"""
    assert -(-m // 128) * -(-n // 128) >= 384
    a, b, bias = random_mx(m, k, 1, lo=118, hi=127, garbage=True), random_mx(n, k, 2, lo=118, hi=127, garbage=True), randn((n,), 3)
    A, B = values64(a), values64(b)
    want, mags = A @ B.t(), A.abs() @ B.abs().t()
    check_sum(mx.matmul(a, b, out_dtype=out), want, mags, k, out)
    want, mags = want + bias.cpu().double(), mags + bias.abs().cpu().double()
    check_sum(mx.matmul(a, b, bias, out_dtype=out), want, mags, k + 1, out)
    check_sum(mx.matmul(a, b, bias, relu=True, out_dtype=out), want.clamp(min=0), mags, k + 1, out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 40000, 200), (2, 40000, 200), (1, 40000, 300), (1, 40000, 401), (1, 32768, 512), (2, 32769, 129), (1, 40001, 100), (2, 40001, 128), (2, 300, 7)])
def test_one_or_two_rows(m, n, k, dtype):
    w = random_mx(n, k, m + n + k, garbage=True)
    x, bias = randn((m, k), 1, dtype), randn((n,), 2)
    W, X, b = values64(w), x.cpu().double(), bias.cpu().double()
    check_sum(mx.linear(x, w), X @ W.t(), X.abs() @ W.abs().t(), k * PIECES[dtype], dtype)
    check_sum(mx.linear(x, w, bias), X @ W.t() + b, X.abs() @ W.abs().t() + b.abs(), k * PIECES[dtype] + 1, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(1, 270001, 100), (1, 81000, 401), (2, 300000, 60)])
def test_gradients_of_few_rows_against_a_large_matrix(m, n, k, dtype):
    w, g = random_mx(n, k, 1, garbage=True), randn((m, n), 2, dtype)
    W, G = w.dequantize().double(), g.double()                                   # (dequantize has its own tests)
    check_sum(mx.linear_input_grad(g, w), (G @ W).cpu(), (G.abs() @ W.abs()).cpu(), n * PIECES[dtype] + 1024, dtype)


@pytest.mark.gpu
def test_quantize_past_32_bits_of_elements():
    """rows x blocks x 4 past 2^31: the kernels' other index"""
    rows = 2 ** 29 + 3
    x = randn((1, 32), 1, torch.bfloat16)
    q, one = mx.quantize(x.expand(rows, 32)), mx.quantize(x)
    for at in range(0, rows, 2 ** 26):
        assert bool((q.codes[at:at + 2 ** 26] == one.codes).all()) and bool((q.scales[at:at + 2 ** 26] == one.scales).all())
    out, v = q.dequantize(torch.bfloat16), one.dequantize(torch.bfloat16)
    del q
    for at in range(0, rows, 2 ** 26):
        assert bool((out[at:at + 2 ** 26] == v).all())


@pytest.mark.gpu
@pytest.mark.parametrize("limit", [None, 0.3])
def test_state_loaded_into_an_optimiser_in_use(limit):
    """the moments go where the kernels write them: into the tensors that a step has already been issued on"""
    make = lambda: [torch.nn.Parameter(randn((300,), 1)), torch.nn.Parameter(randn((70, 1000), 2))]
    a, b = make(), make()
    oa, ob = NV.HipAdam(a, lr=1e-2, max_grad_norm=limit), NV.HipAdam(b, lr=1e-2, max_grad_norm=limit)

    def step(ps, opt, k):
        for i, p in enumerate(ps):
            p.grad = randn(p.shape, 10 * k + i)
        opt.step()
    for k in range(3):
        step(a, oa, k)
        step(b, ob, k)
    saved = {"state": {i: {n: t.clone() for n, t in s.items()} for i, s in oa.state_dict()["state"].items()}, "param_groups": oa.state_dict()["param_groups"]}
    step(b, ob, 7)                                                               # b goes astray, and is taken back
    with torch.no_grad():
        for p, q in zip(a, b):
            q.copy_(p)
    held = [ob.state[p]["exp_avg"].data_ptr() for p in b]
    ob.load_state_dict(saved)
    ob._step.copy_(oa._step)
    assert [ob.state[p]["exp_avg"].data_ptr() for p in b] == held
    for k in range(3, 5):
        step(a, oa, k)
        step(b, ob, k)
        for p, q in zip(a, b):
            assert torch.equal(p.detach(), q.detach())
            for n in ("exp_avg", "exp_avg_sq"):
                assert torch.equal(oa.state[p][n], ob.state[q][n])


@pytest.mark.gpu
@pytest.mark.parametrize("limit", [None, 0.3])
@pytest.mark.parametrize("used", [False, True])
def test_the_step_counter_is_part_of_the_state(limit, used):
    """without it a resumed fit corrects its moments as if they had just begun"""
    import copy
    a, b = torch.nn.Parameter(randn((300,), 1)), torch.nn.Parameter(randn((300,), 1))
    oa, ob = NV.HipAdam([a], lr=1e-2, max_grad_norm=limit), NV.HipAdam([b], lr=1e-2, max_grad_norm=limit)
    assert ob.state_dict()["step"] == 0
    if used:
        b.grad = randn((300,), 9)
        ob.step()
    for k in range(3):
        a.grad = randn((300,), 10 + k)
        oa.step()
    with torch.no_grad():
        b.copy_(a)
    saved = copy.deepcopy(oa.state_dict())
    assert saved["step"] == 3
    ob.load_state_dict(saved)
    for k in range(2):
        a.grad, b.grad = randn((300,), 20 + k), randn((300,), 20 + k)
        oa.step()
        ob.step()
        assert torch.equal(a.detach(), b.detach()) and int(ob.step_count) == 4 + k
    ob.load_state_dict({k: v for k, v in saved.items() if k != "step"})          # a state without one: the counter stays
    assert int(ob.step_count) == 5
    fresh = NV.HipAdam([b], lr=1e-2, max_grad_norm=limit)
    fresh.load_state_dict(copy.deepcopy(saved))
    fresh.reset_state()
    assert fresh.state_dict()["step"] == 0 and not fresh.state_dict()["state"]
