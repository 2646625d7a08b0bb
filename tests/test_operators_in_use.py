"""The clipped update and the 4-bit products where the framework itself calls them: the PCA texture space with a 4-bit basis (host model, kernels, captured step against the
oracle), trackers with a largest gradient norm (eager, captured, sharded), the landmark networks' pointwise convolutions."""
import os
import socket

import numpy as np
import pytest
import torch

from tests.test_gradnorm import coefficient, near_norm, norm64
from tests.test_mx import check_sum, quantize64, values64
from tests.test_texpca import _oracle, _space


# ---- the texture space ----
def test_quantize_host_is_the_definition():
    from vhap_amd import mx
    g = torch.Generator().manual_seed(1)
    x = torch.randn(40, 100, generator=g) * torch.exp(3 * torch.randn(40, 1, generator=g))
    x[3], x[5, 40] = 0, float("nan")
    x[6, 99], x[7] = float("inf"), torch.randn(100, generator=g) * 1e-40
    x[8, :8] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0])
    x[9] = torch.randn(100, generator=g) * 2.0 ** -125
    x[10, 0] = 3.4028234663852886e38
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        y = x.clamp(-6e4, 6e4).to(dt) if dt == torch.float16 else x.to(dt)
        q = mx.quantize_host(y)
        want, byte = quantize64(y)
        assert torch.equal(q.scales.long(), byte)
        got = values64(q)
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want)) and torch.equal(got.isnan(), want.isnan())
    with pytest.raises(TypeError):
        mx.quantize_host(x.double())
    with pytest.raises(ValueError):
        mx.quantize_host(x[:, :0])


@pytest.mark.parametrize("n_tex,T", [(100, 512), (33, 256)])
def test_tex_pca_with_a_4_bit_basis_is_the_model_of_that_basis(n_tex, T):
    from vhap_amd.flame import FlameTexPCA
    sp = _space()
    m = FlameTexPCA(n_tex, tex_size=T, tex_space=sp, basis_format="mxfp4")
    assert m.basis_codes.dtype == torch.uint8 and not hasattr(m, "texture_basis")
    held = m.mx_basis().dequantize()
    basis = torch.from_numpy(sp["tex_dir"]).reshape(-1, 200)[:, :n_tex]
    most = torch.nn.functional.pad(basis.abs(), (0, -n_tex % 32)).view(basis.shape[0], -1, 32).amax(-1).repeat_interleave(32, -1)[:, :n_tex]
    assert bool(((held - basis).abs() <= torch.maximum(basis.abs() / 4, most / 16)).all())          # the bound that the class states
    ref = FlameTexPCA(n_tex, tex_size=T, tex_space={"mean": sp["mean"], "tex_dir": held.numpy().reshape(512, 512, 3, n_tex)})
    code = torch.randn(2, n_tex, generator=torch.Generator().manual_seed(2))
    assert float((m(code) - ref(code)).detach().abs().max()) < 2e-6
    with pytest.raises(ValueError):
        FlameTexPCA(n_tex, tex_size=T, tex_space=sp, basis_format="int4")


@pytest.mark.gpu
@pytest.mark.parametrize("n_tex,T", [(100, 1024), (50, 256), (200, 384)])
def test_tex_pca_mx4_kernels_match_the_model(n_tex, T):
    from vhap_amd import _lib
    from vhap_amd.flame import FlameTexPCA
    L, p = _lib.lib(), (lambda t: t.data_ptr())
    m = FlameTexPCA(n_tex, tex_size=T, tex_space=_space(), basis_format="mxfp4").cuda()
    code = (torch.randn(n_tex, generator=torch.Generator().manual_seed(n_tex + T)) * 2).cuda().requires_grad_()
    ref = m(code[None])[0]
    S, w, mean = m.src_size, m.mx_basis(), m.texture_mean.reshape(-1).contiguous()
    src, base, term = torch.empty(S * S * 3, device="cuda"), torch.empty(3, T, T, device="cuda"), torch.zeros(1, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    _lib.check(L.vhap_tex_pca_mx4_fwd(p(mean), p(w.codes), p(w.scales), p(code.detach()), n_tex, S, T, 0.25, p(src), p(base), p(term), st), "fwd")
    # one product behind both; then the kernel divides by 255 (one rounding) where torch multiplies by 1 / 255 (two): 3 units of 2^-24 of numbers up to 1
    assert float((base - ref.detach()).abs().max()) <= 3 * 2.0 ** -24
    W, c64 = values64(w), code.detach().cpu().double()
    check_sum(src, mean.cpu().double() + W @ c64, mean.cpu().double().abs() + W.abs() @ c64.abs(), 3 * n_tex + 1, torch.float32)
    assert abs(float(term) - 0.25 * float((c64 ** 2).sum())) < 1e-5 * float(term)
    d_base = torch.randn(3, T, T, device="cuda")
    (ref * d_base).sum().backward()
    want = code.grad + 2 * 0.25 * code.detach()
    work, d_code, ones = torch.empty(S * S * 3, device="cuda"), torch.zeros(n_tex, device="cuda"), torch.ones(1, device="cuda")
    nbytes = L.vhap_tex_pca_mx4_bwd_workspace_bytes(n_tex, S)
    ws = torch.empty(nbytes // 4, device="cuda")
    args = (p(w.codes), p(w.scales), p(src), p(d_base), p(code.detach()), n_tex, S, T, 0.25, p(ones), p(work), p(ws))
    assert L.vhap_tex_pca_mx4_bwd(*args, nbytes - 4, p(d_code), st) == _lib.E_WORKSPACE
    _lib.check(L.vhap_tex_pca_mx4_bwd(*args, nbytes, p(d_code), st), "bwd")
    assert float((d_code - want).abs().max() / want.abs().max()) < 1e-4
    first = d_code.clone()
    _lib.check(L.vhap_tex_pca_mx4_bwd(*args, nbytes, p(d_code), st), "bwd")      # adds, and the same bits every time
    again = torch.zeros_like(d_code)
    _lib.check(L.vhap_tex_pca_mx4_bwd(*args, nbytes, p(again), st), "bwd")
    assert torch.equal(again, first) and float((d_code - 2 * first).abs().max()) <= 2.0 ** -22 * float(d_code.abs().max())


def _tracker(flame_model, device="cuda", T=512, H=128, W=128, N=2, seed=3, mx_basis=False, max_grad_norm=None):
    from vhap_amd.config import BaseTrackingConfig
    from vhap_amd.synthetic import make_texture, smooth_noise
    from vhap_amd.tracker import GlobalTracker
    model, topo = flame_model
    cfg = BaseTrackingConfig()
    cfg.device, cfg.model.tex_resolution, cfg.lr.max_grad_norm = device, T, max_grad_norm
    if mx_basis:
        cfg.model.tex_painted, cfg.model.tex_basis_format = False, "mxfp4"
    data = {"rgb": torch.from_numpy(smooth_noise(np.random.default_rng(seed), (N, 3, H, W))).to(device),
            "lmk2d": torch.cat([torch.rand(N, 70, 2, generator=torch.Generator().manual_seed(2)) * W, torch.ones(N, 70, 1)], -1).to(device)}
    tr = GlobalTracker(cfg, model, topo, _space() if mx_basis else make_texture(0, T), data)
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for name, s in (("shape", 0.3), ("expr", 0.3), ("rotation", 0.05), ("jaw_pose", 0.05), ("tex_extra", 0.03), ("lights", 0.05), ("tex_pca", 1.5)):
            if getattr(tr, name, None) is not None:
                getattr(tr, name).add_((torch.randn(getattr(tr, name).shape, generator=g) * s).to(device))
        tr.translation[:, 2] += 0.45
    if device == "cuda":
        tr.render.disturb_rate_fg = tr.render.disturb_rate_bg = None
    return tr, cfg


@pytest.mark.gpu
def test_native_step_with_a_4_bit_basis_matches_the_oracle_on_that_basis(flame_model):
    from vhap_amd.step import NativeStep
    from vhap_amd.tracker import GraphedStep
    stage, H = "rgb_global_tracking", 128
    tr, cfg = _tracker(flame_model, mx_basis=True)
    tr.get_train_parameters(stage)
    sample = tr.get_sample(np.arange(2), device_index=True)
    ns = NativeStep(tr, sample, stage)
    assert ns.pca_mx is not None
    ns.forward()
    ns.backward(1)
    torch.cuda.synchronize()
    n = int(tr.tex_pca.shape[0])
    held = np.zeros((512 * 512 * 3, 200), np.float32)
    held[:, :n] = ns.pca_mx.dequantize().cpu().numpy()
    sp = {"mean": _space()["mean"], "tex_dir": held}
    Eo, logo, P, _ = _oracle(tr, cfg, flame_model, sp, sample, stage, (H, H), tid=(ns.rast[..., 3].long() - 1).cpu())
    got = {k: float(v) for k, v in ns.log_dict().items()}
    Eo = Eo.detach()
    assert abs(got["total"] - float(Eo)) <= 5e-5 * abs(float(Eo)) and abs(got["reg_tex_pca"] - float(logo["reg_tex_pca"].detach())) <= 5e-5 * abs(float(logo["reg_tex_pca"].detach()))
    for k in ("tex_pca", "tex_extra", "shape", "lights"):
        a, b = ns.g[k].detach().cpu().double().reshape(-1), P[k].grad.reshape(-1)
        off = (a - b).abs()
        if k == "tex_extra":
            # |residual| has a kink at 0: a pixel channel whose residual is a rounding of 0 counts -1 here and +1 there, 2 w_photo / (3 n_pixels) times a shading of at most 2,
            # spread over the at most 8 texels it is sampled from.  Two such channels among the 98304 are let pass, nothing else
            flip = 2 * 2 * float(cfg.w.photo) / (3 * 2 * H * H)
            out = off > 1e-3 * float(b.abs().max())
            assert int(out.sum()) <= 16 and float(off.max()) <= flip, (int(out.sum()), float(off.max()), flip)
            continue
        assert float(off.max() / b.abs().max()) < 1e-3, k
    # captured, and with the gradients clipped
    tr.cfg.lr.max_grad_norm = 1.0
    opt = tr.configure_optimizer(tr.get_train_parameters(stage), lr_scale=0.1)
    before = tr.tex_pca.detach().clone()
    st = GraphedStep(tr, sample, opt, stage, warmup=0)
    assert st.ns is not None and st.ns.pca_mx is not None and st.gF.plan is not None
    E = [float(st()) for _ in range(5)]
    torch.cuda.synchronize()
    assert abs(E[0] - float(Eo)) <= 1e-4 * abs(float(Eo)) and E[-1] < E[0] and float((tr.tex_pca.detach() - before).abs().max()) > 0


# ---- trackers with a largest gradient norm ----
def _first_step_is_clipped_adam(st_params, before, opt, share):
    """after ONE step from zero moments: every parameter moved by lr g c / (|g c| + 1e-8) with c from the norm over all gradients"""
    grads = [p.grad.detach().clone() for p in st_params]
    n = norm64(grads, 2.0)
    assert near_norm(float(opt.grad_norm), n) and n > 0
    c = coefficient(n, opt.max_grad_norm)
    assert (c < 1) == (share < 1)
    lr = {id(p): float(g["lr"]) for g in opt.param_groups for p in g["params"]}
    for p, b, g in zip(st_params, before, grads):
        gc, b64 = g.double().cpu() * c, b.double().cpu()
        want = b64 - lr[id(p)] * gc / (gc.abs() + 1e-8)
        # the move is a quotient near 1 of numbers rounded a few times each (under 40 units of 2^-24; where |g c| is near 1e-8 the fp32 sum under the root loses no more),
        # and p rounds once more
        assert bool(((p.detach().double().cpu() - want).abs() <= lr[id(p)] * 40 * 2.0 ** -24 + 2.0 ** -24 * b64.abs() + 2.0 ** -24 * lr[id(p)]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("stage", ["rgb_global_tracking", "rgb_init_texture", "lmk_init_all"])
@pytest.mark.parametrize("share", [0.1, 10.0])
def test_captured_step_with_clipped_gradients(flame_model, stage, share):
    from vhap_amd.tracker import GraphedStep
    tr, cfg = _tracker(flame_model, T=256)
    opt = tr.configure_optimizer(tr.get_train_parameters(stage))
    assert opt.max_grad_norm is None
    sample = tr.get_sample(np.arange(2), device_index=True)
    probe = GraphedStep(tr, sample, opt, stage, warmup=0)                        # (learning rate as configured; what it says is the size of the gradients)
    keep = {id(p): p.detach().clone() for p in probe.params}
    os.environ["VHAP_TEX_KEEP_GRAD"] = "1"
    try:
        probe = GraphedStep(tr, sample, opt, stage, warmup=0)
    finally:
        os.environ.pop("VHAP_TEX_KEEP_GRAD")
    probe()
    torch.cuda.synchronize()
    size = norm64([p.grad for p in probe.params if p.grad is not None], 2.0)
    with torch.no_grad():
        for p in probe.params:
            p.copy_(keep[id(p)])
    tr.cfg.lr.max_grad_norm = size * share
    opt = tr.configure_optimizer(tr.get_train_parameters(stage))
    assert opt.max_grad_norm == size * share
    st = GraphedStep(tr, sample, opt, stage, warmup=0)
    assert st.ns is not None and st.ns.step_optimizer is None and st.gF.plan is not None
    before = [p.detach().clone() for p in st.params]
    E = [float(st())]
    torch.cuda.synchronize()
    _first_step_is_clipped_adam(st.params, before, opt, share)
    for _ in range(4):
        E.append(float(st()))
    assert np.isfinite(E).all() and int(opt.step_count) == 5
    with st.replay_stream():
        for _ in range(3):
            st()
    torch.cuda.synchronize()
    assert int(opt.step_count) == 8 and np.isfinite(float(st.E))


@pytest.mark.gpu
def test_eager_step_with_clipped_gradients(flame_model):
    tr, cfg = _tracker(flame_model, T=128, max_grad_norm=0.5)
    opt = tr.configure_optimizer(tr.get_train_parameters("rgb_global_tracking"))
    params = [p for g in opt.param_groups for p in g["params"]]
    before = [p.detach().clone() for p in params]
    tr.optimize_iter(tr.get_sample(np.arange(2)), opt, "rgb_global_tracking")
    live = [(p, b) for p, b in zip(params, before) if p.grad is not None]
    _first_step_is_clipped_adam([p for p, _ in live], [b for _, b in live], opt, 0.1)
    # torch's optimiser (the host formulation): clipped in place ahead of it
    tr.native = False
    opt = tr.configure_optimizer(tr.get_train_parameters("rgb_global_tracking"))
    assert isinstance(opt, torch.optim.Adam)
    tr.optimize_iter(tr.get_sample(np.arange(2)), opt, "rgb_global_tracking")
    n = norm64([p.grad for g in opt.param_groups for p in g["params"] if p.grad is not None], 2.0)
    assert abs(n - 0.5) <= 0.5 * 2.0 ** -20


@pytest.mark.gpu
def test_an_optimiser_that_does_not_clip_by_itself(flame_model):
    """a HipAdam made without the limit: the eager step clips in place ahead of it, the captured step (which updates inside its plan) refuses it"""
    from vhap_amd.native import HipAdam
    from vhap_amd.tracker import GraphedStep
    tr, cfg = _tracker(flame_model, T=128, max_grad_norm=0.5)
    made = tr.configure_optimizer(tr.get_train_parameters("rgb_global_tracking"))
    opt = HipAdam([{"params": g["params"], "lr": g["lr"]} for g in made.param_groups])
    tr.optimize_iter(tr.get_sample(np.arange(2)), opt, "rgb_global_tracking")
    n = norm64([p.grad for g in opt.param_groups for p in g["params"] if p.grad is not None], 2.0)
    assert abs(n - 0.5) <= 0.5 * 2.0 ** -20
    with pytest.raises(ValueError, match="max_grad_norm"):
        GraphedStep(tr, tr.get_sample(np.arange(2), device_index=True), opt, "rgb_global_tracking", warmup=0)


@pytest.mark.gpu
@pytest.mark.parametrize("stage", ["lmk_init_all"])
def test_captured_step_with_torchs_optimiser(flame_model, stage):
    """torch.optim.Adam inside the captured native step: clipped in place ahead of it"""
    from vhap_amd.tracker import GraphedStep
    tr, cfg = _tracker(flame_model, T=128, max_grad_norm=1e-3)
    made = tr.configure_optimizer(tr.get_train_parameters(stage))
    opt = torch.optim.Adam([{"params": g["params"], "lr": g["lr"]} for g in made.param_groups], capturable=True)
    st = GraphedStep(tr, tr.get_sample(np.arange(2), device_index=True), opt, stage, warmup=0)
    for _ in range(3):
        st()
        torch.cuda.synchronize()
        n = norm64([p.grad for p in st.params if p.grad is not None], 2.0)
        assert abs(n - 1e-3) <= 1e-3 * 2.0 ** -18                                # (two roundings an element, and 1e-6 in the factor's denominator below 2^-18 of the norm)


def test_clipping_on_the_host(flame_model):
    """a CPU tracker's landmark stage: torch's optimiser behind torch's clipping"""
    tr, cfg = _tracker(flame_model, device="cpu", T=64, H=32, W=32, max_grad_norm=0.25)
    opt = tr.configure_optimizer(tr.get_train_parameters("lmk_init_all"))
    tr.optimize_iter(tr.get_sample(np.arange(2)), opt, "lmk_init_all")
    n = norm64([p.grad for g in opt.param_groups for p in g["params"] if p.grad is not None], 2.0)
    assert abs(n - 0.25) <= 0.25 * 2.0 ** -18


def _sharded(rank, world, port, ret):
    import torch.distributed as dist
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    from tests.test_dist_gpu import _build
    from vhap_amd import dist as vdist
    from vhap_amd.tracker import GraphedStep
    tr = _build(128)
    tr.cfg.lr.max_grad_norm = 1.0
    vdist.attach(tr)
    opt = tr.configure_optimizer(tr.get_train_parameters("rgb_global_tracking"), lr_scale=0.1)
    st = GraphedStep(tr, tr.get_sample(np.asarray([0, 1] if rank == 0 else [2, 3]), device_index=True), opt, "rgb_global_tracking", warmup=0)
    assert not st.tex_sharded
    for _ in range(3):
        st()
    torch.cuda.synchronize()
    ret[rank] = (float(opt.grad_norm), [p.detach().cpu() for p in (tr.shape, tr.tex_extra, tr.lights, tr.focal_length)])
    dist.destroy_process_group()


@pytest.mark.gpu
def test_two_ranks_clip_by_the_norm_of_the_averaged_gradients():
    import torch.multiprocessing as mp
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    port = s.getsockname()[1]
    s.close()
    ret = mp.Manager().dict()
    mp.spawn(_sharded, args=(2, port, ret), nprocs=2, join=True)
    assert ret[0][0] == ret[1][0] and ret[0][0] > 0                              # the same norm on both ranks, so the same factor
    assert all(torch.equal(a, b) for a, b in zip(ret[0][1], ret[1][1]))          # and the shared parameters stay replicas


# ---- the landmark networks ----
@pytest.mark.gpu
@pytest.mark.parametrize("N,H,W,Cin,Cout,relu", [(2, 4, 4, 256, 256, True), (1, 64, 64, 256, 68, False), (1, 9, 7, 68, 256, False), (3, 32, 32, 1024, 256, True)])
def test_pointwise_convolution_in_4_bits(N, H, W, Cin, Cout, relu):
    from vhap_amd import landmarks as LM
    g = torch.Generator().manual_seed(Cin + Cout)
    w, bias = torch.randn(Cout, Cin, 1, 1, generator=g) / Cin ** 0.5, torch.randn(Cout, generator=g)
    conv = LM._Conv(w, bias, out_relu=relu, pointwise="mxfp4")
    assert conv.mx_w is not None
    x = torch.randn(N, H, W, Cin, generator=g).cuda()
    y = LM.new_conv(conv, x)
    assert y.shape == (N, H, W, Cout) and y.dtype == torch.float32
    A, B = quantize64(x.view(-1, Cin))[0], quantize64(w.view(Cout, Cin))[0]
    want = A @ B.t() + bias.double()
    check_sum(y.view(-1, Cout), want.clamp(min=0) if relu else want, A.abs() @ B.abs().t() + bias.double().abs(), Cin + 1, torch.float32)
    for kw in (dict(pad=1), dict(stride=2), dict(in_relu=True)):                 # what is no plain pointwise convolution stays one in fp32
        assert LM._Conv(w if "pad" not in kw else torch.randn(Cout, Cin, 3, 3, generator=g), bias, pointwise="mxfp4", **kw).mx_w is None
    with pytest.raises(ValueError):
        LM._Conv(w, bias, pointwise="int4")


@pytest.mark.gpu
def test_networks_run_with_4_bit_pointwise_convolutions():
    from oracle import fan_ref, sfd_ref
    from vhap_amd.face_detector import S3FD
    from vhap_amd.landmarks import FAN2D
    x = torch.rand(2, 3, 64, 64, generator=torch.Generator().manual_seed(1)).cuda()
    sd = fan_ref.random_fan(seed=3, num_modules=2).state_dict()
    a, b = FAN2D(sd, num_modules=2)(x), FAN2D(sd, num_modules=2, pointwise="mxfp4")(x)
    assert len(b) == 2 and all(u.shape == v.shape and bool(torch.isfinite(v).all()) and not torch.equal(u, v) for u, v in zip(a, b))
    sd = sfd_ref.random_s3fd(seed=3).state_dict()
    x = torch.randn(1, 128, 160, 3, generator=torch.Generator().manual_seed(2)).cuda() * 50
    a, b = S3FD(sd)(x), S3FD(sd, pointwise="mxfp4")(x)
    assert all(u.shape == v.shape and bool(torch.isfinite(v).all()) for p, q in zip(a, b) for u, v in zip(p, q))
    assert all(torch.equal(u, v) for p, q in zip(a[:3], b[:3]) for u, v in zip(p, q)) and not torch.equal(a[3][0], b[3][0])     # the heads in front of fc7 are untouched
