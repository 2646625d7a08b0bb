"""The operators of the parameter update and of the 4-bit linear spaces, as measured cases.

    clip      the global norm of a list of gradients, and the gradients scaled to a largest norm
    adam      one Adam step on gradients clipped to a largest global norm
    quantize  numbers to microscaled 4-bit floats (blocks of 32 along the last axis, one power-of-two scale each) and back to the values held
    linear    x W^T + b with W held in microscaled 4-bit floats, and its gradients
    matmul    A B^T + b, both held in microscaled 4-bit floats, with the ReLU of a pointwise convolution

`own` false: elementary torch operations; true: the framework's entry points (vhap_amd.native, vhap_amd.mx)."""
import math

import torch

own = False

VERTS3 = 3 * 5143                     # coordinates of the head mesh
TEXELS3 = 512 * 512 * 3               # channels of the PCA texture grid
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # gradients of a landmark stage of 16 frames: eight tiny tensors, what counts is the latency
        {"name": "clip_landmark_stage", "op": "clip", "set": "tracker", "frames": 16, "tex": 0, "active": True},
        # gradients of a photometric stage: the residual texture (3 x 2048 x 2048) and ten small tensors
        {"name": "clip_photometric_stage", "op": "clip", "set": "tracker", "frames": 64, "tex": 2048, "active": True},
        # gradients of a landmark network: 56 residual blocks, convolutions in bf16 and norms in fp32, views of flat buckets
        {"name": "clip_network_bf16", "op": "clip", "set": "network", "blocks": 56, "width": 256, "active": True},
        # the update behind those two stages
        {"name": "adam_landmark_stage", "op": "adam", "frames": 16, "tex": 0, "active": True},
        {"name": "adam_photometric_stage", "op": "adam", "frames": 64, "tex": 2048, "active": True},
        # the texture basis brought to 4 bits, once per model; values handed on in bf16, which holds them exactly
        {"name": "quantize_texture_basis", "op": "quantize", "rows": TEXELS3, "k": 100, "dtype": "fp32", "back": "bf16"},
        # activations of a deep level on their way into a product, an odd number of rows and columns
        {"name": "quantize_activations_odd", "op": "quantize", "rows": 1023, "k": 257, "dtype": "bf16", "back": "fp32"},
        # base texture from one code, every step of a fit; and the code's gradient
        {"name": "linear_texture_code", "op": "linear", "m": 1, "n": TEXELS3, "k": 100, "dtype": "fp32", "grad": False},
        {"name": "linear_texture_code_grad", "op": "linear", "m": 1, "n": TEXELS3, "k": 100, "dtype": "fp32", "grad": True},
        # vertex offsets of 256 frames from shape and expression, forward and gradients, in bf16
        {"name": "linear_blendshapes_bf16_grad", "op": "linear", "m": 256, "n": VERTS3, "k": 400, "dtype": "bf16", "grad": True},
        # a pointwise convolution of the deepest level of a crop and its mirror image
        {"name": "matmul_pointwise_small", "op": "matmul", "m": 32, "n": 256, "k": 256, "out": "fp32", "relu": False},
        # the face detector's 1024 -> 1024 pointwise layer over 16 frames of 32 x 32
        {"name": "matmul_pointwise_fc7", "op": "matmul", "m": 16384, "n": 1024, "k": 1024, "out": "bf16", "relu": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["clip", "adam", "quantize", "linear", "linear", "matmul"])
    if op == "clip" and rng.random() < 0.5:
        return {"op": op, "set": "network", "blocks": _log_int(rng, 1, 56), "width": rng.choice([64, 100, 128, 256]), "active": rng.random() < 0.75}
    if op in ("clip", "adam"):
        c = {"op": op, "frames": _log_int(rng, 1, 4000), "tex": rng.choice([0, _log_int(rng, 16, 1900)]), "active": rng.random() < 0.75}
        return {**c, "set": "tracker"} if op == "clip" else c
    if op == "quantize":
        k = _log_int(rng, 1, 1200)
        return {"op": op, "rows": _log_int(rng, 1, max(1, min(700000, 60_000_000 // k))), "k": k, "dtype": rng.choice(sorted(DTYPES)), "back": rng.choice(sorted(DTYPES)[::2])}
    if op == "linear":
        m, k = _log_int(rng, 1, 300), _log_int(rng, 1, 512)
        return {"op": op, "m": m, "n": _log_int(rng, 1, max(1, min(700000, 3_900_000 // m))), "k": k, "dtype": rng.choice(sorted(DTYPES)), "grad": rng.random() < 0.5}
    return {"op": op, "m": _log_int(rng, 1, 16000), "n": _log_int(rng, 1, 1024), "k": _log_int(rng, 1, 1024), "out": rng.choice(sorted(DTYPES)), "relu": rng.random() < 0.5}


def _tracker_shapes(case):
    """The parameter tensors of a stage: shape, expression, poses, camera; with a texture the lights, the vertex offset and the texture too."""
    n, t = case["frames"], case["tex"]
    s = [(300,), (n, 100), (n, 3), (n, 3), (n, 3), (n, 3), (n, 6), (1,)]
    return s + [(9, 3), (1, VERTS3 // 3, 3), (3, t, t)] if t else s


def _network_shapes(case):
    """(convolutions, norms) of pre-activation residual blocks of `width` channels: three 3 x 3 convolutions and three norms each."""
    w = case["width"]
    conv = [(w // 2, w, 3, 3), (w // 4, w // 2, 3, 3), (w // 4, w // 4, 3, 3)] * case["blocks"]
    norm = [(w,), (w,), (w // 2,), (w // 2,), (w // 4,), (w // 4,)] * case["blocks"]
    return conv, norm


def _sizes(case):
    """Numbers of elements as (fp32, bf16) of a list of gradients."""
    if case.get("set") == "network":
        conv, norm = _network_shapes(case)
        return sum(math.prod(s) for s in norm), sum(math.prod(s) for s in conv)
    return sum(math.prod(s) for s in _tracker_shapes(case)), 0


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, shape, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda") * scale


def _views(flat, shapes):
    at, out = 0, []
    for s in shapes:
        n = math.prod(s)
        out.append(flat[at:at + n].view(s))
        at += n
    return out


def _codes(g, rows, k):
    """Random microscaled 4-bit numbers: codes [rows, 16 * blocks] (two a byte, the even element in the low half; zero behind k) and scale
    bytes [rows, blocks] (exponent + 127) around 1 / 8."""
    blocks = -(-k // 32)
    byte = torch.randint(0, 256, (rows, blocks * 16), generator=g, device="cuda", dtype=torch.uint8)
    at = torch.arange(blocks * 16, device="cuda") * 2
    byte &= torch.where(at + 1 < k, 255, torch.where(at < k, 15, 0)).to(torch.uint8)
    return byte, torch.randint(121, 128, (rows, blocks), generator=g, device="cuda", dtype=torch.uint8)


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    if op in ("clip", "adam"):
        st = {"op": op}
        if case.get("set") == "network":
            conv, norm = _network_shapes(case)
            flat32, flat16 = (sum(math.prod(s) for s in x) for x in (norm, conv))
            st["flat"] = [_randn(g, (flat32,), 1e-2), _randn(g, (flat16,), 1e-3).to(torch.bfloat16)]
            st["grads"] = _views(st["flat"][0], norm) + _views(st["flat"][1], conv)
            st["results"] = [torch.empty_like(f) for f in st["flat"]]
            st["out"] = _views(st["results"][0], norm) + _views(st["results"][1], conv)
        else:
            # gradients of very different sizes side by side: 1e-4 .. 1 by tensor
            shapes = _tracker_shapes(case)
            st["grads"] = [_randn(g, s, 10.0 ** -(i % 5)) for i, s in enumerate(shapes)]
            st["results"] = st["out"] = [torch.empty_like(x) for x in st["grads"]]
        expected = math.sqrt(sum(float(x.float().square().sum()) for x in st.get("flat", st["grads"])))
        st["max_norm"] = expected * (0.3 if case["active"] else 3.0)
        if op == "adam":
            st.update(lr=[5e-3, 5e-4], betas=(0.9, 0.999), eps=1e-8, t=1)
            st["p"] = [_randn(g, x.shape, 0.1) for x in st["grads"]]
            st["m"] = [_randn(g, x.shape, 10.0 ** -(i % 5)) * 0.1 for i, x in enumerate(st["grads"])]
            st["v"] = [_randn(g, x.shape, 10.0 ** -(i % 5)).square() * 0.1 for i, x in enumerate(st["grads"])]
            del st["out"], st["results"]
            if own:
                # the optimiser that the program keeps, in the middle of a run: one step counted, moments in place
                from vhap_amd.native import HipAdam
                first, last = st["p"][:-1], st["p"][-1:]
                opt = HipAdam([{"params": first, "lr": st["lr"][0]}, {"params": last, "lr": st["lr"][1]}], betas=st["betas"], eps=st["eps"], max_grad_norm=st["max_norm"])
                for p, x, m, v in zip(st["p"], st["grads"], st["m"], st["v"]):
                    p.grad = x
                    opt.state[p].update(exp_avg=m, exp_avg_sq=v)
                opt.advance()
                st["opt"] = opt
        return st
    if op == "quantize":
        x = _randn(g, (case["rows"], case["k"])) * torch.exp(_randn(g, (case["rows"], 1), 1.5))        # rows of different size
        x[torch.rand((case["rows"],), generator=g, device="cuda") < 0.02] = 0                           # and some of nothing
        return {"op": op, "x": x.to(DTYPES[case["dtype"]]), "back": DTYPES[case["back"]]}
    if op == "linear":
        dt = DTYPES[case["dtype"]]
        codes, scales = _codes(g, case["n"], case["k"])
        st = {"op": op, "x": _randn(g, (case["m"], case["k"])).to(dt), "codes": codes, "scales": scales, "bias": _randn(g, (case["n"],)), "grad": case["grad"]}
        if case["grad"]:
            st["x"].requires_grad_()
            st["g"] = _randn(g, (case["m"], case["n"])).to(dt)
        if own:
            from vhap_amd import mx
            st["w"] = mx.MXTensor(codes, scales, (case["n"], case["k"]))
        return st
    a, b = _codes(g, case["m"], case["k"]), _codes(g, case["n"], case["k"])
    st = {"op": op, "a": a, "b": b, "k": case["k"], "bias": _randn(g, (case["n"],)), "relu": case["relu"], "out": DTYPES[case["out"]]}
    if own:
        from vhap_amd import mx
        st["am"], st["bm"] = mx.MXTensor(*a, (case["m"], case["k"])), mx.MXTensor(*b, (case["n"], case["k"]))
    return st


def _coefficient(flat32, max_norm):
    norm = flat32.square().sum().sqrt()
    return norm, torch.clamp(max_norm / (norm + 1e-6), max=1.0)


def _power(e):
    """2^e in 32 bits, -126 <= e <= 127, from the bits: a library's power need not be exact, and values on a border would fall to either side."""
    return ((e + 127) << 23).view(torch.float32)


def _values(codes, scales, k):
    """The numbers that codes and scales stand for, [rows, k] in 32 bits."""
    pair = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()
    magnitude, exponent = pair & 7, pair >> 1 & 3
    size = torch.where(exponent == 0, magnitude * 0.5, ((2 + (pair & 1)) << exponent) * 0.25)
    scale = _power(scales.int() - 127).repeat_interleave(32, -1)
    return (torch.where(pair >= 8, -size, size) * scale)[:, :k]


def _held(x):
    """The values of x [rows, k] after quantisation, in 32 bits."""
    rows, k = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -k % 32)).view(rows, -1, 32)
    most = x.abs().amax(-1, keepdim=True)
    e = torch.clamp(torch.frexp(most).exponent - 3, min=-125)             # floor(log2(most)) - 2
    s = x.abs() * _power(-e)
    step = torch.where(s < 2, 0.5, torch.where(s < 4, 1.0, 2.0))
    q = torch.clamp(torch.round(s / step) * step, max=6.0)                 # halves to even: the code whose last bit is 0
    q = torch.where(most == 0, torch.zeros_like(q), q * _power(e))
    return torch.copysign(q, x).view(rows, -1)[:, :k]


def run(state):
    op = state["op"]
    if op == "clip":
        if own:
            from vhap_amd import native
            _, norm = native.clip_by_global_norm(state["grads"], state["max_norm"], out=state["out"])
            return {"norm": norm, "clipped": state["results"]}
        flats = state["flat"] if "flat" in state else [torch.cat([x.reshape(-1) for x in state["grads"]])]
        norm, c = _coefficient(torch.cat([f.float() for f in flats]), state["max_norm"])
        done = [(f.float() * c).to(f.dtype) for f in flats]
        if "flat" not in state:
            done = [d.view(x.shape) for d, x in zip(done[0].split([x.numel() for x in state["grads"]]), state["grads"])]
        return {"norm": norm, "clipped": done}
    if op == "adam":
        if own:
            state["opt"].step()
            return {"norm": state["opt"].grad_norm, "p": state["p"], "m": state["m"], "v": state["v"]}
        state["t"] += 1
        b1, b2 = state["betas"]
        norm, c = _coefficient(torch.cat([x.reshape(-1) for x in state["grads"]]), state["max_norm"])
        root = math.sqrt(1 - b2 ** state["t"])
        for i, (p, g, m, v) in enumerate(zip(state["p"], state["grads"], state["m"], state["v"])):
            lr = state["lr"][1 if i == len(state["p"]) - 1 else 0]
            g = g * c
            m.add_((g - m) * (1 - b1))
            v.mul_(b2).add_(g * g * (1 - b2))
            p.sub_(lr / (1 - b1 ** state["t"]) * m / (v.sqrt() / root + state["eps"]))
        return {"norm": norm, "p": state["p"], "m": state["m"], "v": state["v"]}
    if op == "quantize":
        if own:
            from vhap_amd import mx
            return mx.quantize(state["x"]).dequantize(state["back"])
        return _held(state["x"]).to(state["back"])
    if op == "linear":
        x = state["x"]
        if own:
            from vhap_amd import mx
            if not state["grad"]:
                return {"y": mx.linear(x, state["w"], state["bias"])}
            bias = state["bias"].detach().requires_grad_()
            y = mx.linear(x, state["w"], bias)
            dx, db = torch.autograd.grad(y, (x, bias), state["g"])
            return {"y": y.detach(), "dx": dx, "db": db}
        w = _values(state["codes"], state["scales"], x.shape[1])
        y = (x.detach().float() @ w.t() + state["bias"]).to(x.dtype)
        if not state["grad"]:
            return {"y": y}
        g = state["g"].float()
        return {"y": y, "dx": (g @ w).to(x.dtype), "db": g.sum(0)}
    if own:
        from vhap_amd import mx
        return mx.matmul(state["am"], state["bm"], bias=state["bias"], relu=state["relu"], out_dtype=state["out"])
    y = _values(*state["a"], state["k"]) @ _values(*state["b"], state["k"]).t() + state["bias"]
    return (torch.clamp(y, min=0) if state["relu"] else y).to(state["out"])


def work(case):
    op = case["op"]
    if op == "clip":
        n32, n16 = _sizes(case)
        return {"bytes": 2 * (4 * n32 + 2 * n16) + 4, "flops": 3 * (n32 + n16)}
    if op == "adam":
        n = _sizes(case)[0]
        return {"bytes": 28 * n + 4, "flops": 16 * n}
    size = {"fp32": 4, "bf16": 2, "fp16": 2}
    k = case["k"]
    row = -(-k // 32) * 17                                   # codes and scales of a row
    if op == "quantize":
        return {"bytes": case["rows"] * (k * (size[case["dtype"]] + size[case["back"]]) + row), "flops": 4 * case["rows"] * k}
    m, n = case["m"], case["n"]
    if op == "linear":
        s = size[case["dtype"]]
        once = {"bytes": n * (row + 4) + s * (m * k + m * n), "flops": 2 * m * n * k}
        if case["grad"]:
            once["bytes"] += s * (m * n + m * k) + 4 * n
            once["flops"] += 2 * m * n * k + m * n
        return once
    return {"bytes": (m + n) * row + 4 * n + size[case["out"]] * m * n, "flops": 2 * m * n * k}


# ---- the definitions in 64 bits ----
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _table64(codes, scales, k):
    """Code by code from the table of the eight magnitudes."""
    table = torch.tensor(E2M1 + [-v for v in E2M1], dtype=torch.float64, device=codes.device)
    out = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.float64, device=codes.device)
    out[:, 0::2], out[:, 1::2] = table[(codes % 16).long()], table[(codes // 16).long()]
    return (out.view(codes.shape[0], -1, 32) * (2.0 ** (scales.double() - 127))[:, :, None]).flatten(1)[:, :k]


def _nearest64(x):
    """The nearest of the fifteen values of each block's grid; between two of them the one with an even code."""
    x = x.double()
    k = x.shape[1]
    done = torch.empty_like(x)
    for at in range(0, k, 32):
        b = x[:, at:at + 32]
        most = b.abs().max(1, keepdim=True).values
        scale = ((most.view(torch.int64) >> 52) - 2 << 52).view(torch.float64)       # the power of two at or below `most`, over four
        scale = torch.where(most > 0, scale, torch.ones_like(most))
        v, best, far = (b / scale).abs(), torch.zeros_like(b), torch.full_like(b, math.inf)
        for value in [E2M1[i] for i in (0, 2, 4, 6, 1, 3, 5, 7)]:                   # the even codes first, so that a tie stays theirs
            d = (v - value).abs()
            best, far = torch.where(d < far, value, best), torch.minimum(d, far)
        done[:, at:at + 32] = torch.where(b < 0, -best, best) * scale * (most > 0)
    return done


def exact(case, seed):
    st, op = prepare(case, seed), case["op"]
    if op in ("clip", "adam"):
        g = [x.double() for x in (st["flat"] if "flat" in st else st["grads"])]
        norm = torch.stack([(x * x).sum() for x in g]).sum().sqrt()
        c = min(1.0, st["max_norm"] / (float(norm) + 1e-6))
        if op == "clip":
            return {"norm": norm, "clipped": [x * c for x in g]}
        b1, b2 = st["betas"]
        m = [b1 * x.double() + (1 - b1) * c * y for x, y in zip(st["m"], g)]
        v = [b2 * x.double() + (1 - b2) * (c * y) ** 2 for x, y in zip(st["v"], g)]
        lr = [st["lr"][0]] * (len(g) - 1) + [st["lr"][1]]
        p = [x.double() - r * (y / (1 - b1 ** 2)) / ((z / (1 - b2 ** 2)).sqrt() + st["eps"]) for x, y, z, r in zip(st["p"], m, v, lr)]
        return {"norm": norm, "p": p, "m": m, "v": v}
    if op == "quantize":
        return _nearest64(st["x"])
    if op == "linear":
        x, w = st["x"].detach().double(), _table64(st["codes"], st["scales"], case["k"])
        y = torch.matmul(x, w.transpose(0, 1).contiguous()) + st["bias"].double()
        if not case["grad"]:
            return {"y": y}
        g = st["g"].double()
        return {"y": y, "dx": torch.matmul(g, w), "db": g.sum(0)}
    y = torch.matmul(_table64(*st["a"], case["k"]), _table64(*st["b"], case["k"]).transpose(0, 1).contiguous()) + st["bias"].double()
    return y.clamp(min=0) if case["relu"] else y
