"""Microscaled 4-bit floating point (MXFP4): matrices held in 4.25 bits an element, and products with them (vhap_amd/csrc/mx.hip).

Rows are cut into blocks of 32 elements: 32 codes of E2M1 (+-{0, 0.5, 1, 1.5, 2, 3, 4, 6}) and one power-of-two scale a block (E8M0: 2^(byte - 127), byte 255 is NaN).

    w  = quantize(x)                      x [..., K] float32 / bfloat16 / float16 -> MXTensor
    x' = w.dequantize(torch.float32)      the values it holds
    y  = linear(x, w, bias)               x [..., K] float, w [N, K] in 4 bits: y [..., N] in x's type; differentiable in x and bias, w is constant
    dx = linear_input_grad(g, w)          what linear's backward computes, g [..., N] -> [..., K]
    y  = matmul(a, b, bias, relu)         both in 4 bits: [M, N] = a [M, K] b [N, K]^T

What it is for here: the linear spaces a fit reads whole in every step and never trains -- the FLAME texture basis, 315 MB in float32, 42 MB like this
(FlameTexPCA(basis_format="mxfp4")) -- and the pointwise convolutions of the landmark networks (pointwise="mxfp4").

All calls enqueue on the current stream of the tensors' device, allocate what they need through torch, and never synchronise.  No CPU path: CPU tensors raise
(MXTensor.dequantize excepted, which also runs on the CPU, in torch operations, for checks and for host-side models)."""
import torch

from . import _lib
from .native import _DTYPE_CODE, on_device
from .ops import _p, _stream

BLOCK = 32


def _chk(rc, what):
    _lib.check(rc, what)


class MXTensor:
    """[..., K] numbers in 4 bits: `codes` uint8 [..., 16 Kb], `scales` uint8 [..., Kb], Kb = ceil(K / 32), both contiguous.  Codes behind K are not read as
    numbers.  `shape` is that of the numbers."""

    def __init__(self, codes, scales, shape):
        shape = torch.Size(int(n) for n in shape)
        if len(shape) < 1 or shape[-1] < 1:
            raise ValueError(f"MXTensor: at least one axis, and at least one element along the last; got {tuple(shape)}")
        kb = -(-shape[-1] // BLOCK)
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError(f"MXTensor: codes and scales are uint8, got {codes.dtype} and {scales.dtype}")
        if codes.shape != shape[:-1] + (16 * kb,) or scales.shape != shape[:-1] + (kb,):
            raise ValueError(f"MXTensor of {tuple(shape)}: codes {tuple(shape[:-1]) + (16 * kb,)}, scales {tuple(shape[:-1]) + (kb,)}; got {tuple(codes.shape)} and "
                             f"{tuple(scales.shape)}")
        if codes.device != scales.device:
            raise ValueError("MXTensor: codes and scales on one device")
        if not codes.is_contiguous() or not scales.is_contiguous() or (codes.numel() and codes.data_ptr() % 16):
            raise ValueError("MXTensor: contiguous codes and scales, the codes 16-byte aligned")
        self.codes, self.scales, self.shape = codes, scales, shape

    @property
    def device(self):
        return self.codes.device

    @property
    def rows(self):
        return self.scales.numel() // self.scales.shape[-1]

    def to(self, device):
        return MXTensor(self.codes.to(device), self.scales.to(device), self.shape)

    def nbytes(self):
        return self.codes.numel() + self.scales.numel()

    def __repr__(self):
        return f"MXTensor({tuple(self.shape)}, device={self.device})"

    @torch.no_grad()
    def dequantize(self, dtype=torch.float32):
        """the numbers as float32 or bfloat16 (both hold them exactly) or float16 (which rounds, and overflows above 65504)"""
        if dtype not in _DTYPE_CODE:
            raise TypeError(f"dequantize to float32, bfloat16 or float16, got {dtype}")
        K = self.shape[-1]
        if self.codes.is_cuda:
            out = torch.empty(self.shape, dtype=dtype, device=self.device)
            with on_device(out):
                _chk(_lib.lib().vhap_mx4_dequantize(_p(self.codes), _p(self.scales), self.rows, K, _p(out), _DTYPE_CODE[dtype], _stream()), "vhap_mx4_dequantize")
            return out
        values = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
        values = torch.cat([values, -values])
        pair = torch.stack([self.codes & 15, self.codes >> 4], -1).flatten(-2).long()
        scale = torch.ldexp(torch.ones((), dtype=torch.float64), self.scales.int() - 127)
        scale = torch.where(self.scales == 255, torch.full_like(scale, float("nan")), scale).repeat_interleave(BLOCK, -1)
        return (values.double()[pair] * scale)[..., :K].to(dtype)


def _floats(t, what):
    if not torch.is_tensor(t) or t.dtype not in _DTYPE_CODE:
        raise TypeError(f"{what}: a float32, bfloat16 or float16 tensor, got {t.dtype if torch.is_tensor(t) else type(t).__name__}")


def _on_hip(t, what):
    if t.device.type != "cuda":
        raise RuntimeError(f"{what}: tensors on a HIP device (no CPU fallback)")


def _rows(t):
    """[..., K] -> (rows, row stride, tensor): a matrix with consecutive elements along K; anything else is copied"""
    t = t.reshape(-1, t.shape[-1]) if t.dim() != 2 else t
    if t.shape[1] > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t.shape[0], (t.stride(0) if t.shape[0] > 1 else t.shape[1]), t


def _matrix(w, what):
    if not isinstance(w, MXTensor):
        raise TypeError(f"{what}: an MXTensor, got {type(w).__name__}")
    if len(w.shape) != 2:
        raise ValueError(f"{what}: a matrix, got {tuple(w.shape)}")


@torch.no_grad()
def quantize(x):
    """x [..., K] -> MXTensor of the same shape: blocks of 32 along the last axis.  The scale is the power of two that puts a block's largest magnitude into
    [4, 8); codes are the nearest ones, halves to the even code, magnitudes above 6 become 6.  A block with a NaN or an infinity becomes NaN as a whole."""
    _floats(x, "quantize")
    _on_hip(x, "quantize")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"quantize: at least one element along the last axis, got {tuple(x.shape)}")
    K, kb = x.shape[-1], -(-x.shape[-1] // BLOCK)
    codes = torch.empty(x.shape[:-1] + (16 * kb,), dtype=torch.uint8, device=x.device)
    scales = torch.empty(x.shape[:-1] + (kb,), dtype=torch.uint8, device=x.device)
    rows, ld, x2 = _rows(x.detach())
    with on_device(codes):
        _chk(_lib.lib().vhap_mx4_quantize(_p(x2), _DTYPE_CODE[x.dtype], ld, rows, K, _p(codes), _p(scales), _stream()), "vhap_mx4_quantize")
    return MXTensor(codes, scales, x.shape)


def _check_bias(bias, n, device, what):
    if bias is None:
        return None
    if not torch.is_tensor(bias) or bias.dtype != torch.float32 or bias.shape != (n,):
        raise ValueError(f"{what}: a float32 bias of {n} elements")
    if bias.device != device:
        raise ValueError(f"{what}: the bias on {device}, got {bias.device}")
    return bias.detach().contiguous()


def _linear(x, w, bias):
    M, ld, x2 = _rows(x)
    y = torch.empty(x.shape[:-1] + (w.shape[0],), dtype=x.dtype, device=x.device)
    with on_device(y):
        _chk(_lib.lib().vhap_mx4_linear(_p(x2), _DTYPE_CODE[x.dtype], ld, M, _p(w.codes), _p(w.scales), w.shape[0], w.shape[1], _p(bias), _p(y), _stream()),
             "vhap_mx4_linear")
    return y


def _input_grad(g, w):
    L = _lib.lib()
    N, K = w.shape
    dx = torch.empty(g.shape[:-1] + (K,), dtype=g.dtype, device=g.device)
    M, ld, g2 = _rows(g)
    nbytes = L.vhap_mx4_linear_input_grad_workspace_bytes(M, N, K)
    ws = torch.empty(nbytes // 4, dtype=torch.float32, device=g.device)
    with on_device(dx):
        _chk(L.vhap_mx4_linear_input_grad(_p(g2), _DTYPE_CODE[g.dtype], ld, M, _p(w.codes), _p(w.scales), N, K, _p(ws), nbytes, _p(dx), 0, _stream()),
             "vhap_mx4_linear_input_grad")
    return dx


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, bias, w):
        ctx.w = w
        return _linear(x, w, None if bias is None else bias.contiguous())

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        w, dx, db = ctx.w, None, None
        if ctx.needs_input_grad[0]:
            dx = _input_grad(g, w)
        if ctx.needs_input_grad[1]:
            M, ld, g2 = _rows(g)
            db = torch.empty(w.shape[0], dtype=torch.float32, device=g.device)
            with on_device(db):
                _chk(_lib.lib().vhap_mx4_column_sums(_p(g2), _DTYPE_CODE[g.dtype], ld, M, w.shape[0], _p(db), _stream()), "vhap_mx4_column_sums")
        return dx, db, None


def _check_pair(x, w, axis, what):
    _floats(x, what)
    _matrix(w, what)
    if x.dim() < 1 or x.shape[-1] != w.shape[axis]:
        raise ValueError(f"{what}: {w.shape[axis]} elements along the last axis for a matrix of {tuple(w.shape)}, got {tuple(x.shape)}")
    if x.device != w.device:
        raise ValueError(f"{what}: tensors on one device, got {x.device} and {w.device}")
    _on_hip(x, what)


def linear(x, w, bias=None):
    """y [..., N] = x [..., K] w^T (+ bias): w an MXTensor [N, K], x float32 / bfloat16 / float16, bias float32 [N]; y in x's type.  The products are exact,
    the sums are float32 in a fixed order, y is rounded once.  Gradients flow to x and bias (once: not twice differentiable)."""
    _check_pair(x, w, 1, "linear")
    _check_bias(bias, w.shape[0], x.device, "linear")
    return _Linear.apply(x, bias, w)


@torch.no_grad()
def linear_input_grad(g, w):
    """dx [..., K] = g [..., N] w for an MXTensor w [N, K]: the gradient of linear's input from that of its output, in g's type"""
    _check_pair(g, w, 0, "linear_input_grad")
    if w.shape[0] == 0:
        return torch.zeros(g.shape[:-1] + (w.shape[1],), dtype=g.dtype, device=g.device)
    return _input_grad(g, w)


@torch.no_grad()
def matmul(a, b, bias=None, relu=False, out_dtype=torch.float32):
    """[M, N] = a [M, K] b [N, K]^T (+ bias float32 [N], then optionally a ReLU), both MXTensors; float32 sums, rounded to out_dtype once.  Not
    differentiable: both operands are codes."""
    _matrix(a, "matmul")
    _matrix(b, "matmul")
    if a.shape[1] != b.shape[1]:
        raise ValueError(f"matmul: operands of one K, got {tuple(a.shape)} and {tuple(b.shape)}")
    if a.device != b.device:
        raise ValueError(f"matmul: tensors on one device, got {a.device} and {b.device}")
    if out_dtype not in _DTYPE_CODE:
        raise TypeError(f"matmul to float32, bfloat16 or float16, got {out_dtype}")
    _on_hip(a, "matmul")
    bias = _check_bias(bias, b.shape[0], a.device, "matmul")
    y = torch.empty(a.shape[0], b.shape[0], dtype=out_dtype, device=a.device)
    with on_device(y):
        _chk(_lib.lib().vhap_mx4_matmul(_p(a.codes), _p(a.scales), a.shape[0], _p(b.codes), _p(b.scales), b.shape[0], a.shape[1], _p(bias), _p(y),
                                        _DTYPE_CODE[out_dtype], _lib.CONV_OUT_RELU if relu else 0, _stream()), "vhap_mx4_matmul")
    return y
