"""Microscaled 4-bit floating point (MXFP4): matrices held in 17 bytes a block of 32 elements, and products with them (vhap_amd/csrc/mx.hip).

Rows are cut into blocks of 32 elements: 32 codes of E2M1 (+-{0, 0.5, 1, 1.5, 2, 3, 4, 6}) and one power-of-two scale a block (E8M0: 2^(byte - 127), byte 255 is NaN).

    w  = quantize(x)                      x [..., K] float32 / bfloat16 / float16 -> MXTensor
    x' = w.dequantize(torch.float32)      the values it holds
    y  = linear(x, w, bias)               x [..., K] float, w [N, K] in 4 bits: y [..., N] in x's type; differentiable in x and bias, w is constant
    dx = linear_input_grad(g, w)          what linear's backward computes, g [..., N] -> [..., K]
    y  = matmul(a, b, bias, relu)         both in 4 bits: [M, N] = a [M, K] b [N, K]^T

What it is for here: the linear spaces a fit reads whole in every step and never trains -- the FLAME texture basis, 315 MB in float32, 53 MB like this
(FlameTexPCA(basis_format="mxfp4")) -- and the pointwise convolutions of the landmark networks (pointwise="mxfp4").

All calls enqueue on the current stream of the tensors' device, allocate what they need through torch, and never synchronise.  No CPU path: CPU tensors raise
(excepted: MXTensor.dequantize, which also runs on the CPU, and quantize_host, which only does, both in torch operations: for models built on the host)."""
import torch

from . import _lib

BLOCK = 32
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


class MXTensor:
    """[..., K] numbers in 4 bits: `codes` uint8 [..., 16 Kb], `scales` uint8 [..., Kb], Kb = ceil(K / 32), both contiguous.  Codes behind K are not read as
    numbers.  `shape` is that of the numbers.  An element past float32's range (its block's byte 253 or 254: quantize makes none) counts as infinite, and what it
    enters is not finite."""

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

    @classmethod
    def _of(cls, codes, scales, shape):
        t = cls.__new__(cls)                              # (quantize's own results: nothing to check)
        t.codes, t.scales, t.shape = codes, scales, shape
        return t

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

    def dequantize(self, dtype=torch.float32):
        """the numbers as float32 or bfloat16 (both hold them exactly) or float16 (which rounds, and overflows above 65504)"""
        if dtype not in DTYPES:
            raise TypeError(f"dequantize to float32, bfloat16 or float16, got {dtype}")
        K = self.shape[-1]
        if self.codes.is_cuda:
            return _lib.host().dequantize(self.codes, self.scales, K, dtype)
        values = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
        values = torch.cat([values, -values])
        pair = torch.stack([self.codes & 15, self.codes >> 4], -1).flatten(-2).long()
        scale = torch.ldexp(torch.ones((), dtype=torch.float64), self.scales.int() - 127)
        scale = torch.where(self.scales == 255, torch.full_like(scale, float("nan")), scale).repeat_interleave(BLOCK, -1)
        return (values.double()[pair] * scale)[..., :K].to(dtype)


def _matrix(w, what):
    if not isinstance(w, MXTensor):
        raise TypeError(f"{what}: an MXTensor, got {type(w).__name__}")
    if len(w.shape) != 2:
        raise ValueError(f"{what}: a matrix, got {tuple(w.shape)}")
    return w.shape


def quantize(x):
    """x [..., K] -> MXTensor of the same shape: blocks of 32 along the last axis.  The scale is the power of two that puts a block's largest magnitude into
    [4, 8); codes are the nearest ones, halves to the even code, magnitudes above 6 become 6.  A block with a NaN or an infinity becomes NaN as a whole."""
    return MXTensor._of(*_lib.host().quantize(x), x.shape)


def quantize_host(x):
    """quantize of a CPU tensor, in torch operations, to the same codes and scales (a model's constants are laid out once, before they move to the device)"""
    if x.dtype not in DTYPES:
        raise TypeError(f"quantize_host: a float32, bfloat16 or float16 tensor, got {x.dtype}")
    if x.is_cuda or x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"quantize_host: a CPU tensor with at least one element along the last axis, got {tuple(x.shape)} on {x.device}")
    K = x.shape[-1]
    v = torch.nn.functional.pad(x.detach().float().reshape(-1, K), (0, -K % BLOCK)).view(-1, -(-K // BLOCK), BLOCK)
    bits = v.view(torch.int32) & 0x7fffffff
    field = bits.amax(-1) >> 23                                            # the largest exponent field; 255: a NaN or an infinity is among them
    byte = torch.where(field == 255, field, (field - 2).clamp(min=0))
    # x / 2^(byte - 127) without leaving fp32 (exact: powers of two built from their bits; byte 0 in two steps of 2^64 and 2^63)
    up = torch.where(byte == 0, torch.full_like(byte, 127 + 64), torch.full_like(byte, 127))
    rest = torch.where(byte == 0, torch.full_like(byte, 127 + 63), (254 - byte).clamp(min=1))
    s = v.abs() * (up << 23).view(torch.float32)[..., None] * (rest << 23).view(torch.float32)[..., None]
    step = torch.where(s < 2, 0.5, torch.where(s < 4, 1.0, 2.0))
    q = (torch.round(s / step) * step).clamp(max=6.0)                       # halves to even
    code = torch.where(q < 2, 2 * q, torch.where(q < 4, q + 2, q / 2 + 4))  # 0, .5, 1, 1.5 | 2, 3 | 4, 6 -> 0 .. 7
    code = torch.nan_to_num(code, nan=0.0).to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)
    code[byte == 255] = 0
    code = code.reshape(v.shape[0], -1)
    kb = -(-K // BLOCK)
    return MXTensor((code[:, 0::2] | code[:, 1::2] << 4).contiguous().view(x.shape[:-1] + (16 * kb,)), byte.to(torch.uint8).view(x.shape[:-1] + (kb,)).contiguous(), x.shape)


def linear(x, w, bias=None):
    """y [..., N] = x [..., K] w^T (+ bias): w an MXTensor [N, K], x float32 / bfloat16 / float16, bias float32 [N]; y in x's type.  The products are exact,
    the sums are float32 in a fixed order, y is rounded once (float32 numbers below 2^-117 lose their last bits, those below 2^-126 may count as 0).  Gradients
    flow to x and bias (once: not twice differentiable; an input with a forward-mode tangent is refused).  In a stream capture, a differentiable call is refused while
    a graph of the same input made on another stream is alive, or one made on the default stream anywhere behind it: its captured backward would end the process."""
    N, K = _matrix(w, "linear")
    return _lib.host().linear(x, w.codes, w.scales, N, K, bias)


def linear_input_grad(g, w):
    """dx [..., K] = g [..., N] w for an MXTensor w [N, K]: the gradient of linear's input from that of its output, in g's type.  Not differentiable itself."""
    N, K = _matrix(w, "linear_input_grad")
    return _lib.host().input_grad(g, w.codes, w.scales, N, K)


def matmul(a, b, bias=None, relu=False, out_dtype=torch.float32):
    """[M, N] = a [M, K] b [N, K]^T (+ bias float32 [N], then optionally a ReLU), both MXTensors; float32 sums, rounded to out_dtype once.  Not
    differentiable: both operands are codes."""
    (M, K), (N, Kb) = _matrix(a, "matmul"), _matrix(b, "matmul")
    if K != Kb:
        raise ValueError(f"matmul: operands of one K, got {tuple(a.shape)} and {tuple(b.shape)}")
    if a.codes.device != b.codes.device:
        raise ValueError(f"matmul: tensors on one device, got {a.device} and {b.device}")
    if out_dtype not in DTYPES:
        raise TypeError(f"matmul to float32, bfloat16 or float16, got {out_dtype}")
    return _lib.host().matmul(a.codes, a.scales, b.codes, b.scales, M, N, K, bias, relu, out_dtype)
