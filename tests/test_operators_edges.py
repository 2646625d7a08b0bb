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
