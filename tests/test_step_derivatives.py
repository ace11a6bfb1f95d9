"""Derivatives of the operators around a decoding step: rotary has both kinds, the others raise instead of leaving
one out. On the CPU by tensors without contents; the values on the GPU."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from nkilab import ops

BF, E4M3, E8M0 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu
B, T, H, HKV, D = 2, 5, 4, 2, 64


def m(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


def turn(x, freqs=None):
    return ops.rotary(x, m(B, dtype=torch.int32), m(16, dtype=torch.float64) if freqs is None else freqs)


def test_a_turn_has_a_forward_derivative():
    for needs in (False, True):  # a gradient as well
        x, dx = m(B, T, H, D).requires_grad_(needs), m(B, T, H, D)
        with fwAD.dual_level():
            out = fwAD.unpack_dual(turn(fwAD.make_dual(x, dx)))
            assert out.tangent is not None and out.tangent.shape == x.shape
            assert out.primal.requires_grad == needs
            if needs:
                assert torch.autograd.grad(out.primal.sum(), x)[0].shape == x.shape
            assert fwAD.unpack_dual(turn(x)).tangent is None
            with pytest.raises(RuntimeError, match="freqs"):
                f = m(16, dtype=torch.float64)
                turn(x, fwAD.make_dual(f, m(16, dtype=torch.float64)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF])
def test_the_forward_derivative_is_the_same_turn(dtype):
    """The operator is linear, so that the tangent comes out of the same call, bit for bit."""
    g = torch.Generator(device="cuda").manual_seed(8)
    x, dx, y = (torch.randn(B, T, H, D, generator=g, device="cuda").to(dtype) for _ in range(3))
    at, parents = torch.tensor([3, 70], dtype=torch.int32, device="cuda"), torch.tensor([[-1, 0, 0, 2, -1]] * B, dtype=torch.int32, device="cuda")
    f = ops.rotary_frequencies(32)[0]

    def call(t):
        return ops.rotary(t, at, f, parents, True, 1.25)

    out, tangent = torch.func.jvp(call, (x,), (dx,))
    assert torch.equal(out, call(x)) and torch.equal(tangent, call(dx))
    # forward over reverse: half the sum of squares has the gradient R^T R x, whose derivative along dx is R^T R dx
    # (torch.func.grad does not take operators with a C++ gradient: it raises)
    leaf = x.clone().requires_grad_()
    with fwAD.dual_level():
        loss = 0.5 * (call(fwAD.make_dual(leaf, dx)).float() ** 2).sum()
        grad, moved = fwAD.unpack_dual(torch.autograd.grad(loss, leaf)[0])
        grad, moved = grad.clone(), moved.clone()
    assert torch.equal(grad, torch.autograd.grad(0.5 * (call(leaf).float() ** 2).sum(), leaf)[0])
    # The turn's transpose after the turn is the magnitude squared. With p = |x1| + |x2| of a pair, the turned entries are up
    # to 1.25 p, rounded by half a step each (bf16 2^-8), and the two turned back again bring 2 x 2^-8 x 1.25^2 p, the
    # last rounding 2^-8 x 1.25^2 p; in fp32 sines, products and sums are some sixteen roundings of 2^-24.
    bound = (3 * 2.0 ** -8 if dtype == BF else 0.0) + 2e-6
    pair = dx.float().abs().clone()
    pair[..., :32] = dx.float()[..., :32].unflatten(-1, (16, 2)).abs().sum(-1, keepdim=True).expand(B, T, H, 16, 2).flatten(-2)
    want = dx.double()
    want[..., :32] *= 1.25 ** 2
    assert ((moved.double() - want).abs() <= bound * 1.25 ** 2 * pair + 1e-30).all()
    with fwAD.dual_level():  # both kinds at once
        leaf = x.clone().requires_grad_()
        out = fwAD.unpack_dual(call(fwAD.make_dual(leaf, dx)))
        assert torch.equal(out.tangent, call(dx))
        assert torch.equal(torch.autograd.grad((out.primal * y).sum(), leaf)[0], torch.autograd.grad((call(leaf) * y).sum(), leaf)[0])


def others():
    i32, e4m3, e8m0 = (lambda *s: m(*s, dtype=torch.int32)), m(20, HKV, 16, D, dtype=E4M3), m(20, HKV, 2, dtype=E8M0)
    q, k, v, f = m(B, T, H, D), m(B, T, HKV, D), m(B, T, HKV, D), m(16, dtype=torch.float64)
    cache, tables, lens = m(20, HKV, 16, D), i32(B, 3), i32(B)
    out = []
    for at in range(3):
        def put(t, at=at):
            return tuple(t if i == at else x for i, x in enumerate((q, k, v)))

        x = (q, k, v)[at]
        out += [(x, lambda t, p=put: ops.attention_tree(*p(t), cache, cache, tables, lens)),
                (x, lambda t, p=put: ops.attention_tree(*p(t), e4m3, e4m3, tables, lens, None, None, e8m0, e8m0)),
                (x, lambda t, p=put: ops.rotary_append(*p(t), cache, cache, tables, lens, f)[at % 2]),
                (x, lambda t, p=put: ops.rotary_append(*p(t), e4m3, e4m3, tables, lens, f, k_scales=e8m0, v_scales=e8m0)[1])]
    out.append((cache, lambda t: ops.attention_tree(q, k, v, t, cache, tables, lens)))
    out.append((m(B, 50), lambda t: ops.sample(t, m(B))[1]))
    out.append((m(B), lambda t: ops.sample(m(B, 50), m(B), t)[1]))
    return out


@pytest.mark.parametrize("at", range(len(others())))
def test_the_others_raise(at):
    x, call = others()[at]
    with fwAD.dual_level(), pytest.raises(NotImplementedError, match="forward"):
        call(fwAD.make_dual(x, torch.empty_like(x)))
    with pytest.raises(NotImplementedError, match="forward"):
        torch.func.jvp(call, (x,), (torch.empty_like(x),))
    out = call(x.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="not implemented"):
        out.sum().backward()
    assert not call(x).requires_grad
