"""The activations of the experts' block by themselves: one row, one non-zero element in it and in every
weight row, so that the projections are products of two numbers of the type, which fp32 holds exactly,
dh is 1, and `saved.h` and the weights' gradients are h, dg and du themselves.

Tolerance: one rounding to the type, and what the fp32 evaluation may be off by, relative to the terms of
a(g) and a'(g): (g^2 + 16) 2^-23.  (The exponent g^2 / 2 has a rounding or two, 2^-24 of it each, and the
approximate exponential is off by (2 + 1.18 g^2 / 2) 2^-23: less than (2 + 0.9 g^2) 2^-23 together, for silu's,
whose exponent is g, less than (3 + 1.2 |g|) 2^-23.  The other factor of Phi is a fit, 1.3 2^-23, with the
roundings of its sum, 2.5 2^-23, and of an approximate quotient, 2 2^-23 twice at most; products and sums
around them add fewer than ten half units.)"""
from __future__ import annotations

import math

import pytest

from conftest import gpu_count

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("reach", [8.0, 12.0])
def test_activations_keep_their_precision_in_the_tails(reach, dtype, act):
    from ugdr_b200 import ops

    if gpu_count() < 1:
        pytest.skip("no GPU")
    dtype, inner, hidden = getattr(torch, dtype), 4096, 8
    g = torch.linspace(-reach, reach, inner, dtype=torch.float64).to(dtype).cuda()
    u = torch.tensor([1.0, -0.75, 1.5, 0.3125], dtype=dtype, device="cuda").repeat(inner // 4)
    x, dy = (torch.zeros(1, hidden, dtype=dtype, device="cuda") for _ in range(2))
    w_in, w_out = torch.zeros(1, 2, inner, hidden, dtype=dtype, device="cuda"), torch.zeros(1, hidden, inner, dtype=dtype,
                                                                                          device="cuda")
    x[0, 0], dy[0, 1], w_out[0, 1], w_in[0, 0, :, 0], w_in[0, 1, :, 0] = 1, 1, 1, g, u
    counts = torch.ones(1, dtype=torch.int32, device="cuda")
    y, saved = ops.expert_ffn_train(x, counts, w_in, w_out, act=act)
    _, dw_in, dw_out = ops.expert_ffn_backward(dy, x, counts, w_in, w_out, saved, act=act)
    ops.check_status()
    assert torch.equal(saved.gu[0, 0], g.float()) and torch.equal(saved.gu[0, 1], u.float())
    assert torch.equal(dw_out[0, 1], saved.h[0])

    g, u = g.double(), u.double()
    if act == "silu":
        s = torch.sigmoid(g)
        a, terms = g * s, (s, s * g * (1 - s))
    else:
        p = 0.5 * torch.special.erfc(-g / math.sqrt(2))
        a, terms = g * p, (p, g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi))
    f, step = torch.finfo(dtype), (g * g + 16) * 2.0 ** -23
    for got, want, size in ((saved.h[0], a * u, (a * u).abs()),
                            (dw_in[0, 0, :, 0], sum(terms) * u, sum(t.abs() for t in terms) * u.abs()),
                            (dw_in[0, 1, :, 0], a, a.abs())):
        off = step * size
        off = off + (want.abs() + off) * f.eps / 2 + f.smallest_normal * f.eps / 2
        bad = ~((got.double() - want).abs() <= off)
        assert not bool(bad.any()), (f"{int(bad.sum())} of {inner}, first at g = {float(g[bad][0])}: {float(got[bad][0])} "
                                     f"for {float(want[bad][0])}")
