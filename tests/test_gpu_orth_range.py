"""rtat_newton_schulz with coefficients that take singular values far above one between steps: up
to 60 has to fit.  G is of rank one, so that one singular value follows the polynomials of the
steps exactly and the error is that of a chain of scalars."""
import pytest

import linear_ref as ref

pytestmark = pytest.mark.gpu
QUINTIC = (3.4445, -4.7750, 2.0315)
HALF = 2.0 ** -11           # half a step of f16, relative

RISING = [
    [(8, 0, 0), (1.5, -0.5, 0)], [(4, 0, 0), QUINTIC], [(9, 0, 0), (1, 0, 0)], [(59, 0, 0), (0.01, 0, 0)],
    [(55, 0, 0), (1.5, -0.5, 0)], [(55, 0, 0), QUINTIC], [(2, 0, 0)] * 5 + [(0.1, 0, 0)], [(300, 0, 0)],
    [(30, 0, 0), (-0.25, 0.002, 0), (1, -0.0002, 0), (2, -0.01, 0)]]


def _bound(coeffs):
    """Relative error of the result.  In step i let u = s^2 and p = a + b u + c u^2.  X, M and P are
    each rounded to f16, element by element and so by at most HALF of their norm, which for rank
    one is the singular value's.  To first order an error of X reaches the step's result times
    k = (|a| + 3 |b| u + 5 |c| u^2) / |p| (at a right angle to G's direction times |a| / |p|, which
    is less), one of M times (|b| u + 2 |c| u^2) / |p|, one of P times (|a| + |b| u + |c| u^2) / |p|,
    and the steps that follow multiply it by their k.  A tenth is added for second order and f32 sums; the
    result is rounded to bf16 (2^-9 relative)."""
    s, err = 1.0, 0.0
    for a, b, c in coeffs:
        u = s * s
        p = abs(a + b * u + c * u * u)
        of_x = (abs(a) + 3 * abs(b) * u + 5 * abs(c) * u * u) / p
        of_m = (abs(b) * u + 2 * abs(c) * u * u) / p
        of_p = (abs(a) + abs(b) * u + abs(c) * u * u) / p
        err = (err + HALF) * of_x + HALF * (of_m + of_p)
        s = s * p
    return 1.1 * err + 2.0 ** -9


def _largest_between(coeffs):
    s, top = 1.0, 1.0
    for a, b, c in coeffs[:-1]:
        s *= abs(a + b * s * s + c * s ** 4)
        top = max(top, s)
    return top


@pytest.mark.parametrize("which", ["f32", "bf16"])
@pytest.mark.parametrize("m,n", [(1, 1), (60, 33), (100, 70), (70, 100), (300, 200), (200, 300)])
@pytest.mark.parametrize("coeffs", RISING, ids=lambda c: "-".join("%g" % s[0] for s in c))
def test_singular_values_up_to_sixty(handle, which, m, n, coeffs):
    import torch
    from rtatblas_amd import native
    assert _largest_between(coeffs) <= 60
    gen = torch.Generator(device="cuda").manual_seed(m + 7 * n)
    # Powers of two, so that G is of rank one in bf16 too.
    u, v = (torch.exp2(torch.randint(-3, 4, (k,), generator=gen, device="cuda").float()) for k in (n, m))
    G = (u[:, None] * v[None, :]).to({"f32": torch.float32, "bf16": torch.bfloat16}[which])
    O = torch.full((n, m), float("nan"), dtype=torch.bfloat16, device="cuda")
    handle.newton_schulz({"f32": native.TYPE_F32, "bf16": native.TYPE_BF16}[which], m, n, G, m, O, m, coeffs)
    want = ref.newton_schulz(G, coeffs)
    assert ((O.double() - want).norm() / want.norm()).item() <= _bound(coeffs)


@pytest.mark.parametrize("m,n", [(90, 128), (700, 600)])
def test_growth_that_the_matrix_does_not_reach(handle, m, n):
    """Coefficients that could take a singular value of one past 60, on a matrix whose largest stays
    near one: the polynomial is then held with the room for 60.  At most 2.9e-3 emulated, with the
    scales for one as with these; the bound is that of the usual steps."""
    import torch
    from rtatblas_amd import native
    coeffs = [(4.0, 0.0, 0.0)] + [QUINTIC] * 5
    gen = torch.Generator(device="cuda").manual_seed(m)
    G = torch.randn(n, m, generator=gen, device="cuda")
    O = torch.empty(n, m, dtype=torch.bfloat16, device="cuda")
    handle.newton_schulz(native.TYPE_F32, m, n, G, m, O, m, coeffs)
    want = ref.newton_schulz(G, coeffs)
    assert ((O.double() - want).norm() / want.norm()).item() <= 2.0 ** -9 + 3e-3
