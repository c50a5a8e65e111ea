"""rtat_newton_schulz on the GPU against the same iteration in 64 bits.  The relative error in
2-norm is at most 2^-9 from rounding the result to bf16 (half a step) and 3e-3 from the f16
products: twice the largest error of an emulation of them on the CPU over four kinds of spectra."""
import pytest

import linear_ref as ref

pytestmark = pytest.mark.gpu
QUINTIC = (3.4445, -4.7750, 2.0315)
BOUND = 2.0 ** -9 + 3e-3


def _types():
    import torch
    from rtatblas_amd import native
    return {"bf16": (torch.bfloat16, native.TYPE_BF16), "f16": (torch.float16, native.TYPE_F16),
            "f32": (torch.float32, native.TYPE_F32)}


def _update(gen, b, n, m, kind):
    """b matrices, row-major (n, m) = column-major m x n."""
    import torch
    g = torch.randn(b, n, m, generator=gen, device="cuda")
    if kind == "strong":        # sixteen strong directions over a floor of 1 %
        r = min(16, n, m)
        g = torch.bmm(torch.randn(b, n, r, generator=gen, device="cuda"),
                      torch.randn(b, r, m, generator=gen, device="cuda")) / 4 + 0.01 * g
    return g


def _run(handle, which, G, coeffs, pad=0, inplace=False):
    import torch
    dt, ty = _types()[which]
    b, n, m = G.shape
    full = torch.full((b, n, m + pad), float("nan"), dtype=dt, device="cuda")
    full[..., :m] = G.to(dt)
    O = full if inplace else torch.full((b, n, m + pad), float("nan"), dtype=torch.bfloat16, device="cuda")
    src = full.clone()
    handle.newton_schulz(ty, m, n, full, m + pad, O, m + pad, coeffs, batch=b, strideg=n * (m + pad), strideo=n * (m + pad))
    assert bool(torch.isnan(O[..., m:]).all())
    return src[..., :m], O[..., :m]


def _check(src, O, coeffs, bound=BOUND):
    for g, o in zip(src, O):
        want = ref.newton_schulz(g, coeffs)
        assert ((o.double() - want).norm() / want.norm()).item() <= bound


@pytest.mark.parametrize("which", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kind", ["noise", "strong"])
@pytest.mark.parametrize("m,n", [(1, 1), (1, 50), (33, 20), (64, 64), (128, 128), (100, 300), (300, 100), (129, 127),
                                 (500, 64), (257, 640), (768, 520)])
def test_shapes(handle, which, kind, m, n):
    coeffs = [QUINTIC] * 5
    gen = __import__("torch").Generator(device="cuda").manual_seed(m * 31 + n)
    src, O = _run(handle, which, _update(gen, 1, n, m, kind), coeffs, pad=(m + n) % 4)
    _check(src, O, coeffs)


@pytest.mark.parametrize("m,n", [(4100, 4200), (4250, 4099), (2048, 4100), (3000, 1990)])
def test_large(handle, m, n):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(m)
    src, O = _run(handle, "bf16", _update(gen, 1, n, m, "strong"), [QUINTIC] * 5)
    _check(src, O, [QUINTIC] * 5)


@pytest.mark.parametrize("steps", [1, 2, 3, 6])
def test_steps_and_other_coefficients(handle, steps):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(steps)
    coeffs = [(3.4445 - 0.1 * i, -4.7750 + 0.1 * i, 2.0315) for i in range(steps)]
    for m, n in ((96, 200), (200, 96)):
        src, O = _run(handle, "f32", _update(gen, 1, n, m, "noise"), coeffs)
        _check(src, O, coeffs)
    # Newton's cubic
    src, O = _run(handle, "bf16", _update(gen, 1, 64, 64, "noise"), [(1.5, -0.5, 0.0)] * steps)
    _check(src, O, [(1.5, -0.5, 0.0)] * steps)


@pytest.mark.parametrize("m,n", [(72, 40), (130, 260), (260, 130)])
def test_batch_and_in_place(handle, m, n):
    import torch
    coeffs = [QUINTIC] * 5
    gen = torch.Generator(device="cuda").manual_seed(m)
    G = _update(gen, 5, n, m, "noise") * torch.tensor([1.0, 1e-6, 1e6, 1e-3, 1.0], device="cuda")[:, None, None]
    src, O = _run(handle, "bf16", G, coeffs, pad=2)
    _check(src, O, coeffs)
    src2, O2 = _run(handle, "bf16", G, coeffs, pad=2, inplace=True)
    assert torch.equal(O, O2)
    for i in range(5):          # each matrix alone gives the same bits
        _, one = _run(handle, "bf16", G[i:i + 1], coeffs, pad=2)
        assert torch.equal(one[0], O[i])


@pytest.mark.parametrize("m,n", [(48, 80), (200, 150)])
def test_scales_zero_and_not_finite(handle, m, n):
    """Norms far outside f32's squares, a zero matrix, and one matrix of a batch that holds an
    infinity or a NaN: its result is NaN throughout, the others are as without it."""
    import torch
    coeffs = [QUINTIC] * 5
    gen = torch.Generator(device="cuda").manual_seed(n)
    base = _update(gen, 6, n, m, "noise")
    G = base.clone()
    G[1] *= 1e30
    G[2] = 0
    G[3, 4, 5] = float("inf")
    G[4, 7, 1] = float("nan")
    src, O = _run(handle, "f32", G, coeffs)
    _check(src[[0, 1, 5]], O[[0, 1, 5]], coeffs)
    assert bool((O[2] == 0).all()) and bool(torch.isnan(O[3:5]).all())
    _, plain = _run(handle, "f32", base, coeffs)
    assert torch.equal(plain[0], O[0]) and torch.equal(plain[5], O[5])
    # without eps only a zero norm is undefined; a tiny one is not
    dt, ty = _types()["f32"]
    tiny = (base[:1] * 1e-36).contiguous()
    o = torch.empty(1, n, m, dtype=torch.bfloat16, device="cuda")
    handle.newton_schulz(ty, m, n, tiny, m, o, m, coeffs, eps=0.0)
    want = ref.newton_schulz(tiny[0].double() * 1e36, coeffs, 0.0)
    assert ((o[0].double() - want).norm() / want.norm()).item() <= BOUND
