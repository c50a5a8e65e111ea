"""16-bit products whose operands are laid out anew before the product: one of them or both, k padded
or not, every op combination, and the gradient's form, whose partial sums share the scratch with the
copies.  And direct loads at the largest leading dimension they take."""
import pytest

import linear_ref as ref
from test_gpu_linear import Mat, N, T, _gen, _op, _types, _within

pytestmark = pytest.mark.gpu


def _odd(r, c, dt, gen, scale=1.0):
    """Columns an odd number of elements apart."""
    return Mat(r, c, dt, 1 - r % 2, 1, gen, scale)


def _even(r, c, dt, gen, scale=1.0):
    """Columns on sixteen bytes."""
    return Mat(r, c, dt, -r % 8, 0, gen, scale)


def _lent(h, nbytes, form):
    """Runs form() with a lent buffer of that size; returns whether the buffer was written."""
    import torch
    ws = torch.full((nbytes,), 0xa5, dtype=torch.uint8, device="cuda")
    h.set_workspace(ws, nbytes)
    form()
    torch.cuda.synchronize()
    return bool((ws != 0xa5).any())


@pytest.mark.parametrize("ta", [N, T])
@pytest.mark.parametrize("tb", [N, T])
@pytest.mark.parametrize("packed", ["a", "b", "ab"])
@pytest.mark.parametrize("which,size", [("bf16", (1101, 1203, 1003)), ("f16", (2051, 640, 1090)), ("bf16", (1024, 1500, 1152))])
def test_packed_forward_and_gradient(ta, tb, packed, which, size):
    """The buffer is written, so the product was packed; 1 KiB of it is too little, so it was not: both
    within the bounds, nothing outside the results touched."""
    import torch
    from rtatblas_amd import native
    dt, ty = _types()[which]
    m, n, k = size
    gen = _gen(m + n + ta + 2 * tb)
    A = (_odd if "a" in packed else _even)(*((k, m) if ta == T else (m, k)), dt, gen, k ** -0.5)
    B = (_odd if "b" in packed else _even)(*((n, k) if tb == T else (k, n)), dt, gen)
    bias, C, Z = Mat(m, 1, dt, 0, 0, gen), Mat(m, n, dt, 3, 1, gen), Mat(m, n, dt, 2, 0, gen, 2.0)
    opA, opB = _op(A.m, ta), _op(B.m, tb)
    (y, yb), _ = ref.forward(0.75, opA, opB, k, bias.m[:, 0], ref.SILU, -1.0, C.m, dt, dt)
    g, e = ref.product(1.5, opA, opB, k)
    dz, de = g * ref.slope(Z.m.double(), ref.GELU), 1.13 * e + 2 * (ref.SLOPE_ERR + ref.U) * g.abs()
    h = native.Handle(torch.cuda.current_stream())
    lib = native.load()
    try:
        def forward():
            D = Mat(m, n, dt, 1, 0)
            h.gemm_ep(ty, ta, tb, m, n, k, 0.75, A.ptr, A.ld, B.ptr, B.ld, D.ptr, D.ld, act=ref.SILU, bias=bias.ptr, beta=-1.0,
                      C=C.ptr, ldc=C.ld)
            assert _within(D.m, y, yb) and D.padding_kept()

        def gradient():
            D, db = Mat(m, n, dt, 1, 0), torch.full((m,), float("nan"), device="cuda")
            h.gemm_dact(ty, ta, tb, m, n, k, 1.5, A.ptr, A.ld, B.ptr, B.ld, ref.GELU, Z.ptr, Z.ld, D.ptr, D.ld, dbias=db)
            assert _within(D.m, dz, ref.rounded(dz, de, dt)) and D.padding_kept()
            assert _within(db, dz.sum(1), de.sum(1) + (n + 2) * ref.U * dz.abs().sum(1))

        sums = lib.rtat_dbias_workspace_bytes(m, n)
        assert _lent(h, 16 << 20, forward) and not _lent(h, 1 << 10, forward)
        assert _lent(h, 16 << 20, gradient) and _lent(h, sums, gradient)
        # The handle's own scratch grows for the copies while the sums have their place in the old block.
        h.set_workspace(None, 0)
        gradient()
        gradient()
        forward()
        assert A.padding_kept() and B.padding_kept() and C.padding_kept() and Z.padding_kept()
    finally:
        torch.cuda.synchronize()
        h.close()


@pytest.mark.parametrize("which", ["bf16", "f16"])
@pytest.mark.parametrize("far", ["a", "b"])
def test_direct_loads_at_the_largest_leading_dimension(handle, which, far):
    """Rows 2^23 - 8 elements apart: the last row of a tile of 256 starts 4.28e9 bytes behind its first,
    within the 32 bits of an offset.  The sizes take the largest tile."""
    import torch
    dt, ty = _types()[which]
    ld, k, small, large = (1 << 23) - 8, 128, 512, 32768
    gen = _gen(9)
    buf = torch.empty(ld * (small - 1) + k, dtype=dt, device="cuda")
    X = torch.as_strided(buf, (k, small), (1, ld))
    X.copy_((torch.randn(k, small, generator=gen, device="cuda") * k ** -0.5).to(dt))
    W = Mat(k, large, dt, 0, 0, gen)
    if far == "a":
        D = Mat(small, large, dt)
        handle.gemm_ep(ty, T, N, small, large, k, 1.0, buf, ld, W.ptr, W.ld, D.ptr, D.ld)
        y, e = ref.product(1.0, X.T, W.m, k)
    else:
        D = Mat(large, small, dt)
        handle.gemm_ep(ty, T, N, large, small, k, 1.0, W.ptr, W.ld, buf, ld, D.ptr, D.ld)
        y, e = ref.product(1.0, W.m.T, X, k)
    assert _within(D.m, y, ref.rounded(y, e, dt))
