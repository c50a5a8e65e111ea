"""A few columns over a long k: past 20480 (32768 for more than 1024 rows) in slices, with a lent
workspace in one piece.  Every element against 64 bits, every epilogue, and the gradient's form."""
import pytest

import linear_ref as ref
from test_gpu_linear import Mat, N, T, _gen, _types, _within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lend", [False, True])
@pytest.mark.parametrize("which", ["bf16", "f16"])
@pytest.mark.parametrize("size", [(16, 1, 20480), (16, 1, 20488), (1, 16, 65536), (100, 3, 40008), (1024, 16, 24576),
                                  (1025, 2, 32776), (2049, 4, 33000)])
def test_long_k(size, which, lend):
    import torch
    from rtatblas_amd import native
    dt, ty = _types()[which]
    m, n, k = size
    gen = _gen(m + n + k)
    A, B = Mat(k, m, dt, 0, 0, gen, k ** -0.5), Mat(k, n, dt, 0, 0, gen)
    bias, C, D, Z = Mat(m, 1, dt, 0, 0, gen), Mat(m, n, dt, 3, 0, gen), Mat(m, n, dt, 5), Mat(m, n, dt, 1)
    h = native.Handle(torch.cuda.current_stream())
    try:
        if lend:
            ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
            h.set_workspace(ws, ws.numel())
        h.gemm_ep(ty, T, N, m, n, k, 0.75, A.ptr, A.ld, B.ptr, B.ld, D.ptr, D.ld, act=ref.SILU, bias=bias.ptr, aux=Z.ptr,
                  ldaux=Z.ld, beta=2.0, C=C.ptr, ldc=C.ld)
        (y, yb), (z, zb) = ref.forward(0.75, A.m.T, B.m, k, bias.m[:, 0], ref.SILU, 2.0, C.m, dt, dt)
        assert _within(D.m, y, yb) and _within(Z.m, z, zb) and D.padding_kept() and Z.padding_kept()
        db = torch.full((m,), float("nan"), device="cuda")
        h.gemm_dact(ty, T, N, m, n, k, 1.0, A.ptr, A.ld, B.ptr, B.ld, ref.GELU, C.ptr, C.ld, D.ptr, D.ld, dbias=db)
        g, e = ref.product(1.0, A.m.T, B.m, k)
        want, e = g * ref.slope(C.m.double(), ref.GELU), 1.13 * e + 2 * (ref.SLOPE_ERR + ref.U) * g.abs()
        assert _within(D.m, want, ref.rounded(want, e, dt)) and D.padding_kept()
        assert _within(db, want.sum(1), e.sum(1) + (n + 2) * ref.U * want.abs().sum(1))
    finally:
        torch.cuda.synchronize()
        h.close()
