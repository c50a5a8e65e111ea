"""The linear-layer operators as programs use them: recorded into HIP graphs and replayed on new
inputs, on streams of their own, with a lent workspace, on a handle inside a capture that owns no
scratch, a few columns at a time, far into long operands, and twice with the same bits."""
import pytest

import linear_ref as ref
from test_gpu_linear import Mat, N, T, _gen, _op, _operands, _types, _within

pytestmark = pytest.mark.gpu
QUINTIC = (3.4445, -4.7750, 2.0315)


@pytest.mark.parametrize("size", [(100, 5, 1000), (4096, 3, 4104), (33, 16, 8), (17, 1, 24), (2048, 13, 8192), (1, 2, 256),
                                  (500, 16, 40), (65, 4, 2056)])
@pytest.mark.parametrize("which", ["bf16", "f16"])
def test_few_columns(handle, size, which):
    """Products of up to sixteen columns with every epilogue, and the gradient's form."""
    import torch
    dt, ty = _types()[which]
    m, n, k = size
    gen = _gen(m + n + k)
    A, B = _operands(gen, dt, T, N, m, n, k, 0, 0)
    A, B = (Mat(*x.m.shape, dt, -x.m.shape[0] % 8, 0, gen) for x in (A, B))
    bias, C, D, Z = Mat(m, 1, dt, 0, 0, gen), Mat(m, n, dt, 3, 0, gen), Mat(m, n, dt, 5), Mat(m, n, dt, 1)
    for act in range(5):
        handle.gemm_ep(ty, T, N, m, n, k, 0.75, A.ptr, A.ld, B.ptr, B.ld, D.ptr, D.ld, act=act, bias=bias.ptr, aux=Z.ptr,
                       ldaux=Z.ld, beta=2.0, C=C.ptr, ldc=C.ld)
        (y, yb), (z, zb) = ref.forward(0.75, A.m.T, B.m, k, bias.m[:, 0], act, 2.0, C.m, dt, dt)
        assert _within(D.m, y, yb) and _within(Z.m, z, zb) and D.padding_kept() and Z.padding_kept()
        db = torch.full((m,), float("nan"), device="cuda")
        handle.gemm_dact(ty, T, N, m, n, k, 1.0, A.ptr, A.ld, B.ptr, B.ld, act, C.ptr, C.ld, D.ptr, D.ld, dbias=db)
        g, e = ref.product(1.0, A.m.T, B.m, k)
        want, e = g * ref.slope(C.m.double(), act), 1.13 * e + 2 * (ref.SLOPE_ERR + ref.U) * g.abs()
        assert _within(D.m, want, ref.rounded(want, e, dt)) and D.padding_kept()
        assert _within(db, want.sum(1), e.sum(1) + (n + 2) * ref.U * want.abs().sum(1))
    f = Mat(m, n, torch.float32, 0, 0, gen)
    f0 = f.m.clone()
    handle.gemm_ep(ty, T, N, m, n, k, 1.0, A.ptr, A.ld, B.ptr, B.ld, f.ptr, f.ld, d_type=0, beta=1.0, C=f.ptr, ldc=f.ld)
    (y, yb), _ = ref.forward(1.0, A.m.T, B.m, k, None, 0, 1.0, f0, dt, torch.float32)
    assert _within(f.m, y, yb)


def _step(h, ty, bufs, sizes):
    """A layer's forward and backward pass and its update orthogonalised, on torch tensors."""
    t, d, f = sizes
    X, W, b, Z, Y, dY, dZ, dW, dX, db, O = bufs
    h.gemm_ep(ty, T, N, f, t, d, 1.0, W, d, X, d, Y, f, act=ref.GELU, bias=b, aux=Z, ldaux=f)
    h.gemm_ep_backward(ty, T, N, f, t, d, 1.0, W, d, X, d, dY, f, act=ref.GELU, aux=Z, ldaux=f, dZ=dZ, lddz=f, dA=dW, ldda=d,
                       da_type=0, dB=dX, lddb=d, dbias=db)
    h.newton_schulz(0, d, f, dW, d, O, d, [QUINTIC] * 3)


def _bufs(gen, dt, sizes):
    import torch
    t, d, f = sizes

    def rnd(*s):
        return torch.randn(*s, generator=gen, device="cuda").to(dt)

    def new(*s, dtype=dt):
        return torch.zeros(*s, dtype=dtype, device="cuda")

    return [rnd(t, d), rnd(f, d), rnd(f), new(t, f), new(t, f), rnd(t, f), new(t, f), new(f, d, dtype=torch.float32), new(t, d),
            new(f, dtype=torch.float32), new(f, d, dtype=torch.bfloat16)]


@pytest.mark.parametrize("sizes", [(64, 128, 96), (333, 201, 150), (1024, 512, 1500)])
@pytest.mark.parametrize("lend", [False, True])
def test_graph_replays_match_eager(sizes, lend):
    """Captured once, replayed on new inputs with eager work between the replays."""
    import torch
    from rtatblas_amd import native
    dt, ty = _types()["bf16"]
    gen = _gen(sum(sizes))
    t, d, f = sizes
    bufs = _bufs(gen, dt, sizes)
    h, cap = native.Handle(), torch.cuda.Stream()
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    try:
        h.set_stream(cap)
        if lend:
            h.set_workspace(ws, ws.numel())
        torch.cuda.synchronize()
        _step(h, ty, bufs, sizes)                 # first launches, and the handle's scratch
        cap.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=cap):
            _step(h, ty, bufs, sizes)
        for rep in range(3):
            for i in (0, 1, 5):
                bufs[i].copy_(torch.randn(bufs[i].shape, generator=gen, device="cuda").to(dt))
            torch.cuda.synchronize()
            _step(h, ty, bufs, sizes)
            cap.synchronize()
            want = [x.clone() for x in bufs]
            for i in (3, 4, 6, 7, 8, 9, 10):
                bufs[i].zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(bufs, want)), rep
    finally:
        torch.cuda.synchronize()
        h.close()


def test_capture_on_a_handle_without_scratch():
    """Nothing is allocated inside a capture: what needs scratch says so and leaves the capture
    usable, an unaligned product runs without it."""
    import torch
    from rtatblas_amd import native
    dt, ty = _types()["bf16"]
    m, n, k = 1501, 1203, 1001
    gen = _gen(2)
    A, B = _operands(gen, dt, T, N, m, n, k, 0, 1)
    D, Z = Mat(m, n, dt, 1), Mat(m, n, dt, 0, 0, gen)
    db = torch.zeros(m, device="cuda")
    G, O = torch.randn(300, 200, generator=gen, device="cuda"), torch.empty(300, 200, dtype=torch.bfloat16, device="cuda")
    warm = native.Handle(torch.cuda.current_stream())     # the kernels' code on the device
    warm.gemm_ep(ty, T, N, m, n, k, 1.0, A.ptr, A.ld, B.ptr, B.ld, D.ptr, D.ld, act=ref.SILU)
    warm.set_workspace(torch.empty(256, dtype=torch.uint8, device="cuda"), 256)
    warm.gemm_ep(ty, T, N, m, n, k, 1.0, A.ptr, A.ld, B.ptr, B.ld, D.ptr, D.ld, act=ref.SILU)
    st = warm.gemm_dact(ty, T, N, m, n, k, 1.0, A.ptr, A.ld, B.ptr, B.ld, 1, Z.ptr, Z.ld, D.ptr, D.ld, dbias=db, check=False)
    assert native.STATUS_NAMES[st] == "ALLOC_FAILED"      # a lent buffer that is too small
    torch.cuda.synchronize()
    h, cap = native.Handle(), torch.cuda.Stream()
    try:
        h.set_stream(cap)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=cap):
            a = h.newton_schulz(0, 200, 300, G, 200, O, 200, [QUINTIC], check=False)
            b = h.gemm_dact(ty, T, N, m, n, k, 1.0, A.ptr, A.ld, B.ptr, B.ld, 1, Z.ptr, Z.ld, D.ptr, D.ld, dbias=db, check=False)
            h.gemm_ep(ty, T, N, m, n, k, 1.0, A.ptr, A.ld, B.ptr, B.ld, D.ptr, D.ld, act=ref.SILU)
        assert native.STATUS_NAMES[a] == native.STATUS_NAMES[b] == "ALLOC_FAILED"
        (y, yb), _ = ref.forward(1.0, A.m.T, B.m, k, None, ref.SILU, 0.0, None, dt, dt)
        for _ in range(3):
            D.m.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert _within(D.m, y, yb)
    finally:
        torch.cuda.synchronize()
        h.close()
        warm.close()


def test_two_handles_on_two_streams():
    """Independent work interleaved on two streams gives what each gives alone."""
    import torch
    from rtatblas_amd import native
    dt, ty = _types()["f16"]
    sizes = (700, 333, 512)
    jobs = []
    for seed in (1, 2):
        bufs = _bufs(_gen(seed), dt, sizes)
        h = native.Handle(torch.cuda.current_stream())
        _step(h, ty, bufs, sizes)
        torch.cuda.synchronize()
        jobs.append((h, bufs, [x.clone() for x in bufs]))
    streams = [torch.cuda.Stream() for _ in jobs]
    try:
        for (h, bufs, _), s in zip(jobs, streams):
            h.set_stream(s)
            for i in (3, 4, 6, 7, 8, 9, 10):
                bufs[i].zero_()
        torch.cuda.synchronize()
        for _ in range(4):
            for h, bufs, _ in jobs:
                _step(h, ty, bufs, sizes)
        torch.cuda.synchronize()
        for _, bufs, want in jobs:
            assert all(torch.equal(a, b) for a, b in zip(bufs, want))
    finally:
        torch.cuda.synchronize()
        for h, _, _ in jobs:
            h.close()


@pytest.mark.parametrize("size", [(512, 200, 8192), (1001, 300, 3000), (2048, 2048, 512)])
def test_lent_workspace_and_repeated_bits(size):
    """With a lent buffer products are not cut along k and unaligned ones use the buffer if it is
    large enough; every form is within the bounds, and a repeated call gives the same bits."""
    import torch
    from rtatblas_amd import native
    dt, ty = _types()["bf16"]
    m, n, k = size
    gen = _gen(m)
    h = native.Handle(torch.cuda.current_stream())
    try:
        for shift in (0, 1):
            A, B = _operands(gen, dt, T, T, m, n, k, shift, shift)
            (y, yb), _ = ref.forward(1.0, A.m.T, B.m.T, k, None, ref.RELU, 0.0, None, dt, dt)
            for lent in (0, 1 << 10, 64 << 20):
                ws = torch.empty(lent + 3, dtype=torch.uint8, device="cuda")[3:] if lent else None   # any address
                h.set_workspace(ws, lent)
                got = []
                for _ in range(2):
                    D = Mat(m, n, dt)
                    h.gemm_ep(ty, T, T, m, n, k, 1.0, A.ptr, A.ld, B.ptr, B.ld, D.ptr, D.ld, act=ref.RELU)
                    assert _within(D.m, y, yb)
                    got.append(D.m.clone())
                assert torch.equal(*got)
                torch.cuda.synchronize()
                h.set_workspace(None, 0)
    finally:
        torch.cuda.synchronize()
        h.close()


def test_offsets_past_32_bits(handle):
    """The last columns of a result and an operand whose element offsets pass 2^31 and 2^32."""
    import torch
    dt, ty = _types()["bf16"]
    m, n, k, ld = 64, 40, 64, 1 << 27
    gen = _gen(4)
    B = torch.empty(ld * (n - 1) + k, dtype=dt, device="cuda")
    D = torch.empty(ld * (n - 1) + m, dtype=dt, device="cuda")
    A = Mat(m, k, dt, 0, 0, gen)
    Bv, Dv = torch.as_strided(B, (k, n), (1, ld)), torch.as_strided(D, (m, n), (1, ld))
    Bv.copy_(torch.randn(k, n, generator=gen, device="cuda").to(dt))
    handle.gemm_ep(ty, N, N, m, n, k, 1.0, A.ptr, A.ld, B, ld, D, ld)
    y, e = ref.product(1.0, A.m, Bv, k)
    assert _within(Dv, y, ref.rounded(y, e, dt))
    # ... and as the operand that is contiguous along its columns
    Dt = Mat(n, m, dt)
    handle.gemm_ep(ty, T, T, n, m, k, 1.0, B, ld, A.ptr, A.ld, Dt.ptr, Dt.ld)
    assert _within(Dt.m, y.T, ref.rounded(y.T, e.T, dt))


def test_update_batch_of_padded_rows(handle):
    """A batch of one-workgroup updates and a batch of larger ones, strides longer than the
    matrices: what lies between them stays as it was."""
    import torch
    for n, m in ((70, 100), (150, 260)):
        gen = _gen(m)
        b, gap = 3, 1000
        G = torch.full((b, n * m + gap), 7.0, device="cuda")
        G[:, :n * m] = torch.randn(b, n * m, generator=gen, device="cuda")
        O = torch.full((b, n * m + gap), 7.0, dtype=torch.bfloat16, device="cuda")
        handle.newton_schulz(0, m, n, G, m, O, m, [QUINTIC] * 5, batch=b, strideg=n * m + gap, strideo=n * m + gap)
        assert bool((O[:, n * m:] == 7).all())
        for g, o in zip(G, O):
            want = ref.newton_schulz(g[:n * m].reshape(n, m), [QUINTIC] * 5)
            got = o[:n * m].reshape(n, m).double()
            assert ((got - want).norm() / want.norm()).item() <= 2.0 ** -9 + 3e-3


def test_more_rows_than_a_launch_of_few_columns_holds(handle):
    """A single column of more than 2^27 rows: two gigabytes of A."""
    import torch
    dt, ty = _types()["bf16"]
    m, k = (1 << 27) + 17, 8
    gen = _gen(6)
    A = torch.randn(m, k, generator=gen, device="cuda", dtype=dt)
    b = torch.randn(k, generator=gen, device="cuda", dtype=dt)
    D = torch.full((m + 8,), float("nan"), device="cuda", dtype=dt)
    handle.gemm_ep(ty, T, N, m, 1, k, 1.0, A, k, b, k, D, m)
    assert torch.isnan(D[m:]).all()
    for first in (0, 1 << 26, m - 5000):
        y, e = ref.product(1.0, A[first:first + 5000], b[:, None], k)
        assert _within(D[first:first + 5000, None], y, ref.rounded(y, e, dt))


@pytest.mark.parametrize("side", [72, 1600, 2048, 2304])
@pytest.mark.parametrize("ops", [(T, N), (N, N), (N, T), (T, T)])
def test_any_number_of_panels(handle, side, ops):
    """From part of one panel of k to more than any ring of panels holds, whole and not, at sides
    that run on different tiles, with NaN behind every column of the operands."""
    import torch
    dt, ty = _types()["bf16"]
    gen = _gen(side)
    D = Mat(side, side, dt, 8)
    for k in (8, 56, 64, 72, 128, 136, 192, 200, 256, 264, 320, 328, 384, 440, 576):
        shapes = [(side, k) if op == N else (k, side) for op in (ops[0], ops[1])]
        shapes[1] = (k, side) if ops[1] == N else (side, k)
        A, B = (Mat(r, c, dt, 8, 0, gen) for r, c in shapes)
        handle.gemm_ep(ty, *ops, side, side, k, 1.0, A.ptr, A.ld, B.ptr, B.ld, D.ptr, D.ld)
        a, b = A.m if ops[0] == N else A.m.T, B.m if ops[1] == N else B.m.T
        y, e = ref.product(1.0, a, b, k)
        assert _within(D.m, y, ref.rounded(y, e, dt)) and D.padding_kept(), k
