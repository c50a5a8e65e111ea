"""rtat_gemm_ep, rtat_gemm_ep_backward and rtat_gemm_dact on the GPU against 64 bits, element by
element, within bounds that count the roundings (linear_ref.py): every activation, both types,
all op combinations, odd sizes and strides, one column to many tiles, empty dimensions, in-place
residuals, padding left alone, and the layer's forward and backward pass run together."""
import pytest

import linear_ref as ref

pytestmark = pytest.mark.gpu
N, T = 111, 112


def _types():
    import torch
    from rtatblas_amd import native
    return {"bf16": (torch.bfloat16, native.TYPE_BF16), "f16": (torch.float16, native.TYPE_F16),
            "f32": (torch.float32, native.TYPE_F32)}


class Mat:
    """A column-major r x c matrix with leading dimension r + pad, its start shifted by `shift`
    elements, NaN in the padding; .m is the (r, c) view."""

    def __init__(self, r, c, dtype, pad=0, shift=0, gen=None, scale=1.0, fill=None):
        import torch
        self.ld = max(r + pad, 1)
        self.buf = torch.full((shift + self.ld * c + 1,), float("nan"), dtype=dtype, device="cuda")
        self.m = torch.as_strided(self.buf, (r, c), (1, self.ld), shift)
        self.ptr = self.buf.data_ptr() + shift * self.buf.element_size()
        if gen is not None:
            self.m.copy_((torch.randn(r, c, generator=gen, device="cuda") * scale).to(dtype))
        elif fill is not None:
            self.m.fill_(fill)
        self.before = self.buf.clone()

    def padding_kept(self):
        """Everything outside the matrix is still what it was, bit for bit."""
        import torch
        a, b = self.buf.clone(), self.before.clone()
        for x in (a, b):
            torch.as_strided(x, self.m.shape, (1, self.ld), self.m.storage_offset()).zero_()
        es = {2: torch.int16, 4: torch.int32}[a.element_size()]
        return torch.equal(a.view(es), b.view(es))


def _gen(seed):
    import torch
    return torch.Generator(device="cuda").manual_seed(seed)


def _op(x, trans):
    return x.T if trans == T else x


def _within(got, want, bound):
    import torch
    d = (got.double() - want).abs()
    ok = bool((d <= bound).all())
    if not ok:
        bad = (d - bound).argmax()
        print("worst: got %g want %g bound %g" % (got.double().flatten()[bad], want.flatten()[bad], bound.flatten()[bad]))
    return ok


def _operands(gen, dt, ta, tb, m, n, k, pad, shift):
    A = Mat(*((k, m) if ta == T else (m, k)), dt, pad, shift, gen, max(k, 1) ** -0.5)
    B = Mat(*((n, k) if tb == T else (k, n)), dt, pad, shift, gen)
    return A, B


SIZES = [(1, 1, 1), (5, 1, 3), (200, 1, 64), (129, 7, 65), (64, 64, 64), (128, 16, 512), (131, 70, 129),
         (256, 128, 1000), (300, 520, 77), (512, 300, 8), (1000, 17, 2048), (640, 700, 320)]


@pytest.mark.parametrize("ta", [N, T])
@pytest.mark.parametrize("tb", [N, T])
@pytest.mark.parametrize("size", SIZES)
def test_forward_ops_and_sizes(handle, ta, tb, size):
    """bias + GELU + aux + residual for every op combination; aligned and odd storage."""
    m, n, k = size
    for which, pad, shift in (("bf16", 0, 0), ("f16", 0, 0), ("bf16", 3, 1), ("f16", 8, 8)):
        dt, ty = _types()[which]
        gen = _gen(m * 7 + n * 3 + k)
        A, B = _operands(gen, dt, ta, tb, m, n, k, pad, shift)
        bias = Mat(m, 1, dt, 0, shift, gen)
        C = Mat(m, n, dt, pad, shift, gen)
        D, Z = Mat(m, n, dt, pad, shift), Mat(m, n, dt, pad, shift)
        handle.gemm_ep(ty, ta, tb, m, n, k, 1.25, A.ptr, A.ld, B.ptr, B.ld, D.ptr, D.ld, act=ref.GELU, bias=bias.ptr,
                       aux=Z.ptr, ldaux=Z.ld, beta=-0.5, C=C.ptr, ldc=C.ld)
        (y, yb), (z, zb) = ref.forward(1.25, _op(A.m, ta), _op(B.m, tb), k, bias.m[:, 0], ref.GELU, -0.5, C.m, dt, dt)
        assert _within(D.m, y, yb) and _within(Z.m, z, zb), (which, pad)
        assert D.padding_kept() and Z.padding_kept()


@pytest.mark.parametrize("ta", [N, T])
@pytest.mark.parametrize("tb", [N, T])
@pytest.mark.parametrize("size", [(3001, 3003, 129), (3000, 3080, 200), (2817, 4096, 64), (4096, 2816, 72), (3333, 2900, 1),
                                  (2560, 3584, 640)])
def test_forward_many_tiles(handle, ta, tb, size):
    """Enough tiles for the largest tile shape, 16-byte aligned columns, ragged edges and k."""
    m, n, k = size
    for which in ("bf16", "f16"):
        dt, ty = _types()[which]
        gen = _gen(m + n)
        A = Mat(*((k, m) if ta == T else (m, k)), dt, 0, 0, gen, k ** -0.5)
        B = Mat(*((n, k) if tb == T else (k, n)), dt, 0, 0, gen)
        A, B = (Mat(x.m.shape[0], x.m.shape[1], dt, -x.m.shape[0] % 8, 0, gen) for x in (A, B))
        C, D, Z = Mat(m, n, dt, 1, 0, gen), Mat(m, n, dt, 5), Mat(m, n, dt, -m % 8)
        handle.gemm_ep(ty, ta, tb, m, n, k, 0.5, A.ptr, A.ld, B.ptr, B.ld, D.ptr, D.ld, act=ref.SILU, aux=Z.ptr, ldaux=Z.ld,
                       beta=1.0, C=C.ptr, ldc=C.ld)
        (y, yb), (z, zb) = ref.forward(0.5, _op(A.m, ta), _op(B.m, tb), k, None, ref.SILU, 1.0, C.m, dt, dt)
        assert _within(D.m, y, yb) and _within(Z.m, z, zb)
        assert D.padding_kept() and Z.padding_kept()
        # the gradient's form of the same product, sums of many columns
        db = torch_empty(m)
        handle.gemm_dact(ty, ta, tb, m, n, k, 0.5, A.ptr, A.ld, B.ptr, B.ld, ref.GELU, C.ptr, C.ld, D.ptr, D.ld, dbias=db)
        g, e = ref.product(0.5, _op(A.m, ta), _op(B.m, tb), k)
        want, e = g * ref.slope(C.m.double(), ref.GELU), 1.13 * e + 2 * (ref.SLOPE_ERR + ref.U) * g.abs()
        assert _within(D.m, want, ref.rounded(want, e, dt)) and D.padding_kept()
        assert _within(db, want.sum(1), e.sum(1) + (n + 2) * ref.U * want.abs().sum(1))


def torch_empty(m):
    import torch
    return torch.full((m,), float("nan"), device="cuda")


@pytest.mark.parametrize("act", range(5))
@pytest.mark.parametrize("which", ["bf16", "f16"])
def test_forward_activations(handle, act, which):
    """Arguments from far below to far above 0, straight through a product with the unit matrix."""
    import torch
    dt, ty = _types()[which]
    m, n = 96, 40
    z = torch.cat([torch.linspace(-30, 30, m * n // 2), torch.linspace(-3, 3, m * n // 2)]).reshape(m, n).to(dt).cuda()
    A, B, D = Mat(m, m, dt, fill=0.0), Mat(m, n, dt), Mat(m, n, torch.float32)
    A.m.copy_(torch.eye(m))
    B.m.copy_(z)
    handle.gemm_ep(ty, N, N, m, n, m, 1.0, A.ptr, A.ld, B.ptr, B.ld, D.ptr, D.ld, d_type=0, act=act)
    want = ref.act(z.double(), act)
    assert _within(D.m, want, ref.rounded(want, ref.ACT_ERR * (1 + z.double().abs()), torch.float32))


def test_forward_infinite_and_nan_arguments(handle):
    import torch
    dt, ty = _types()["bf16"]
    inf = float("inf")
    z = torch.tensor([inf, 1e30, -1e30, float("nan"), 0.0, -0.0, 3e38, -3e38], device="cuda").to(dt)
    m = z.numel()
    A, B, D = Mat(m, 1, dt), Mat(1, 1, dt, fill=1.0), Mat(m, 1, torch.float32)
    A.m.copy_(z[:, None])
    for act in range(5):
        handle.gemm_ep(ty, N, N, m, 1, 1, 1.0, A.ptr, A.ld, B.ptr, B.ld, D.ptr, D.ld, d_type=0, act=act)
        got = D.m[:, 0].cpu()
        assert got[0] == inf and torch.isnan(got[3]) and got[4] == 0
        assert got[1] == z[1].float().item() and (act == 0 or got[2] == 0)
        # the gradient stays finite where the argument is
        G, S = Mat(m, 1, dt, fill=1.0), Mat(m, 1, dt)
        handle.gemm_ep_backward(ty, N, N, m, 1, 1, 1.0, A.ptr, A.ld, B.ptr, B.ld, G.ptr, G.ld, act=act, aux=A.ptr, ldaux=A.ld,
                                dZ=S.ptr, lddz=S.ld, dbias=torch.empty(m, device="cuda"))
        if act:
            s = S.m[:, 0].float().cpu()
            want = [1, 1, 0, None, 0.5 if act != ref.RELU else 0, 0.5 if act != ref.RELU else 0, 1, 0]
            for i, w in enumerate(want):
                assert torch.isnan(s[i]) if w is None and act != ref.RELU else (w is None or s[i] == w), (act, i, s)


def test_forward_f32_result_and_in_place_residual(handle):
    """d_type F32 with C == D (a weight gradient accumulated in 32 bits), and D == C in 16 bits."""
    import torch
    for which, ddt in (("bf16", "f32"), ("f16", "f32"), ("bf16", "bf16")):
        for pad in (0, 1):
            dt, ty = _types()[which]
            dd, dty = _types()[ddt]
            m, n, k = 260, 129, 300
            gen = _gen(5)
            A, B = _operands(gen, dt, N, T, m, n, k, pad, 0)
            D = Mat(m, n, dd, pad, 0, gen)
            C0 = D.m.clone()
            handle.gemm_ep(ty, N, T, m, n, k, 0.75, A.ptr, A.ld, B.ptr, B.ld, D.ptr, D.ld, d_type=dty, beta=1.0, C=D.ptr, ldc=D.ld)
            (y, yb), _ = ref.forward(0.75, A.m, B.m.T, k, None, 0, 1.0, C0, dt, dd)
            assert _within(D.m, y, yb), (which, ddt, pad)
            assert D.padding_kept()


def test_forward_empty_dimensions_and_unread_operands(handle):
    import torch
    dt, ty = _types()["bf16"]
    m, n = 70, 33
    gen = _gen(8)
    bias, C, D = Mat(m, 1, dt, 0, 0, gen), Mat(m, n, dt, 0, 0, gen), Mat(m, n, dt)
    bad = Mat(m, 64, dt)                      # NaN throughout: never read
    want = ref.act(bias.m.double(), ref.SILU) + 2.0 * C.m.double()
    for k, alpha, A in ((0, 1.0, None), (64, 0.0, bad.ptr)):
        D.m.fill_(float("nan"))
        handle.gemm_ep(ty, N, N, m, n, k, alpha, A, m, A, 64, D.ptr, D.ld, act=ref.SILU, bias=bias.ptr, beta=2.0, C=C.ptr, ldc=C.ld)
        assert _within(D.m, want, ref.rounded(want, ref.ACT_ERR * (1 + bias.m.double().abs()) + 4 * ref.U * want.abs(), dt))
    handle.gemm_ep(ty, N, N, m, n, 0, 1.0, None, m, None, 1, D.ptr, D.ld)   # C NULL with beta 0
    assert bool((D.m == 0).all())
    before = D.buf.clone()
    assert handle.gemm_ep(ty, N, N, 0, n, 4, 1.0, None, 1, None, 4, None, 1, check=False) == 0
    assert handle.gemm_ep(ty, N, N, m, 0, 4, 1.0, None, m, None, 4, None, m, check=False) == 0
    torch.cuda.synchronize()
    assert torch.equal(D.buf.view(torch.int16), before.view(torch.int16))


@pytest.mark.parametrize("ta", [N, T])
@pytest.mark.parametrize("tb", [N, T])
@pytest.mark.parametrize("which,pad,grads,act", [("bf16", 0, "bf16", ref.GELU_TANH), ("f16", 3, "f32", ref.NONE),
                                                 ("bf16", 1, "f32", ref.SILU), ("f16", 8, "f16", ref.RELU)])
def test_backward(handle, ta, tb, which, pad, grads, act):
    """dZ and dbias against the formula; dA and dB against the products of dZ as stored."""
    import torch
    dt, ty = _types()[which]
    gd, gty = _types()[grads]
    for m, n, k in ((1, 1, 1), (130, 1, 70), (65, 200, 129), (300, 260, 136)):
        gen = _gen(m + n + k)
        A, B = _operands(gen, dt, ta, tb, m, n, k, pad, 0)
        dD, Z, dZ = Mat(m, n, dt, pad, 0, gen), Mat(m, n, dt, pad, 0, gen, 2.0), Mat(m, n, dt, pad)
        dA = Mat(*A.m.shape, gd, pad, 0, gen)
        dB = Mat(*B.m.shape, gd, pad)
        dA0 = dA.m.clone()
        db = torch.full((m,), float("nan"), device="cuda")
        handle.gemm_ep_backward(ty, ta, tb, m, n, k, 0.5, A.ptr, A.ld, B.ptr, B.ld, dD.ptr, dD.ld, act=act,
                                aux=Z.ptr, ldaux=Z.ld, dZ=dZ.ptr, lddz=dZ.ld, dA=dA.ptr, ldda=dA.ld, da_type=gty, da_beta=1.0,
                                dB=dB.ptr, lddb=dB.ld, db_type=gty, dbias=db)
        dz = dD.m.double() * ref.slope(Z.m.double(), act)
        err = (ref.SLOPE_ERR + ref.U) * dD.m.double().abs() * 2
        stored = dD.m if act == ref.NONE else dZ.m
        if act != ref.NONE:
            assert _within(dZ.m, dz, ref.rounded(dz, err, dt)) and dZ.padding_kept()
        assert _within(db, dz.sum(1), err.sum(1) + (n + 2) * ref.U * dz.abs().sum(1))
        opA, opB = _op(A.m, ta), _op(B.m, tb)
        want, e = ref.product(0.5, stored, opB.T, n)
        want, e = (want.T, e.T) if ta == T else (want, e)
        want, e = want + dA0.double(), e + 2 * ref.U * (want.abs() + dA0.double().abs())
        assert _within(dA.m, want, ref.rounded(want, e, gd)) and dA.padding_kept()
        want, e = ref.product(0.5, opA.T, stored, m)
        want, e = (want.T, e.T) if tb == T else (want, e)
        assert _within(dB.m, want, ref.rounded(want, e, gd)) and dB.padding_kept()


def test_backward_in_place_and_parts(handle):
    """dZ over dD; single outputs; empty dimensions write zeros."""
    import torch
    dt, ty = _types()["bf16"]
    m, n, k = 200, 90, 64
    gen = _gen(3)
    A, B = _operands(gen, dt, T, N, m, n, k, 0, 0)
    dD, Z = Mat(m, n, dt, 0, 0, gen), Mat(m, n, dt, 0, 0, gen)
    dz = dD.m.double() * ref.slope(Z.m.double(), ref.SILU)
    err = 2 * (ref.SLOPE_ERR + ref.U) * dD.m.double().abs()
    db = torch.empty(m, device="cuda")
    handle.gemm_ep_backward(ty, T, N, m, n, k, 1.0, None, 1, None, 1, dD.ptr, dD.ld, act=ref.SILU, aux=Z.ptr, ldaux=Z.ld, dbias=db)
    assert _within(db, dz.sum(1), err.sum(1) + (n + 2) * ref.U * dz.abs().sum(1))
    handle.gemm_ep_backward(ty, T, N, m, n, k, 1.0, None, 1, None, 1, dD.ptr, dD.ld, act=ref.SILU, aux=Z.ptr, ldaux=Z.ld,
                            dZ=dD.ptr, lddz=dD.ld)
    assert _within(dD.m, dz, ref.rounded(dz, err, dt))
    # no columns: the weight's gradient and the sums are sums over nothing
    dA = Mat(k, m, dt, fill=7.0)
    db.fill_(7.0)
    handle.gemm_ep_backward(ty, T, N, m, 0, k, 1.0, None, 1, None, 1, None, m, act=ref.SILU, dA=dA.ptr, ldda=dA.ld, dbias=db)
    assert bool((dA.m == 0).all()) and bool((db == 0).all())


@pytest.mark.parametrize("act", range(5))
@pytest.mark.parametrize("which,pad,size", [("bf16", 0, (512, 300, 128)), ("f16", 1, (131, 70, 65)), ("bf16", 8, (1, 9, 3)),
                                            ("f16", 0, (264, 1, 40)), ("bf16", 2, (1500, 260, 96)),
                                            ("bf16", 0, (300, 20, 1024)), ("f16", 3, (77, 130, 2100))])
def test_dact(handle, act, which, pad, size):
    import torch
    dt, ty = _types()[which]
    m, n, k = size
    for ta, tb in ((N, N), (T, N)):
        gen = _gen(m + act)
        A, B = _operands(gen, dt, ta, tb, m, n, k, pad, 0)
        Z, D = Mat(m, n, dt, pad, 0, gen, 2.0), Mat(m, n, dt, pad)
        db = torch.full((m,), float("nan"), device="cuda")
        handle.gemm_dact(ty, ta, tb, m, n, k, 1.5, A.ptr, A.ld, B.ptr, B.ld, act, Z.ptr, Z.ld, D.ptr, D.ld, dbias=db)
        g, e = ref.product(1.5, _op(A.m, ta), _op(B.m, tb), k)
        s = ref.slope(Z.m.double(), act)
        want = g * s
        e = 1.13 * e + 2 * (ref.SLOPE_ERR + ref.U) * g.abs()
        assert _within(D.m, want, ref.rounded(want, e, dt)) and D.padding_kept()
        assert _within(db, want.sum(1), e.sum(1) + (n + 2) * ref.U * want.abs().sum(1))
        again = torch.empty_like(db)
        handle.gemm_dact(ty, ta, tb, m, n, k, 1.5, A.ptr, A.ld, B.ptr, B.ld, act, Z.ptr, Z.ld, Z.ptr, Z.ld, dbias=again)
        assert torch.equal(again, db) and torch.equal(Z.m, D.m)    # in place, and the same bits


def test_gradient_against_differences_of_the_forward_call(handle):
    """L = sum(G * D) of the forward call itself (f32 result), moved along a direction V of A by
    +-h in steps that A represents exactly.  A central difference is off by at most
    h^2 / 6 max|act'''| sum |G| |dz|^3 (|act'''| <= 2 for the smooth ones), and by the f32 errors
    of the two values over 2 h."""
    import torch
    dt, ty = _types()["f16"]
    m, n, k, h = 64, 48, 32, 2.0 ** -5
    gen = _gen(11)
    for act in (ref.GELU, ref.GELU_TANH, ref.SILU):
        A, B = Mat(m, k, dt), Mat(k, n, dt)
        A.m.copy_(torch.randint(-8, 9, (m, k), generator=gen, device="cuda") / 32)
        B.m.copy_(torch.randint(-8, 9, (k, n), generator=gen, device="cuda") / 16)
        V = torch.randint(-1, 2, (m, k), generator=gen, device="cuda").to(dt)
        G, Z = Mat(m, n, dt, 0, 0, gen), Mat(m, n, dt)
        base, vals, errs = A.m.clone(), [], 0.0
        for s in (1, -1):
            A.m.copy_(base + s * h * V)
            D = Mat(m, n, torch.float32)
            handle.gemm_ep(ty, N, N, m, n, k, 1.0, A.ptr, A.ld, B.ptr, B.ld, D.ptr, D.ld, d_type=0, act=act)
            (y, yb), _ = ref.forward(1.0, A.m, B.m, k, None, act, 0.0, None, dt, torch.float32)
            vals.append((G.m.double() * D.m.double()).sum().item())
            errs += (G.m.double().abs() * yb).sum().item()
        A.m.copy_(base)
        D = Mat(m, n, torch.float32)
        handle.gemm_ep(ty, N, N, m, n, k, 1.0, A.ptr, A.ld, B.ptr, B.ld, D.ptr, D.ld, d_type=0, act=act, aux=Z.ptr, ldaux=Z.ld)
        dA, dZ = Mat(m, k, torch.float32), Mat(m, n, dt)
        handle.gemm_ep_backward(ty, N, N, m, n, k, 1.0, A.ptr, A.ld, B.ptr, B.ld, G.ptr, G.ld, act=act, aux=Z.ptr, ldaux=Z.ld,
                                dZ=dZ.ptr, lddz=dZ.ld, dA=dA.ptr, ldda=dA.ld, da_type=0)
        along = (dA.m.double() * V.double()).sum().item()
        dz = (V.double() @ B.m.double()).abs()
        g = G.m.double().abs()
        # dZ is rounded to 16 bits, and so is the Z it is taken at (second derivative <= 1.2)
        rounding = (g * 1.13 * dz).sum().item() * ref.STEP[dt] + (g * 1.2 * Z.m.double().abs() * dz).sum().item() * ref.STEP[dt]
        bound = (g * dz ** 3).sum().item() * 2 * h * h / 6 + errs / (2 * h) + rounding + 1e-5 * g.sum().item()
        assert abs((vals[0] - vals[1]) / (2 * h) - along) <= bound, act


def test_layer_trains(handle):
    """The operators as a training step uses them: two layers forward, the backward pass through
    both, the two weights' updates orthogonalised.  Every gradient against autograd in 64 bits on
    the same inputs; 16-bit tensors between the calls cost at most a few half steps."""
    import torch
    dt, ty = _types()["f16"]
    from rtatblas_amd import native
    t, d, f = 300, 128, 520
    gen = _gen(21)

    def rnd(*s, scale=1.0):
        return (torch.randn(*s, generator=gen, device="cuda") * scale).to(dt)

    X, W1, W2 = rnd(t, d), rnd(f, d, scale=d ** -0.5), rnd(d, f, scale=f ** -0.5)
    b1, b2, dY = rnd(f, scale=0.1), rnd(d, scale=0.1), rnd(t, d)
    Z1, H, Y, dZ1 = (torch.empty(t, c, dtype=dt, device="cuda") for c in (f, f, d, f))
    handle.gemm_ep(ty, T, N, f, t, d, 1.0, W1, d, X, d, H, f, act=ref.GELU, bias=b1, aux=Z1, ldaux=f)
    handle.gemm_ep(ty, T, N, d, t, f, 1.0, W2, f, H, f, Y, d, bias=b2, beta=1.0, C=X, ldc=d)
    dW2, dW1 = (torch.empty(*w.shape, device="cuda") for w in (W2, W1))
    db2, db1 = torch.empty(d, device="cuda"), torch.empty(f, device="cuda")
    dX = torch.empty(t, d, dtype=dt, device="cuda")
    handle.gemm_ep_backward(ty, T, N, d, t, f, 1.0, W2, f, H, f, dY, d, dA=dW2, ldda=f, da_type=0, dbias=db2)
    handle.gemm_dact(ty, N, N, f, t, d, 1.0, W2, f, dY, d, ref.GELU, Z1, f, dZ1, f, dbias=db1)
    handle.gemm_ep_backward(ty, T, N, f, t, d, 1.0, W1, d, X, d, dZ1, f, dA=dW1, ldda=d, da_type=0, dB=dX, lddb=d)
    leaves = [x.double().requires_grad_(True) for x in (X, W1, W2, b1, b2)]
    x, w1, w2, c1, c2 = leaves
    y = ref.act(x @ w1.T + c1, ref.GELU) @ w2.T + c2 + x
    want = torch.autograd.grad(y, leaves, dY.double())
    step = ref.STEP[dt]

    def rel(a, b):
        return ((a.double() - b).norm() / b.norm()).item()

    # each 16-bit tensor in a chain adds a relative error of at most half a step in 2-norm; the
    # longest chain here holds four (Z, dZ, the result; H for dW2)
    assert rel(Y, y.detach()) <= 4 * step
    assert rel(dX.double() + dY.double(), want[0]) <= 4 * step
    for got, w in ((dW1, want[1]), (dW2, want[2]), (db1, want[3]), (db2, want[4])):
        assert rel(got, w) <= 4 * step
    coeffs = [(3.4445, -4.7750, 2.0315)] * 5
    for g in (dW1, dW2):
        o = torch.empty(*g.shape, dtype=torch.bfloat16, device="cuda")
        handle.newton_schulz(native.TYPE_F32, g.shape[1], g.shape[0], g, g.shape[1], o, g.shape[1], coeffs)
        assert rel(o, ref.newton_schulz(g, coeffs)) <= 2.0 ** -9 + 3e-3
