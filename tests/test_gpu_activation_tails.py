"""Activations and slopes far below and above zero, relative to their own size, in every kernel that
applies them: tiles, slices joined, a few columns, and the elementwise pass of the backward call.

Bounds, in half steps U of f32.  GELU: the tail of the normal distribution is off by 6.2 (1 + z^2)
with exact elementary functions (emulated over 400001 arguments); the exponential and the
reciprocal of the hardware are good to one step, two half steps, each, and the product with z
rounds once: 12 (1 + z^2).  GELU_TANH and SILU: the argument y of the exponential is a product
of at most four roundings, so the exponential is off by 4 y half steps, and 8 more cover the functions
and products.  A slope adds two terms with such errors, one factor more in each: 16 in place of 12
and 8, relative to the sum of the terms' sizes."""
import math

import pytest

import linear_ref as ref
from test_gpu_linear import Mat, N, T, _types, _within

pytestmark = pytest.mark.gpu
U = ref.U
SMOOTH = (ref.GELU, ref.GELU_TANH, ref.SILU)


def _arguments(dt):
    """Values of the type from -far to far, evenly spread, each sign's neighbourhood of zero too."""
    import torch
    far = 12.5
    z = torch.cat([torch.linspace(-far, far, 4096), torch.logspace(-3, 0, 1024), -torch.logspace(-3, 0, 1024)])
    return z.to(dt).cuda()


def _y(z, a):
    return (math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3)).abs() if a == ref.GELU_TANH else z.abs()


def _value(z, a):
    """act(z) in 64 bits by expressions that keep the tail, and the error allowed."""
    import torch
    if a == ref.GELU:
        y = z * torch.special.erfc(-z / math.sqrt(2)) / 2
        return y, 12 * U * (1 + z * z) * y.abs()
    y = ref.act(z, a)
    return y, U * (8 + 4 * _y(z, a)) * y.abs()


def _slope(z, a):
    import torch
    if a == ref.GELU:
        p, d = torch.special.erfc(-z / math.sqrt(2)) / 2, torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        return p + z * d, 16 * U * (1 + z * z) * (p + z.abs() * d)
    y = _y(z, a)
    p = torch.sigmoid(torch.where(z < 0, -y, y))
    rest = torch.sigmoid(torch.where(z < 0, y, -y))
    dy = math.sqrt(8 / math.pi) * (1 + 3 * 0.044715 * z * z) if a == ref.GELU_TANH else torch.ones_like(z)
    # 1 - p is formed from p, so it has p's error in full: a half step of 1 + exp, two of the reciprocal,
    # one for second order.
    return p + z * dy * p * rest, U * (16 + 4 * y) * (p + z.abs() * dy * p * rest) + z.abs() * dy * p * 4 * U


def _seen(z, a):
    """Arguments whose result, and the factors on the way to it, are normal numbers of f32."""
    return (z >= 0) | (_y(z, a) < 80 if a != ref.GELU else z > -12.4)



def _unit_product(z, dt, way):
    """Operands whose product is z laid out m x n, exactly: a unit matrix and z, k from m on zeros."""
    import torch
    n = 4 if way == "few" else 32
    m = z.numel() // n
    k = 16384 if way == "slices" else m
    ta = N if way == "tiles" else T
    A = Mat(*((k, m) if ta == T else (m, k)), dt, fill=0.0)
    (A.m.T if ta == T else A.m)[:, :m].copy_(torch.eye(m))
    B = Mat(k, n, dt, fill=0.0)
    B.m[:m].copy_(z.reshape(m, n))
    return m, n, k, ta, A, B


@pytest.mark.parametrize("way", ["tiles", "few", "slices"])
@pytest.mark.parametrize("a", SMOOTH)
@pytest.mark.parametrize("which", ["bf16", "f16"])
def test_values(handle, which, a, way):
    import torch
    dt, ty = _types()[which]
    z = _arguments(dt)
    m, n, k, ta, A, B = _unit_product(z, dt, way)
    want, err = _value(z.double().reshape(m, n), a)
    seen = _seen(z.double().reshape(m, n), a)
    for d_which in ("f32", which):
        ddt, dty = _types()[d_which]
        D = Mat(m, n, ddt)
        handle.gemm_ep(ty, ta, N, m, n, k, 1.0, A.ptr, A.ld, B.ptr, B.ld, D.ptr, D.ld, d_type=dty, act=a)
        assert _within(D.m[seen], want[seen], ref.rounded(want, err, ddt)[seen]), d_which


@pytest.mark.parametrize("way", ["pass", "tiles", "few", "slices"])
@pytest.mark.parametrize("a", SMOOTH)
@pytest.mark.parametrize("which", ["bf16", "f16"])
def test_slopes(handle, which, a, way):
    """A gradient of ones: the slopes themselves, rounded and, as sums of one column, in f32."""
    import torch
    dt, ty = _types()[which]
    z = _arguments(dt)
    n = 1
    m = z.numel() // 8
    for part in z.reshape(8, m):
        Z, D = Mat(m, n, dt), Mat(m, n, dt)
        Z.m.copy_(part[:, None])
        db = torch.full((m,), float("nan"), device="cuda")
        if way == "pass":
            G = Mat(m, n, dt, fill=1.0)
            handle.gemm_ep_backward(ty, N, N, m, n, 1, 1.0, None, m, None, 1, G.ptr, G.ld, act=a, aux=Z.ptr, ldaux=Z.ld,
                                    dZ=D.ptr, lddz=D.ld, dbias=db)
        else:
            k = {"tiles": 64, "few": 64, "slices": 16384}[way]
            # Few columns need k-contiguous operands; tiles and slices take the others.
            ta = T if way == "few" else N
            A = Mat(*((k, m) if ta == T else (m, k)), dt, fill=0.0)
            (A.m.T if ta == T else A.m)[:, :1].fill_(1.0)
            B = Mat(k, n, dt, fill=0.0)
            B.m[0] = 1.0
            handle.gemm_dact(ty, ta, N, m, n, k, 1.0, A.ptr, A.ld, B.ptr, B.ld, a, Z.ptr, Z.ld, D.ptr, D.ld, dbias=db)
        z64 = part.double()
        want, err = _slope(z64, a)
        seen = _seen(z64, a)
        assert _within(db[seen], want[seen], ref.rounded(want, err, torch.float32)[seen])
        assert _within(D.m[:, 0][seen], want[seen], ref.rounded(want, err, dt)[seen])
