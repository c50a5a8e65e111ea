"""What the linear-layer entry points refuse, and what they accept without work.  Every call here
returns before anything is launched, so a handle that has never seen a device will do: the test
runs without a GPU."""
import ctypes as C

import pytest

from rtatblas_amd import native

BF16, F16, F32 = native.TYPE_BF16, native.TYPE_F16, native.TYPE_F32
N, T = native.OP_N, native.OP_T
OK, ALLOC, INVALID, UNSUPPORTED, NULL_HANDLE, ENUM = 0, 2, 3, 7, 9, 10
LONG = 2 ** 31 - 1000
P = 4096                       # a pointer that is never followed


class Bare(native.Handle):
    """The binding's methods on a zeroed block in place of a handle."""

    def __init__(self):
        self.lib = native.load()
        self.block = C.create_string_buffer(4096)
        self.h = C.addressof(self.block)

    def close(self):
        self.h = None


@pytest.fixture()
def bare():
    return Bare()


def ep(h, **kw):
    a = dict(type=BF16, ta=N, tb=N, m=4, n=3, k=2, alpha=1.0, A=P, lda=4, B=P, ldb=2, D=P, ldd=4, check=False)
    a.update(kw)
    return h.gemm_ep(**a)


@pytest.mark.parametrize("change,status", [
    (dict(type=F32), ENUM), (dict(type=1), ENUM), (dict(ta=113), ENUM), (dict(tb=0), ENUM), (dict(d_type=F16), ENUM),
    (dict(act=5), ENUM), (dict(act=-1), ENUM), (dict(m=-1), INVALID), (dict(n=-1), INVALID), (dict(k=-1), INVALID),
    (dict(lda=3), INVALID), (dict(ldb=1), INVALID), (dict(ldd=3), INVALID), (dict(A=None), INVALID), (dict(B=None), INVALID),
    (dict(D=None), INVALID), (dict(ta=T, lda=1), INVALID), (dict(tb=T, ldb=2), INVALID), (dict(beta=1.0), INVALID),
    (dict(beta=1.0, C=P, ldc=3), INVALID), (dict(aux=P, ldaux=3), INVALID), (dict(m=0, D=None), OK), (dict(n=0, A=None), OK),
    (dict(k=LONG, ldb=LONG), UNSUPPORTED), (dict(m=LONG, lda=LONG, ldd=LONG), UNSUPPORTED),
    (dict(n=2 ** 30 - 1023), UNSUPPORTED), (dict(n=2 ** 30 - 1024, D=None), INVALID)])
def test_gemm_ep(bare, change, status):
    assert ep(bare, **change) == status


def test_null_handle_and_null_scalars(bare):
    lib = bare.lib
    one = C.byref(C.c_float(1.0))
    args = [BF16, N, N, 4, 3, 2, one, P, 4, P, 2, None, one, None, 0, BF16, P, 4]
    assert lib.rtat_gemm_ep(None, *args) == NULL_HANDLE
    assert lib.rtat_gemm_ep(bare.h, *args[:6], None, *args[7:]) == INVALID
    assert lib.rtat_gemm_ep(bare.h, *args[:12], None, *args[13:]) == INVALID
    assert lib.rtat_gemm_ep_backward(None, *args[:11], 0, None, 0, P, 4, None) == NULL_HANDLE
    assert lib.rtat_gemm_ep_backward(bare.h, *args[:11], 0, None, 0, P, 4, None) == INVALID
    assert lib.rtat_gemm_dact(None, *args[:11], 0, None, 0, P, 4, None) == NULL_HANDLE
    assert lib.rtat_newton_schulz(None, F32, 4, 4, 1, P, 4, 0, 1, (C.c_float * 3)(), 0.0, P, 4, 0) == NULL_HANDLE


@pytest.mark.parametrize("change,status", [
    (dict(type=F32), ENUM), (dict(act=9), ENUM), (dict(ta=1), ENUM), (dict(dA=P, ldda=4, da_type=F16), ENUM),
    (dict(dB=P, lddb=2, db_type=7), ENUM), (dict(m=-1), INVALID), (dict(dA=P, ldda=3), INVALID), (dict(dB=P, lddb=1), INVALID),
    (dict(dD=None, dbias=P), INVALID), (dict(lddd=3), INVALID), (dict(act=2, aux=None, dZ=P, lddz=4), INVALID),
    (dict(act=2, aux=P, ldaux=3, dZ=P, lddz=4), INVALID), (dict(act=2, aux=P, ldaux=4, dZ=P, lddz=3), INVALID),
    (dict(act=2, aux=P, ldaux=4, dA=P, ldda=4), INVALID), (dict(dA=P, ldda=4, B=None), INVALID),
    (dict(dB=P, lddb=2, A=None), INVALID), (dict(dB=P, lddb=2, lda=3), INVALID), (dict(), OK), (dict(m=0, n=0, dD=None), OK), (dict(n=LONG), UNSUPPORTED)])
def test_backward(bare, change, status):
    a = dict(type=BF16, ta=N, tb=N, m=4, n=3, k=2, alpha=1.0, A=P, lda=4, B=P, ldb=2, dD=P, lddd=4, check=False)
    a.update(change)
    assert bare.gemm_ep_backward(**a) == status


@pytest.mark.parametrize("change,status", [
    (dict(type=F32), ENUM), (dict(act=5), ENUM), (dict(k=-1), INVALID), (dict(Z=None), INVALID), (dict(ldz=3), INVALID),
    (dict(D=None), INVALID), (dict(ldd=3), INVALID), (dict(A=None), INVALID), (dict(m=0), OK)])
def test_dact(bare, change, status):
    a = dict(type=F16, ta=N, tb=N, m=4, n=3, k=2, alpha=1.0, A=P, lda=4, B=P, ldb=2, act=4, Z=P, ldz=4, D=P, ldd=4, check=False)
    a.update(change)
    assert bare.gemm_dact(**a) == status


@pytest.mark.parametrize("change,status", [
    (dict(g_type=5), ENUM), (dict(m=-1), INVALID), (dict(batch=-1), INVALID), (dict(coeffs=[]), INVALID),
    (dict(coeffs=[(1, 1, 1)] * 33), INVALID), (dict(eps=-1.0), INVALID), (dict(eps=float("nan")), INVALID), (dict(G=None), INVALID),
    (dict(eps=float("inf")), INVALID), (dict(m=2 ** 30 - 1024, n=2 ** 30 - 1024, ldg=2 ** 30, ldo=2 ** 30), ALLOC),
    (dict(O=None), INVALID), (dict(ldg=3), INVALID), (dict(ldo=3), INVALID), (dict(batch=65536), INVALID), (dict(m=0, G=None), OK),
    (dict(n=LONG), UNSUPPORTED), (dict(n=0), OK), (dict(batch=0), OK)])
def test_newton_schulz(bare, change, status):
    a = dict(g_type=F32, m=4, n=3, G=P, ldg=4, O=P, ldo=4, coeffs=[(1.5, -0.5, 0.0)], check=False)
    a.update(change)
    assert bare.newton_schulz(**a) == status


def test_names_and_workspace_sizes():
    assert [native.activation_name(a) for a in range(native.ACT_COUNT)] == ["none", "relu", "gelu", "gelu_tanh", "silu"]
    assert native.activation_name(-1) is None and native.activation_name(native.ACT_COUNT) is None
    lib = native.load()
    assert lib.rtat_dbias_workspace_bytes(0, 5) == 0 and lib.rtat_dbias_workspace_bytes(100, 1) >= 400
    assert lib.rtat_newton_schulz_workspace_bytes(0, 4, 1) == 0
    one, six = (lib.rtat_newton_schulz_workspace_bytes(1000, 333, b) for b in (1, 6))
    # 1024 x 384 padded: two f16 and one f32 copy, and two 384 x 384 f16 matrices
    assert lib.rtat_newton_schulz_workspace_bytes(2 ** 30 - 1024, 2 ** 30 - 1024, 1) == 2 ** 64 - 1
    assert lib.rtat_newton_schulz_workspace_bytes(2 ** 30 - 1024, 2 ** 20, 65535) == 2 ** 64 - 1
    assert one >= 8 * 1024 * 384 + 4 * 384 * 384 and 5 * one < six <= 6 * one
