"""Plain 64-bit forms of the linear-layer operators (rtat_gemm_ep, its gradients,
rtat_gemm_dact, rtat_newton_schulz) and the error bounds their tests are written in.  Works on
torch tensors of any device; matrices are (rows, cols) as the formulas have them, whatever
their storage."""
import math

import torch

U = 2.0 ** -24                      # half a step of f32
STEP = {torch.bfloat16: torch.finfo(torch.bfloat16).eps / 2,
        torch.float16: torch.finfo(torch.float16).eps / 2, torch.float32: U}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
NONE, RELU, GELU, GELU_TANH, SILU = range(5)
# f32 evaluation of an activation, relative to 1 + |z|: exp2 of a rounded argument, a reciprocal
# and a few products (8 half steps), and 1.5e-7 |z| of the erfc approximation.
ACT_ERR = 8 * U + 1.5e-7
# ... and of a slope, which adds products of factors up to z (1 + 0.134 z^2) p (1 - p) < 1:
# 32 half steps.
SLOPE_ERR = 32 * U + 1.5e-7
LIPSCHITZ = 1.13                    # largest slope of any of them


def act(z, a):
    if a == RELU:
        return torch.where(z < 0, torch.zeros_like(z), z)
    if a == GELU:
        return z * torch.special.ndtr(z)
    if a == GELU_TANH:
        return z * torch.sigmoid(math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3))
    if a == SILU:
        return z * torch.sigmoid(z)
    return z


def slope(z, a):
    if a == RELU:
        return (z > 0).to(z.dtype)
    if a == GELU:
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if a == GELU_TANH:
        c = math.sqrt(8 / math.pi)
        p = torch.sigmoid(c * (z + 0.044715 * z ** 3))
        return p + z * c * (1 + 3 * 0.044715 * z * z) * p * (1 - p)
    if a == SILU:
        p = torch.sigmoid(z)
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


def rounded(ref, err, dtype):
    """Bound on |rounded f32 value - ref| when the f32 value is within err of ref."""
    return err + STEP[dtype] * (ref.abs() + err) + TINY[dtype]


def product(alpha, A, B, k):
    """alpha A B in f64 and the bound of its f32 evaluation: exact products of 16-bit factors, k
    additions in any order, two half steps each (the matrix cores may cut instead of round), the
    factor alpha."""
    z = alpha * (A.double() @ B.double())
    s = abs(alpha) * (A.double().abs() @ B.double().abs())
    return z, (2 * k + 2) * U * s


def forward(alpha, A, B, k, bias, a, beta, C, aux_dtype, d_dtype):
    """D and aux with their bounds."""
    z, err = product(alpha, A, B, k)
    if bias is not None:
        z = z + bias.double()[:, None]
        err = err + U * z.abs()
    aux = (z, rounded(z, err, aux_dtype))
    y = act(z, a)
    if a != NONE:
        err = LIPSCHITZ * err + ACT_ERR * (1 + z.abs())
    if beta != 0:
        y = y + beta * C.double()
        err = err + 2 * U * (y.abs() + abs(beta) * C.double().abs())
    return (y, rounded(y, err, d_dtype)), aux


def newton_schulz(G, coeffs, eps=1e-7):
    X = G.double()
    X = X / (torch.linalg.matrix_norm(X) + eps)
    for a, b, c in coeffs:
        if X.shape[0] <= X.shape[1]:
            M = X @ X.T
            X = a * X + (b * M + c * (M @ M)) @ X
        else:
            M = X.T @ X
            X = a * X + X @ (b * M + c * (M @ M))
    return X
