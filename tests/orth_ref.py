"""Float64 statements of the orthogonalised update, and the same with the kernels' roundings (test infrastructure)."""
import torch

QUINTIC = (3.4445, -4.7750, 2.0315)


def exact(g, steps=5, eps=1e-7):
    """X <- a X + (b A + c A A) X from G / (|G|_F + eps), in float64."""
    a, b, c = QUINTIC
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = x / (x.square().sum().sqrt() + eps)
    for _ in range(steps):
        A = x @ x.t()
        x = a * x + (b * A + c * A @ A) @ x
    return x.t() if tall else x


def _half(x, scale):
    return (x * scale).float().half().double() / scale


def rounded(g, steps=5, eps=1e-7):
    """The same with every rounding to fp16 that the kernels make (X = hi + lo, products of hi, off-diagonals of A and B),
    sums in float64: what the number formats alone cost."""
    a, b, c = QUINTIC
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = x / (x.square().sum().sqrt() + eps)
    hi = _half(x, 1024.0)
    lo = _half(x - hi, 1024.0)
    for _ in range(steps):
        A = hi @ hi.t()
        d = A.diagonal().clone()
        o = _half(A - torch.diag(d), 8192.0)
        sq = o @ o
        B = b * o + c * (sq + (d[:, None] + d[None, :]) * o)
        e = b * d + c * (sq.diagonal() + d * d)
        B = _half(B - torch.diag(B.diagonal()), 4096.0)
        x = a * (hi + lo) + e[:, None] * hi + B @ hi
        hi = _half(x, 1024.0)
        lo = _half(x - hi, 1024.0)
    return x.t() if tall else x


def bounds(g, steps=5, eps=1e-7):
    """(exact result, bound on the elements' error, bound on the error's 2-norm) before the rounding of the output.  The
    kernels' errors are another draw of the same roundings (their fp32 sums, 2^-24, add nothing that shows beside 2^-11):
    1.5 times the norm and 3 times the largest error of the emulation, and 1e-6 for matrices so small that it rounds exactly."""
    ref = exact(g, steps, eps)
    d = rounded(g, steps, eps) - ref
    return ref, 3 * float(d.abs().max()) + 1e-6, 1.5 * float(d.norm()) + 1e-6 * ref.numel() ** 0.5
