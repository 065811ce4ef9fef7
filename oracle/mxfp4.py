"""MXFP4 (microscaled 4-bit floating point) in 64 bits on the CPU: the definition behind mv_op_quantize_mxfp4, mv_op_linear_mxfp4 and mv_op_gemm_mxfp4.

No reference counterpart: the format is the published OCP microscaling one (blocks of 32, element type E2M1, scale type E8M0)."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def blocks(k: int) -> int:
    return (k + 31) // 32


def quantize(w: np.ndarray):
    """w float64 [N][K] -> codes uint8 [N][16 nb], scales uint8 [N][nb]."""
    n, k = w.shape
    nb = blocks(k)
    x = np.zeros((n, nb * 32))
    x[:, :k] = w
    x = x.reshape(n, nb, 32)
    bad = ~np.isfinite(x).all(-1)
    mag = np.where(bad[..., None], 0.0, np.abs(x))
    top = mag.max(-1)
    e = np.where(top > 0, np.frexp(np.where(top > 0, top, 1.0))[1] - 3, -127).clip(-127, 127)
    y = np.minimum(mag / np.ldexp(1.0, e)[..., None], 6.0)
    # nearest grid point; of two equally near ones the one whose code is even
    d = np.abs(y[..., None] - GRID)
    near = d == d.min(-1, keepdims=True)
    even = near & (np.arange(8) % 2 == 0)
    q = np.where(even.any(-1), even.argmax(-1), near.argmax(-1)).astype(np.uint8)
    q = q + 8 * np.signbit(x).astype(np.uint8)
    q = np.where(bad[..., None], 0, q).astype(np.uint8).reshape(n, nb * 32)
    scales = np.where(bad, 255, e + 127).astype(np.uint8)
    return q[:, 0::2] | (q[:, 1::2] << 4), scales


def values(codes: np.ndarray, scales: np.ndarray, k: int) -> np.ndarray:
    """codes, scales -> float64 [N][K]."""
    q = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1)
    v = np.where(q >= 8, -1.0, 1.0) * GRID[q & 7]
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int32) - 127))
    return (v * np.repeat(s, 32, axis=1))[:, :k]


def product(x, w, w2=None, bias=None, bias2=None, residual=None):
    """x [M][K], w / w2 [N][K] float64 -> y float64 [M][N] and a bound on what one rounding of the sums can move, per unit of (additions x half step):
    the sum of magnitudes that enter an output, carried through the gate (|silu'| < 1.1, and silu itself for the other factor)."""
    def lin(m, b):
        y, s = x @ m.T, np.abs(x) @ np.abs(m).T
        return (y, s) if b is None else (y + b, s + np.abs(b))

    y, s = lin(w, bias)
    if w2 is not None:
        u, su = lin(w2, bias2)
        with np.errstate(over="ignore"):
            a = y / (1.0 + np.exp(-y))
        # exp in fp32 costs a relative error that grows with its argument: |y| steps
        s = 1.1 * s * (np.abs(u) + su * 2.0 ** -14) + np.abs(a) * su + np.abs(a * u) * (np.abs(y) + 8) / 64
        y = a * u
    if residual is not None:
        y, s = y + residual, s + np.abs(residual)
    return y, s
