"""MXFP4 operators on the GPU at the ends of fp32: the gate's exponential far below zero, blocks of the smallest numbers."""
import numpy as np
import pytest
import torch

from oracle import mxfp4 as o_mx
from test_mxfp4_gpu import N, check_quantised, dev, hip_quantize, product, ptr, stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["linear", "gemm"])
@pytest.mark.parametrize("m,n", [(3, 40), (16, 5000), (300, 1200), (1100, 3000)])
def test_gate_in_fp32(kind, m, n):
    """One column of K is not zero, so y = x w and u are exact and only the gate rounds.  silu(y) u = y / (1 + exp(-y)) * u: the exponential within 2 steps
    of 2^-23, then three roundings of half a step (2^-24) each: 7 half steps of the result; 8 are allowed."""
    k = 64
    fours, y = np.array([-4.0, -6.0, -3.0, -2.0, 4.0, 1.5]), np.array([1.0, 4.0, 6.0, 12.0, 3.0, 2.0])  # y = -72 .. 48
    w = np.zeros((n, k))
    w[:, 5] = fours[np.arange(n) % 6]
    w2 = np.zeros((n, k))
    w2[:, 5] = 1.0
    x = np.zeros((m, k))
    x[:, 5] = y[np.arange(m) % 6]
    wc, w2c, xc = o_mx.quantize(w), o_mx.quantize(w2), o_mx.quantize(x)
    for v, c in ((w, wc), (w2, w2c), (x, xc)):
        assert np.array_equal(o_mx.values(*c, k), v)
    act = torch.from_numpy(x).bfloat16().cuda() if kind == "linear" else (dev(xc[0]), dev(xc[1]))
    got = product(kind, act, (dev(wc[0]), dev(wc[1])), w2=(dev(w2c[0]), dev(w2c[1])), out_dtype=torch.float32, k=k)
    a, u = x @ w.T, x @ w2.T
    want = a / (1 + np.exp(-a)) * u
    worst = np.abs(got.cpu().double().numpy() - want) / np.abs(want) * 2 ** 24
    assert worst.max() <= 8, f"{worst.max():.1f} half steps at y = {a.flat[worst.argmax()]}"


def test_quantiser_of_the_smallest_fp32_numbers():
    """Blocks below 2^-125 have the exponent -127: their codes stand for multiples of 2^-128, and a number one bit off a tie is rounded by that bit."""
    g = torch.Generator().manual_seed(6)
    bits = torch.randint(0, 1 << 23, (64, 96), generator=g, dtype=torch.int32)  # subnormal numbers
    bits[::2] >>= torch.randint(0, 20, (32, 96), generator=g, dtype=torch.int32)
    tie = torch.ldexp(torch.tensor([1, 3, 5, 7, 10, 14, 20], dtype=torch.float64), torch.tensor(-129.0)).float()  # between two codes each
    row = torch.cat([tie, torch.nextafter(tie, tie * 2), torch.nextafter(tie, tie * 0), torch.full((11,), 2.0 ** -149)]).view(1, 32).repeat(1, 3)
    w = torch.cat([bits.view(torch.float32), row, (bits >> 1).view(torch.float32)])
    w = torch.cat([w, -w]).cuda()
    check_quantised(w, *hip_quantize(w))


def test_an_output_in_a_gap_of_x():
    """A whole output between two rows of strided x, and the rows themselves stay."""
    m, n, k, ld = 3, 40, 96, 1000
    g = torch.Generator().manual_seed(2)
    room = torch.randn(m, ld, generator=g).bfloat16().cuda()
    keep = room.clone()
    w = tuple(map(dev, o_mx.quantize(torch.randn(n, k, generator=g).double().numpy())))
    want = product("linear", room[:, :k], w, k=k)
    for row, at in ((0, k), (1, 500), (2, ld - m * n)):
        room.copy_(keep)
        out = room.view(-1)[row * ld + at:row * ld + at + m * n]
        N.check(N.lib().mv_op_linear_mxfp4(stream(), m, n, k, ptr(room), ld, ptr(w[0]), ptr(w[1]), None, None, None, None, None, 0, ptr(out)))
        torch.cuda.synchronize()
        assert torch.equal(out.view(m, n), want) and torch.equal(room[:, :k], keep[:, :k])
