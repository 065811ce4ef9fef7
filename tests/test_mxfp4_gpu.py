"""MXFP4 quantiser and products (mv_op_quantize_mxfp4, mv_op_linear_mxfp4, mv_op_gemm_mxfp4) on the GPU against oracle/mxfp4.py (64 bits).

The quantiser and its values are exact.  A product's tolerance counts roundings: a term passes the additions inside one matrix instruction (at most
128), one per instruction along K (at most K / 32) and one per partial sum that is joined (at most 64), each off by at most 2^-23 of the magnitudes
summed; the output's own rounding is half a step (2^-8 bf16, 2^-24 fp32)."""
import ctypes as C

import numpy as np
import pytest
import torch

from conftest import load_pkg
from oracle import mxfp4 as o_mx

pytestmark = pytest.mark.gpu

N = load_pkg("_native")
CODE = {torch.bfloat16: 0, torch.float32: 1}


def ptr(t):
    return C.c_void_p(t.data_ptr()) if t is not None else None


def stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def bits64(t):
    return t.detach().cpu().double().numpy()


def hip_quantize(w, k=None, deq=True):
    n, ld = w.shape[0], w.stride(0)
    k = w.shape[1] if k is None else k
    nb = o_mx.blocks(k)
    codes = torch.full((n + 1, 16 * nb), 0x5A, dtype=torch.uint8, device="cuda")  # one row more than is quantised: it stays as it is
    scales = torch.full((n + 1, nb), 0x5A, dtype=torch.uint8, device="cuda")
    d = torch.full((n + 1, k), 7.0, dtype=torch.bfloat16, device="cuda") if deq else None
    N.check(N.lib().mv_op_quantize_mxfp4(stream(), n, k, CODE[w.dtype], ptr(w), ld, ptr(codes), ptr(scales), ptr(d)))
    torch.cuda.synchronize()
    assert bool((codes[n] == 0x5A).all()) and bool((scales[n] == 0x5A).all()) and (d is None or bool((d[n] == 7).all()))
    return codes[:n], scales[:n], None if d is None else d[:n]


def check_quantised(w, codes, scales, deq):
    c, s = o_mx.quantize(bits64(w))
    assert np.array_equal(scales.cpu().numpy(), s)
    assert np.array_equal(codes.cpu().numpy(), c)
    if deq is not None:
        assert np.array_equal(bits64(deq), o_mx.values(c, s, w.shape[1]), equal_nan=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,k", [(1, 1), (1, 31), (3, 32), (5, 33), (2, 64), (7, 100), (33, 257), (64, 2048), (300, 1111)])
@pytest.mark.parametrize("pad", [0, 1, 8])
def test_quantiser_is_exact(n, k, dtype, pad):
    g = torch.Generator().manual_seed(n * 1000 + k)
    w = (torch.randn(n, k + pad, generator=g) * torch.exp(4 * torch.randn(n, 1, generator=g))).to(dtype)
    w[0, 0] = 0
    w[n - 1, max(0, k - 32):] = 0  # a block of zeros
    w = w.cuda()[:, :k]
    check_quantised(w, *hip_quantize(w))
    check_quantised(w, *hip_quantize(w, deq=False))


def test_quantiser_over_all_bf16_numbers_and_ties():
    """Every bf16 bit pattern against itself and a large neighbour; and every tie of the grid at every block exponent."""
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    w = every.view(-1, 32).cuda()  # blocks of one exponent; some hold infinities and NaN
    check_quantised(w, *hip_quantize(w))
    fine = torch.where(torch.isfinite(every.float()), every, torch.zeros_like(every)).view(-1, 1).expand(-1, 32).clone()
    fine[:, 1:] = 0
    fine = fine.cuda()
    check_quantised(fine, *hip_quantize(fine))
    tie = torch.tensor([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7]).repeat(2)
    tie[16:] *= -1
    t32 = torch.ldexp(tie.double().view(1, 32), torch.arange(-126, 125, dtype=torch.float64).view(-1, 1)).float()
    t32 = torch.cat([t32, torch.nextafter(t32, torch.zeros_like(t32)), torch.nextafter(t32, t32 * 2)]).cuda()
    check_quantised(t32, *hip_quantize(t32))


def test_quantiser_marks_blocks_that_are_not_finite():
    w = torch.randn(4, 96)
    w[0, 5], w[1, 40], w[2, 95], w[3, 0] = float("inf"), float("-inf"), float("nan"), 3.0e38
    for dt in (torch.bfloat16, torch.float32):
        d = w.to(dt).cuda()
        codes, scales, deq = hip_quantize(d)
        check_quantised(d, codes, scales, deq)
        assert (scales.cpu() == 255).nonzero().tolist() == [[0, 0], [1, 1], [2, 2]]


def test_quantiser_in_place():
    w = (torch.randn(40, 256) * 0.1).bfloat16().cuda()
    c, s = o_mx.quantize(bits64(w))
    codes, scales = torch.zeros(40, 128, dtype=torch.uint8, device="cuda"), torch.zeros(40, 8, dtype=torch.uint8, device="cuda")
    N.check(N.lib().mv_op_quantize_mxfp4(stream(), 40, 256, 0, ptr(w), 256, ptr(codes), ptr(scales), ptr(w)))
    torch.cuda.synchronize()
    assert np.array_equal(bits64(w), o_mx.values(c, s, 256))


def make(g, n, k, spread=1.0):
    codes, scales = o_mx.quantize((torch.randn(n, k, generator=g) * torch.exp(spread * torch.randn(n, 1, generator=g))).double().numpy())
    return codes, scales


def make_fast(g, n, k):
    """Random codes and scales, zeros past K."""
    nb = o_mx.blocks(k)
    q = torch.randint(0, 256, (n, 16 * nb), generator=g).numpy().astype(np.uint8)
    cols = np.arange(32 * nb).reshape(-1, 2)
    q &= ((cols[:, 0] < k) * 15 + (cols[:, 1] < k) * 240).astype(np.uint8)
    return q, torch.randint(118, 128, (n, nb), generator=g).numpy().astype(np.uint8)


def dev(a):
    return torch.from_numpy(a).cuda()


def product(kind, x, w, w2=None, bias=None, bias2=None, residual=None, out_dtype=torch.bfloat16, k=None, in_place=False):
    """x: bf16 tensor, or (codes, scales); returns the output and asserts that the row behind it is left alone."""
    m = (x if kind == "linear" else x[0]).shape[0]
    n = w[0].shape[0]
    out = torch.full((m + 1, n), 7.0, dtype=out_dtype, device="cuda")
    if in_place:
        out[:m] = residual
        residual = out
    act = (ptr(x), x.stride(0)) if kind == "linear" else (ptr(x[0]), ptr(x[1]))
    w2 = w2 or (None, None)
    fn = N.lib().mv_op_linear_mxfp4 if kind == "linear" else N.lib().mv_op_gemm_mxfp4
    N.check(fn(stream(), m, n, k, *act, ptr(w[0]), ptr(w[1]), ptr(w2[0]), ptr(w2[1]), ptr(bias), ptr(bias2), ptr(residual), CODE[out_dtype], ptr(out)))
    torch.cuda.synchronize()
    assert bool((out[m] == 7).all())
    return out[:m]


def within(got, want, size, k, dtype):
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    tol = (128 + k / 32 + 64) * 2.0 ** -23 * size + half * np.abs(want) + 1e-37
    got = bits64(got)
    assert got.shape == want.shape
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[0]}: {got[bad][0]} against {want[bad][0]}, {np.abs(got - want)[bad][0] / tol[bad][0]:.2f} tolerances"


SHAPES = [(1, 1, 1), (1, 16, 32), (2, 2562, 2048), (3, 17, 33), (5, 40, 96), (16, 64, 128), (17, 100, 127), (33, 48, 640), (48, 320, 4096), (64, 129, 1000),
          (65, 260, 512), (100, 1000, 736), (128, 128, 256), (130, 257, 511), (200, 512, 1024), (257, 300, 2080), (512, 520, 288), (300, 1030, 31)]


def case(kind, m, n, k, gated, bias, residual, dtype, pad=0, make=make):
    g = torch.Generator().manual_seed(m * 7 + n * 3 + k)
    if kind == "linear":
        x = torch.randn(m, k + pad, generator=g).bfloat16().cuda()[:, :k]
        x64 = bits64(x)
    else:
        xc = make(g, m, k)
        x, x64 = (dev(xc[0]), dev(xc[1])), o_mx.values(*xc, k)
    w, w2 = make(g, n, k), make(g, n, k) if gated else None
    b = torch.randn(n, generator=g).bfloat16() if bias else None
    b2 = torch.randn(n, generator=g).bfloat16() if bias and gated else None
    res = torch.randn(m, n, generator=g).to(dtype) if residual else None
    f = lambda t: None if t is None else t.double().numpy()  # noqa: E731
    want, size = o_mx.product(x64, o_mx.values(*w, k), None if w2 is None else o_mx.values(*w2, k), f(b), f(b2), f(res))
    up = lambda t: None if t is None else t.cuda()  # noqa: E731
    args = dict(x=x, w=(dev(w[0]), dev(w[1])), w2=None if w2 is None else (dev(w2[0]), dev(w2[1])), bias=up(b), bias2=up(b2), residual=up(res), out_dtype=dtype, k=k)
    return args, want, size


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("kind", ["linear", "gemm"])
def test_product(kind, m, n, k):
    for gated, bias, residual, dtype in ((False, False, False, torch.bfloat16), (False, True, True, torch.float32), (True, False, False, torch.bfloat16),
                                         (True, True, True, torch.bfloat16)):
        args, want, size = case(kind, m, n, k, gated, bias, residual, dtype)
        within(product(kind, **args), want, size, k, dtype)


# Products large enough for the row kernels of several tiles and for every tiled kernel: whole and short stages, rows of scales that are and are not
# aligned (ceil(K / 32) a multiple of 4 or not), rows that begin on a cache line (a multiple of 8) and that do not, ragged last tiles, an odd number of
# stages.
LARGE = [(25, 6000, 1500), (30, 9000, 600), (700, 900, 1088), (600, 1500, 1100), (1100, 1300, 640), (1537, 4100, 320), (2049, 4100, 200), (1300, 6200, 1000),
         (1100, 8300, 225), (2300, 3900, 289), (513, 2500, 2049), (3000, 3100, 1024),
         (90, 1900, 1130), (88, 3700, 1116), (112, 10078, 517), (88, 4010, 2100),
         (18, 8049, 1280), (36, 8191, 1024), (74, 6529, 1280), (67, 6273, 955),
         (17, 4201, 512), (17, 8151, 1078), (546, 5411, 65), (193, 8603, 256), (18, 41090, 512), (40, 9001, 640), (250, 3000, 2000), (100, 9003, 1110), (227, 8366, 250)]


@pytest.mark.parametrize("m,n,k", LARGE)
@pytest.mark.parametrize("kind", ["linear", "gemm"])
def test_large_product(kind, m, n, k):
    for gated, bias, residual, dtype in ((False, False, False, torch.bfloat16), (True, True, True, torch.float32)):
        args, want, size = case(kind, m, n // 2 if gated else n, k, gated, bias, residual, dtype, make=make_fast)
        within(product(kind, **args), want, size, k, dtype)


@pytest.mark.parametrize("pad", [1, 2, 8])
@pytest.mark.parametrize("m,n,k", [(700, 900, 1088), (1100, 1300, 640), (1300, 6200, 1000), (2300, 3900, 289)])
def test_large_linear_of_strided_rows(m, n, k, pad):
    args, want, size = case("linear", m, n, k, False, True, False, torch.bfloat16, pad, make=make_fast)
    within(product("linear", **args), want, size, k, torch.bfloat16)


@pytest.mark.parametrize("kind", ["linear", "gemm"])
def test_large_products_repeat_and_leave_nan_in_its_row(kind):
    """Tiled kernels: the same bits on every run; a NaN block reaches its own weight row, and with 4-bit x its own x row, and nothing else."""
    for m, n, k in ((1100, 1300, 640), (2100, 4000, 416)):
        args, _, _ = case(kind, m, n, k, False, False, False, torch.float32, make=make_fast)
        first = product(kind, **args)
        for _ in range(3):
            assert torch.equal(product(kind, **args), first)
        args["w"][1][n - 3, 5] = 255
        if kind == "gemm":
            args["x"][1][m - 2, 1] = 255
        got = product(kind, **args)
        nan = torch.isnan(got)
        want = torch.zeros_like(nan)
        want[:, n - 3] = True
        if kind == "gemm":
            want[m - 2] = True
        assert torch.equal(nan, want) and torch.equal(got[~nan], first[~nan])


@pytest.mark.parametrize("pad", [1, 3, 8])
@pytest.mark.parametrize("m,n,k", [(2, 100, 640), (20, 64, 333), (150, 200, 1024), (300, 300, 500)])
def test_linear_of_strided_rows(m, n, k, pad):
    args, want, size = case("linear", m, n, k, False, True, False, torch.float32, pad)
    within(product("linear", **args), want, size, k, torch.float32)


@pytest.mark.parametrize("kind", ["linear", "gemm"])
@pytest.mark.parametrize("m", [2, 40, 300])
def test_residual_in_place(kind, m):
    args, want, size = case(kind, m, 272, 512, False, False, True, torch.bfloat16)
    within(product(kind, in_place=True, **args), want, size, 512, torch.bfloat16)


@pytest.mark.parametrize("kind", ["linear", "gemm"])
@pytest.mark.parametrize("m", [2, 40, 300])
def test_extreme_and_nan_scales(kind, m):
    """The smallest block exponents (values below the smallest normal bf16) still count, the largest do not overflow on the way, and a NaN block
    reaches the outputs of its own weight row or its own x row alone."""
    n, k = 80, 256
    g = torch.Generator().manual_seed(5)
    args, _, _ = case(kind, m, n, k, False, False, False, torch.float32)
    wc, ws = make(g, n, k, 0.0)
    ws[0], ws[1], ws[2] = 0, 1, 250
    if kind == "linear":
        x = torch.randn(m, k, generator=g)
        x64 = (x * 2.0 ** 100).bfloat16().double().numpy()
        args["x"] = torch.from_numpy(x64).bfloat16().cuda()
        ws[2] = 140
    else:
        xc, xs = make(g, m, k, 0.0)
        xs[:, 1] = 227
        ws[2] = 20
        args["x"], x64 = (dev(xc), dev(xs)), o_mx.values(xc, xs, k)
    args["w"] = (dev(wc), dev(ws))
    want, size = o_mx.product(x64, o_mx.values(wc, ws, k))
    within(product(kind, **args), want, size, k, torch.float32)
    ws[7, 3] = 255
    args["w"] = (dev(wc), dev(ws))
    got = product(kind, **args)
    assert bool(torch.isnan(got[:, 7]).all()) and not bool(torch.isnan(torch.cat([got[:, :7], got[:, 8:]], 1)).any())
    if kind == "gemm":
        ws[7, 3], xs[m - 1, 0] = 127, 255
        args["w"], args["x"] = (dev(wc), dev(ws)), (dev(xc), dev(xs))
        got = product(kind, **args)
        assert bool(torch.isnan(got[m - 1]).all()) and not bool(torch.isnan(got[: m - 1]).any())


@pytest.mark.parametrize("kind", ["linear", "gemm"])
def test_empty_calls_touch_nothing(kind):
    args, _, _ = case(kind, 4, 16, 64, False, False, False, torch.float32)
    out = torch.full((4, 16), 7.0, device="cuda")
    act = (ptr(args["x"]), 64) if kind == "linear" else (ptr(args["x"][0]), ptr(args["x"][1]))
    fn = N.lib().mv_op_linear_mxfp4 if kind == "linear" else N.lib().mv_op_gemm_mxfp4
    for m, n in ((0, 16), (4, 0)):
        N.check(fn(stream(), m, n, 64, *act, ptr(args["w"][0]), ptr(args["w"][1]), None, None, None, None, None, 1, ptr(out)))
    N.check(N.lib().mv_op_quantize_mxfp4(stream(), 0, 64, 1, ptr(out), 64, None, None, None))
    torch.cuda.synchronize()
    assert bool((out == 7).all())


@pytest.mark.parametrize("m", [2, 40, 300])
def test_results_do_not_depend_on_the_batch_or_the_run(m):
    """A row's result has the same bits on every run."""
    for kind in ("linear", "gemm"):
        args, _, _ = case(kind, m, 400, 2048, True, True, True, torch.bfloat16)
        first = product(kind, **args)
        for _ in range(5):
            assert torch.equal(product(kind, **args), first)


def test_products_on_two_streams_and_in_a_graph():
    """Calls share nothing: two streams at once, and a captured chain (quantise -> 4-bit product -> bf16 product) replayed on new inputs between
    eager calls."""
    m, n, k = 48, 640, 512
    g = torch.Generator().manual_seed(11)
    w, wb = tuple(map(dev, make(g, n, k))), tuple(map(dev, make(g, k, n)))
    x = torch.randn(m, k, generator=g).bfloat16().cuda()
    bufs = lambda: (torch.zeros(m, k // 2, dtype=torch.uint8, device="cuda"), torch.zeros(m, k // 32, dtype=torch.uint8, device="cuda"),  # noqa: E731
                    torch.zeros(m, n, dtype=torch.bfloat16, device="cuda"), torch.zeros(m, k, dtype=torch.float32, device="cuda"))

    def chain(src, b):
        lib, s = N.lib(), stream()
        N.check(lib.mv_op_quantize_mxfp4(s, m, k, 0, ptr(src), k, ptr(b[0]), ptr(b[1]), None))
        N.check(lib.mv_op_gemm_mxfp4(s, m, n, k, ptr(b[0]), ptr(b[1]), ptr(w[0]), ptr(w[1]), None, None, None, None, None, 0, ptr(b[2])))
        N.check(lib.mv_op_linear_mxfp4(s, m, k, n, ptr(b[2]), n, ptr(wb[0]), ptr(wb[1]), None, None, None, None, None, 1, ptr(b[3])))
        return b[3]

    want = chain(x, bufs()).clone()
    c64, s64 = o_mx.quantize(bits64(x))
    y, size = o_mx.product(o_mx.values(c64, s64, k), o_mx.values(w[0].cpu().numpy(), w[1].cpu().numpy(), k))
    mid = bufs()
    chain(x, mid)
    within(mid[2], y, size, k, torch.bfloat16)
    z, zsize = o_mx.product(bits64(mid[2]), o_mx.values(wb[0].cpu().numpy(), wb[1].cpu().numpy(), n))
    within(mid[3], z, zsize, n, torch.float32)

    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    b1, b2 = bufs(), bufs()
    torch.cuda.synchronize()
    for _ in range(8):
        with torch.cuda.stream(s1):
            chain(x, b1)
        with torch.cuda.stream(s2):
            chain(x, b2)
    torch.cuda.synchronize()
    assert torch.equal(b1[3], want) and torch.equal(b2[3], want)

    static, gb = x.clone(), bufs()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        chain(static, gb)
    for i in range(4):
        new = torch.randn(m, k, generator=g).bfloat16().cuda()
        static.copy_(new)
        graph.replay()
        eager = chain(new, bufs())
        torch.cuda.synchronize()
        assert torch.equal(gb[3], eager)


@pytest.mark.parametrize("kind", ["linear", "gemm"])
@pytest.mark.parametrize("m,n,k,gated", [(1, 512, 1024, False), (18, 8049, 1280, False), (64, 16384, 1024, False), (130, 9000, 1111, False), (250, 8200, 1000, True),
                                         (384, 16384, 512, False), (2048, 8192, 300, True)])
def test_every_tile_repeats_and_replays(kind, m, n, k, gated):
    """A captured call without one before it, replayed between eager ones: the same bits every time, and a NaN block of the weights reaches its own column
    alone."""
    args, want, size = case(kind, m, n, k, gated, False, False, torch.float32, make=make_fast)
    x, w, w2 = args["x"], args["w"], args["w2"] or (None, None)
    out = torch.zeros(m, n, device="cuda")
    act = (ptr(x), x.stride(0)) if kind == "linear" else (ptr(x[0]), ptr(x[1]))
    fn = N.lib().mv_op_linear_mxfp4 if kind == "linear" else N.lib().mv_op_gemm_mxfp4
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        N.check(fn(stream(), m, n, k, *act, ptr(w[0]), ptr(w[1]), ptr(w2[0]), ptr(w2[1]), None, None, None, 1, ptr(out)))
    graph.replay()
    torch.cuda.synchronize()
    within(out, want, size, k, torch.float32)
    first = out.clone()
    for _ in range(3):
        out.zero_()
        graph.replay()
        eager = product(kind, **args)
        torch.cuda.synchronize()
        assert torch.equal(out, first) and torch.equal(eager, first)
    w[1][n // 2, -1] = 255
    graph.replay()
    torch.cuda.synchronize()
    nan = torch.isnan(out)
    assert bool(nan[:, n // 2].all()) and int(nan.sum()) == m and torch.equal(out[~nan], first[~nan])


@pytest.mark.parametrize("kind", ["linear", "gemm"])
@pytest.mark.parametrize("m,n,k", [(5, 33, 95), (70, 300, 640), (1100, 1300, 640), (2300, 3900, 416)])
def test_buffers_at_odd_elements(kind, m, n, k):
    """Everything but the codes may begin at any element: outputs, residuals, biases, bf16 rows, scale bytes."""
    args, want, size = case(kind, m, n, k, False, True, True, torch.bfloat16, make=make_fast)

    def shift(t, dtype):
        room = torch.empty(t.numel() + 1, dtype=dtype, device="cuda")
        room[1:] = t.reshape(-1)
        return room[1:].view(t.shape)

    args["w"] = (args["w"][0], shift(args["w"][1], torch.uint8))
    args["bias"], args["residual"] = shift(args["bias"], torch.bfloat16), shift(args["residual"], torch.bfloat16)
    if kind == "linear":
        args["x"] = shift(args["x"].contiguous(), torch.bfloat16)
    else:
        args["x"] = (args["x"][0], shift(args["x"][1], torch.uint8))
    room = torch.full((m * n + 2,), 7.0, dtype=torch.bfloat16, device="cuda")
    out = room[1:m * n + 1]
    act = (ptr(args["x"]), k) if kind == "linear" else (ptr(args["x"][0]), ptr(args["x"][1]))
    fn = N.lib().mv_op_linear_mxfp4 if kind == "linear" else N.lib().mv_op_gemm_mxfp4
    N.check(fn(stream(), m, n, k, *act, ptr(args["w"][0]), ptr(args["w"][1]), None, None, ptr(args["bias"]), None, ptr(args["residual"]), 0, ptr(out)))
    torch.cuda.synchronize()
    assert float(room[0]) == 7 and float(room[-1]) == 7
    within(out.view(m, n), want, size, k, torch.bfloat16)


@pytest.mark.parametrize("m", [3, 70, 1100, 2300])
def test_infinities_and_nan_in_x_stay_in_their_rows(m):
    n, k = 1300 if m < 2000 else 3900, 429
    args, _, _ = case("linear", m, n, k, False, False, False, torch.float32, make=make_fast)
    first = product("linear", **args)
    args["x"] = args["x"].clone()
    args["x"][m - 1, k - 1], args["x"][0, 0] = float("nan"), float("inf")
    got = product("linear", **args)
    assert not bool(torch.isfinite(got[m - 1]).any()) and not bool(torch.isfinite(got[0]).all())
    assert torch.equal(got[1: m - 1], first[1: m - 1])


def codes_on_the_gpu(g, rows, k):
    nb = o_mx.blocks(k)
    assert k % 32 == 0
    return (torch.randint(0, 256, (rows, 16 * nb), generator=g, device="cuda", dtype=torch.uint8),
            torch.randint(120, 127, (rows, nb), generator=g, device="cuda", dtype=torch.uint8))


def host(c):
    return c[0].cpu().numpy(), c[1].cpu().numpy()


def rows_of(c, pick):
    return c[0][pick].contiguous(), c[1][pick].contiguous()


@pytest.fixture
def room():
    """Hands back what a test of large buffers took."""
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("kind,m,n,k", [("linear", 270000, 16, 8192), ("linear", 140000, 16384, 32), ("gemm", 140000, 16384, 64), ("linear", 2, 600000, 16384),
                                        ("gemm", 300, 600000, 16384), ("gemm", 1100000, 8, 8192)])
def test_offsets_past_32_bits(kind, m, n, k, room):
    """x, weights or output of more than 2^31 elements or 2^32 bytes: the last rows and columns against 64 bits."""
    g = torch.Generator(device="cuda").manual_seed(m + n)
    w = codes_on_the_gpu(g, n, k)
    x = codes_on_the_gpu(g, m, k) if kind == "gemm" else torch.randn(m, k, generator=g, device="cuda", dtype=torch.bfloat16)
    out = torch.full((m, n), 7.0, dtype=torch.bfloat16, device="cuda")
    act = (ptr(x), k) if kind == "linear" else (ptr(x[0]), ptr(x[1]))
    fn = N.lib().mv_op_linear_mxfp4 if kind == "linear" else N.lib().mv_op_gemm_mxfp4
    N.check(fn(stream(), m, n, k, *act, ptr(w[0]), ptr(w[1]), None, None, None, None, None, 0, ptr(out)))
    torch.cuda.synchronize()
    rows = torch.unique(torch.tensor([0, m // 2, max(0, m - 2), m - 1])).cuda()
    cols = torch.unique(torch.tensor([0, n // 2, n - 3, n - 1])).cuda()
    x64 = bits64(x[rows]) if kind == "linear" else o_mx.values(*host(rows_of(x, rows)), k)
    want, size = o_mx.product(x64, o_mx.values(*host(rows_of(w, cols)), k))
    within(out[rows][:, cols], want, size, k, torch.bfloat16)
    assert int((out == 7).sum()) < 0.05 * m * n  # no part was left out


def test_quantiser_offsets_past_32_bits(room):
    rows, k = 300000, 8192
    w = torch.randn(rows, k, device="cuda", dtype=torch.bfloat16)
    codes, scales, deq = hip_quantize(w)
    for lo in (0, rows // 2, rows - 50):
        check_quantised(w[lo:lo + 50], codes[lo:lo + 50], scales[lo:lo + 50], deq[lo:lo + 50])


@pytest.mark.parametrize("kind", ["linear", "gemm"])
@pytest.mark.parametrize("m,n", [(140000000, 1), (1, 140000000)])
def test_more_workgroups_than_one_grid_dimension_takes(kind, m, n, room):
    """8.75 million workgroups of 512 threads; two columns of K, so a result is a sum of two products: at most three fp32 half steps of their magnitudes
    (2^-24 each), then the output's own half step, 2^-8."""
    g = torch.Generator(device="cuda").manual_seed(m % 1000 + n % 1000)
    k = 2

    def two(rows):  # codes of the first two columns, zeros behind them; scale 1
        b = torch.zeros(rows, 16, dtype=torch.uint8, device="cuda")
        b[:, 0] = torch.randint(0, 256, (rows,), generator=g, device="cuda", dtype=torch.uint8)
        return b, torch.full((rows, 1), 127, dtype=torch.uint8, device="cuda")

    def values(c):
        table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
        return torch.stack([table[(c[0][:, 0] & 15).int()], table[(c[0][:, 0] >> 4).int()]], 1)

    w = two(n)
    x = two(m) if kind == "gemm" else torch.randn(m, k, generator=g, device="cuda", dtype=torch.bfloat16)
    out = torch.full((m, n), 7.5, dtype=torch.bfloat16, device="cuda")
    act = (ptr(x), k) if kind == "linear" else (ptr(x[0]), ptr(x[1]))
    fn = N.lib().mv_op_linear_mxfp4 if kind == "linear" else N.lib().mv_op_gemm_mxfp4
    N.check(fn(stream(), m, n, k, *act, ptr(w[0]), ptr(w[1]), None, None, None, None, None, 0, ptr(out)))
    torch.cuda.synchronize()
    long, short = (x, w) if m > n else (w, x)
    short = (values(short) if isinstance(short, tuple) else short).double()
    out = out.view(-1)
    for lo in range(0, max(m, n), 20000000):
        part = tuple(t[lo:lo + 20000000] for t in long) if isinstance(long, tuple) else long[lo:lo + 20000000]
        terms = (values(part) if isinstance(part, tuple) else part).double() * short
        want, size = terms.sum(1), terms.abs().sum(1)
        assert bool(((out[lo:lo + 20000000].double() - want).abs() <= 3 * 2.0 ** -24 * size + 2.0 ** -8 * want.abs()).all()), lo
