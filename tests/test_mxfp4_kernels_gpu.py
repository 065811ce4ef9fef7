"""Every kernel of the MXFP4 products in every form, on shapes that are shown to reach it, where its loop runs past its prologue: more stages than LDS holds and
more groups of scales than are asked for ahead (tiles), more than one step per wave (row kernels).  test_mxfp4_kernels_cpu.py asserts the list without a GPU."""
import ctypes as C

import pytest
import torch

import test_mxfp4_gpu as base
from conftest import load_pkg
from test_mxfp4_gpu import CODE, case, make_fast, product, ptr, stream, within

pytestmark = pytest.mark.gpu

N = load_pkg("_native")

# kernel (0-2: few rows, 3-7: tiles), gated, form (row kernels: whole lines; tiles: scales by direct transfers), x by direct transfers, M, N, K, elements
# between rows of x
LINEAR = [
    (0, 0, 0, 0, 1, 33, 1533, 0), (0, 0, 0, 1, 1, 32, 1518, 0), (0, 0, 1, 1, 1, 32, 2560, 0), (0, 1, 0, 0, 1, 32, 1529, 0), (0, 1, 0, 1, 1, 32, 1518, 0),
    (0, 1, 1, 1, 1, 32, 2304, 0), (1, 0, 0, 0, 1, 11988, 3033, 0), (1, 0, 0, 1, 2, 8694, 2094, 0), (1, 0, 1, 1, 1, 10262, 3584, 0),
    (1, 1, 0, 0, 3, 8188, 3040, 1), (1, 1, 0, 1, 2, 8175, 4640, 0), (1, 1, 1, 1, 2, 8178, 4608, 0), (2, 0, 0, 0, 17, 6398, 1693, 0),
    (2, 0, 0, 1, 17, 6450, 1661, 1), (2, 0, 1, 1, 19, 6883, 2304, 0), (2, 1, 0, 0, 17, 5629, 1597, 0), (2, 1, 0, 1, 17, 5614, 1678, 0),
    (2, 1, 1, 1, 12, 11794, 2304, 0), (3, 0, 0, 0, 17, 10916, 2201, 0), (3, 0, 0, 1, 17, 11742, 2077, 1), (3, 0, 1, 0, 17, 8437, 2030, 1),
    (3, 0, 1, 1, 19, 8794, 2048, 0), (3, 1, 0, 0, 34, 3446, 2190, 1), (3, 1, 0, 1, 33, 3481, 2112, 0), (3, 1, 1, 0, 17, 4430, 2176, 1),
    (3, 1, 1, 1, 17, 4338, 2030, 0), (4, 0, 0, 0, 67, 10449, 1565, 0), (4, 0, 0, 1, 82, 8273, 1696, 0), (4, 0, 1, 0, 75, 8912, 1529, 0),
    (4, 0, 1, 1, 65, 8320, 1657, 1), (4, 1, 0, 0, 18, 8654, 2589, 0), (4, 1, 0, 1, 18, 12383, 1550, 0), (4, 1, 1, 0, 17, 8582, 1536, 1),
    (4, 1, 1, 1, 17, 8411, 1646, 0), (5, 0, 0, 0, 129, 11101, 1600, 1), (5, 0, 0, 1, 130, 11214, 1568, 0), (5, 0, 1, 0, 134, 12107, 1533, 0),
    (5, 0, 1, 1, 199, 8240, 1536, 0), (5, 1, 0, 0, 67, 10373, 1568, 1), (5, 1, 0, 1, 82, 8344, 1550, 0), (5, 1, 1, 0, 66, 9172, 1536, 1),
    (5, 1, 1, 1, 65, 8674, 1518, 0), (6, 0, 0, 1, 324, 11091, 1568, 0), (6, 0, 1, 1, 667, 5892, 1536, 0), (6, 1, 0, 1, 129, 11227, 1565, 1),
    (6, 1, 1, 1, 135, 11507, 1518, 0), (7, 0, 0, 1, 965, 8202, 1550, 0), (7, 0, 1, 1, 926, 8885, 1518, 0), (7, 1, 0, 1, 329, 11200, 1550, 0),
    (7, 1, 1, 1, 321, 11339, 1529, 1),
]
GEMM = [
    (0, 0, 0, 1, 1, 32, 1568, 0), (0, 0, 1, 1, 1, 32, 2286, 0), (0, 1, 0, 1, 1, 32, 1550, 0), (0, 1, 1, 1, 1, 32, 2286, 0), (1, 0, 0, 1, 3, 8305, 2670, 0),
    (1, 0, 1, 1, 3, 9725, 2286, 0), (1, 1, 0, 1, 17, 3915, 1565, 0), (1, 1, 1, 1, 3, 8191, 5629, 0), (2, 0, 0, 1, 17, 5000, 1661, 0),
    (2, 0, 1, 1, 17, 4893, 2304, 0), (2, 1, 0, 1, 17, 4926, 1550, 0), (2, 1, 1, 1, 17, 17154, 2304, 0), (3, 0, 0, 1, 17, 8239, 3104, 0),
    (3, 0, 1, 1, 33, 3782, 3193, 0), (3, 1, 0, 1, 17, 4165, 3097, 0), (3, 1, 1, 1, 17, 2901, 3310, 0), (4, 0, 0, 1, 67, 8343, 2574, 0),
    (4, 0, 1, 1, 65, 8221, 2542, 0), (4, 1, 0, 1, 17, 8827, 2621, 0), (4, 1, 1, 1, 2, 12330, 6909, 0), (5, 0, 0, 1, 136, 10883, 2112, 0),
    (5, 0, 1, 1, 130, 11390, 2176, 0), (5, 1, 0, 1, 68, 8537, 2080, 0), (5, 1, 1, 1, 69, 8382, 2048, 0), (6, 0, 0, 1, 262, 11758, 1550, 0),
    (6, 0, 1, 1, 279, 11462, 1536, 0), (6, 1, 0, 1, 134, 8519, 1568, 0), (6, 1, 1, 1, 133, 8403, 1536, 0), (7, 0, 0, 1, 774, 9516, 1597, 0),
    (7, 0, 1, 1, 647, 10886, 1661, 0), (7, 1, 0, 1, 263, 11570, 1565, 0), (7, 1, 1, 1, 273, 11222, 1536, 0),
]
CASES = [("linear", *c) for c in LINEAR] + [("gemm", *c) for c in GEMM]


def chosen(kind, m, n, k, gated, ldx, x=4096, codes=4096, scales=4096):
    """What mv_debug_mxfp4_kernel says, by name."""
    out = (C.c_int32 * 8)()
    N.check(N.lib().mv_debug_mxfp4_kernel(int(kind == "gemm"), m, n, k, ldx, int(gated), x, codes, scales, out))
    return dict(zip(("kernel", "lines", "x_direct", "s_direct", "steps", "bufs", "groups", "ahead"), out))


def reaches(got, kernel, form, x_direct):
    """Is that this kernel in this form, with its loop past the prologue?"""
    if kernel < 3:
        return (got["kernel"], got["lines"], got["x_direct"]) == (kernel, form, x_direct) and got["steps"] > 1
    return ((got["kernel"], got["s_direct"], got["x_direct"]) == (kernel, form, x_direct) and got["steps"] > got["bufs"] + 1
            and got["groups"] > got["ahead"] + 1)


@pytest.mark.parametrize("kind,kernel,gated,form,x_direct,m,n,k,pad", CASES)
def test_kernel(kind, kernel, gated, form, x_direct, m, n, k, pad):
    full = kernel % 2 == 0  # every second kernel with everything around the product
    dtype = torch.float32 if full else torch.bfloat16
    args, want, size = case(kind, m, n, k, bool(gated), full, full, dtype, pad, make=make_fast)
    x = args["x"] if kind == "linear" else args["x"][0]
    assert reaches(chosen(kind, m, n, k, gated, k + pad, x.data_ptr(), args["w"][0].data_ptr(), args["w"][1].data_ptr()), kernel, form, x_direct)
    first = product(kind, **args)
    within(first, want, size, k, dtype)
    for _ in range(3):
        assert torch.equal(product(kind, **args), first)
    args["w"][1][n // 3, -1] = 255  # a NaN block in a last group of scales: its own column and nothing else
    nan = torch.isnan(product(kind, **args))
    assert bool(nan[:, n // 3].all()) and int(nan.sum()) == m


# one shape of each tile, the first replayed without a call before it
REPLAYED = [c for i, c in enumerate(CASES) if c[1] >= 3 and c[8] == 0 and not any(d[:3] == c[:3] and d[8] == 0 for d in CASES[:i])]


@pytest.mark.parametrize("kind,kernel,gated,form,x_direct,m,n,k,pad", REPLAYED)
def test_tile_replays(kind, kernel, gated, form, x_direct, m, n, k, pad):
    base.test_every_tile_repeats_and_replays(kind, m, n, k, bool(gated))


@pytest.mark.parametrize("stride,tiled", [(1 << 22, True), ((1 << 22) + 64, False)])
def test_rows_far_apart(stride, tiled):
    """Rows 8 MB apart, 2.5 GB of them: tiles count bytes in 32 bits up to a stride of 2^23, the row kernels take what is beyond."""
    m, n, k = 300, 3000, 640
    args, want, size = case("linear", m, n, k, False, False, False, torch.float32, make=make_fast)
    room = torch.empty(m * stride, dtype=torch.bfloat16, device="cuda")
    x = room.as_strided((m, k), (stride, 1))
    x.copy_(args["x"])
    assert (chosen("linear", m, n, k, False, stride)["kernel"] >= 3) == tiled and chosen("linear", m, n, k, False, k)["kernel"] >= 3
    out = torch.full((m, n), 7.0, device="cuda")
    N.check(N.lib().mv_op_linear_mxfp4(stream(), m, n, k, ptr(x), stride, ptr(args["w"][0]), ptr(args["w"][1]), None, None, None, None, None, CODE[torch.float32], ptr(out)))
    torch.cuda.synchronize()
    within(out, want, size, k, torch.float32)
    del room, x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("kind,kernel,gated,form,x_direct,m,n,k,pad", [c for c in CASES if c[0] == "linear" and c[4] == 1])
def test_nan_between_rows_of_x(kind, kernel, gated, form, x_direct, m, n, k, pad):
    """What lies between the rows of x and behind the last one is not read, or not used: NaN there, beside a K that ends inside a block."""
    k -= 5 if k % 32 == 0 else 0
    ld = (k + 127) // 64 * 64 + (0 if kernel > 2 or form else 2)
    args, want, size = case("linear", m, n, k, bool(gated), False, False, torch.float32, make=make_fast)
    room = torch.full((m + 1, ld), float("nan"), dtype=torch.bfloat16, device="cuda")
    room[:m, :k] = args["x"]
    args["x"] = room[:m, :k]
    assert reaches(chosen("linear", m, n, k, gated, ld, room.data_ptr()), kernel, form, x_direct)
    within(product("linear", **args), want, size, k, torch.float32)
