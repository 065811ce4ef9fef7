"""The shapes of test_mxfp4_kernels_gpu.py reach what they are listed for, and leave no kernel and no form of one out.  No GPU."""
import pytest

from test_mxfp4_kernels_gpu import CASES, N, chosen, reaches


@pytest.mark.parametrize("kind,kernel,gated,form,x_direct,m,n,k,pad", CASES)
def test_shape_reaches_its_kernel(kind, kernel, gated, form, x_direct, m, n, k, pad):
    got = chosen(kind, m, n, k, gated, k + pad)
    assert reaches(got, kernel, form, x_direct), got


def test_every_kernel_in_every_form():
    listed = {c[:5] for c in CASES}
    assert len(listed) == len(CASES)
    for kind in ("linear", "gemm"):
        for kernel in range(8):
            for gated in (0, 1):
                for form in (0, 1):
                    # rows of x that begin at odd elements: bf16 alone, neither on whole lines nor in the two largest tiles
                    for x_direct in (1,) if kind == "gemm" or kernel > 5 or (kernel < 3 and form) else (0, 1):
                        assert (kind, kernel, gated, form, x_direct) in listed


def test_the_choice_goes_by_sizes_and_alignment():
    assert chosen("gemm", 2048, 8192, 4096, False, 0)["kernel"] == 7 and chosen("linear", 1, 100, 100, False, 100)["kernel"] == 0
    assert chosen("linear", 2048, 8192, 4096, False, 4097)["kernel"] == 5  # the two largest tiles have no registers for rows at odd elements
    assert chosen("linear", 2048, 8192, 4096, False, 1 << 23)["kernel"] < 3
    a = chosen("linear", 16, 2048, 4096, False, 4096)
    assert a["lines"] and not chosen("linear", 16, 2048, 4096, False, 4096, x=4096 + 64)["lines"]
    assert not chosen("linear", 16, 2048, 4096, False, 4096, scales=4097)["s_direct"]
    for bad in (dict(m=0), dict(n=0), dict(k=0), dict(ldx=99)):
        with pytest.raises(ValueError):
            chosen(**{**dict(kind="linear", m=5, n=5, k=100, gated=False, ldx=100), **bad})
