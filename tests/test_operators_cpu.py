"""No-GPU checks of the MXFP4 products and the logit controls: the struct's layout, what the calls refuse (before any device work), and the 64-bit
definitions against hand-made values."""
import ctypes as C

import numpy as np
import pytest

from conftest import load_pkg
from oracle import logits as o_lg
from oracle import mxfp4 as o_mx

N = load_pkg("_native")
A = 4096  # an address aligned to everything; refused calls never follow it


def refused(code, text):
    assert code == N.MV_ERR_INVALID
    assert text in N.lib().mv_last_error().decode()
    with pytest.raises(ValueError):
        N.check(code)


def test_struct_layout():
    s = N.mv_logit_controls
    assert C.sizeof(s) == 128 and s.ld_history.offset == 56 and s.bias_ids.offset == 72 and s.ld_mask.offset == 112


def quantize(n=4, k=64, dtype=0, w=A, ldw=64, codes=A, scales=A, deq=None):
    return N.lib().mv_op_quantize_mxfp4(None, n, k, dtype, w, ldw, codes, scales, deq)


@pytest.mark.parametrize("kw,text", [(dict(n=-1), "shape"), (dict(k=0), "shape"), (dict(k=2 ** 31 - 1, ldw=2 ** 40), "shape"), (dict(dtype=2), "dtype"),
                                     (dict(dtype=3), "dtype"), (dict(ldw=63), "ldw"), (dict(ldw=-64), "ldw"), (dict(w=None), "null"), (dict(codes=None), "null"),
                                     (dict(scales=None), "null"), (dict(codes=A + 8), "aligned"), (dict(w=A + 1), "aligned"),
                                     (dict(w=A + 2, dtype=1), "aligned"), (dict(deq=A + 1), "aligned"), (dict(), "on top"),
                                     (dict(codes=2 * A), "on top"), (dict(codes=2 * A, scales=3 * A, deq=A, dtype=1), "on top"),
                                     (dict(codes=2 * A, scales=3 * A, deq=A, ldw=65), "on top")])
def test_quantize_refuses(kw, text):
    refused(quantize(**kw), text)


def linear(m=4, n=8, k=64, x=A, ldx=64, codes=A, scales=A, codes2=None, scales2=None, bias=None, bias2=None, residual=None, out_dtype=0, out=2 * A):
    return N.lib().mv_op_linear_mxfp4(None, m, n, k, x, ldx, codes, scales, codes2, scales2, bias, bias2, residual, out_dtype, out)


def gemm(m=4, n=8, k=64, x=A, xs=A, codes=A, scales=A, codes2=None, scales2=None, bias=None, bias2=None, residual=None, out_dtype=0, out=2 * A):
    return N.lib().mv_op_gemm_mxfp4(None, m, n, k, x, xs, codes, scales, codes2, scales2, bias, bias2, residual, out_dtype, out)


@pytest.mark.parametrize("fn", [linear, gemm])
@pytest.mark.parametrize("kw,text", [(dict(m=-1), "negative"), (dict(n=-1), "negative"), (dict(k=0), "positive"), (dict(k=-5), "positive"),
                                     (dict(out=A), "on top"), (dict(m=2 ** 31 - 1), "too large"), (dict(n=2 ** 31 - 1), "too large"),
                                     (dict(out_dtype=2), "out_dtype"), (dict(codes=None), "null"), (dict(scales=None), "null"), (dict(out=None), "null"),
                                     (dict(x=None), "x"), (dict(codes2=A), "together"), (dict(scales2=A), "together"), (dict(bias2=A), "bias2"),
                                     (dict(codes=A + 4), "16 bytes"), (dict(codes2=A + 4, scales2=A), "16 bytes"), (dict(out=A + 1), "element"),
                                     (dict(out=A + 2, out_dtype=1), "element"), (dict(residual=A + 2, out_dtype=1), "element"), (dict(bias=A + 1), "element")])
def test_products_refuse(fn, kw, text):
    refused(fn(**kw), text)


def test_products_refuse_their_own():
    refused(linear(ldx=63), "ldx")
    refused(linear(x=A + 1), "x")
    refused(gemm(x=A + 8), "x_codes")
    refused(gemm(xs=None), "x_scales")


def controls(rows=2, vocab=64, dtype=0, logits=A, uncond=None, ld=64, out_dtype=0, out=2 * A, ld_out=64, allowed=None, null=False, **c):
    s = N.mv_logit_controls(**c)
    return N.lib().mv_op_logit_controls(None, rows, vocab, dtype, logits, uncond, ld, None if null else s, out_dtype, out, ld_out, allowed)


@pytest.mark.parametrize("kw,text", [(dict(rows=-1), "shape"), (dict(vocab=0), "shape"), (dict(dtype=2), "dtype"), (dict(out_dtype=3), "dtype"), (dict(ld=63), "stride"),
                                     (dict(ld_out=63), "stride"), (dict(null=True), "null"), (dict(logits=None), "null"), (dict(out=None), "null"),
                                     (dict(uncond=A), "guidance"), (dict(out=A, out_dtype=1), "on top"), (dict(out=A, ld_out=65), "on top"),
                                     (dict(uncond=3 * A, guidance=A, out=3 * A, ld_out=65), "on top"), (dict(history=A, history_cap=8, ld_history=7), "ld_history"), (dict(history_cap=8), "history_cap"),
                                     (dict(history_cap=-1), "negative"), (dict(n_bias=-1), "negative"), (dict(n_masks=-1), "negative"),
                                     (dict(bias_ids=A, n_bias=3), "go together"), (dict(bias=A, n_bias=3), "go together"), (dict(n_bias=3), "go together"),
                                     (dict(bias_ids=A, bias=A, n_bias=3, ld_bias=2), "ld_bias"), (dict(mask_index=A), "masks"), (dict(n_masks=2), "masks"),
                                     (dict(masks=A, n_masks=2, ld_mask=1), "ld_mask"), (dict(masks=A, n_masks=1, ld_mask=2), "mask_index"),
                                     (dict(logits=A + 1), "aligned"), (dict(out=A + 2, out_dtype=1), "aligned"), (dict(uncond=A + 1, guidance=A), "aligned"),
                                     (dict(guidance=A + 2), "aligned"), (dict(history=A + 1, history_cap=8, ld_history=8), "aligned"), (dict(allowed=A + 2), "aligned"),
                                     (dict(masks=A + 2, n_masks=2, ld_mask=2), "aligned"), (dict(vocab=2 ** 31 - 1, ld=2 ** 31, ld_out=2 ** 31), "too large"),
                                     (dict(history=A, history_cap=2 ** 31 - 1, ld_history=2 ** 31), "too large"),
                                     (dict(bias_ids=A, bias=A, n_bias=2 ** 31 - 1), "too large"),
                                     (dict(rows=2 ** 31 - 1, vocab=8193, ld=8193, ld_out=8193), "too large")])
def test_controls_refuse(kw, text):
    refused(controls(**kw), text)


def test_definitions_by_hand():
    w = np.zeros((1, 33))
    w[0, :8] = [6, -6.5, 7.9, 0.25, 0.75, -1.25, 5.0, 3.5]
    w[0, 32] = -2.0 ** -10
    codes, scales = o_mx.quantize(w)
    assert scales.tolist() == [[127, 115]]
    assert o_mx.values(codes, scales, 33)[0, :8].tolist() == [6, -6, 6, 0, 1, -1, 4, 4] and o_mx.values(codes, scales, 33)[0, 32] == -2.0 ** -10
    out, n, _ = o_lg.controls(np.array([[1.0, -1.0, 2.0, 0.0]]), history=np.array([[1, 0, 0, 2]]), prompt_len=np.array([1]), repetition=np.array([2.0]),
                              presence=np.array([0.5]), frequency=np.array([0.25]), bias_ids=np.array([[3, 3]]), bias=np.array([[1.0, 2.0]]),
                              masks=np.array([[0b1011]], dtype=np.uint32))
    assert out[0].tolist() == [0.5 - 0.5 - 0.5, -2.0, -np.inf, 2.0] and n.tolist() == [3]
