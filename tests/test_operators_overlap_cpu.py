"""What the MXFP4 operators and the logit controls refuse because an output shares bytes with another buffer: the first and the last byte of each, before
any device work (the addresses are made up)."""
import pytest

from conftest import load_pkg

N = load_pkg("_native")
BASE = 1 << 40
ROOM = 1 << 30


def places(*names):
    return {n: BASE + i * ROOM for i, n in enumerate(names)}


def refused(code):
    assert code == N.MV_ERR_INVALID
    assert "on top of" in N.lib().mv_last_error().decode()


def around(size, out_size, align):
    """Addresses relative to a buffer of `size` bytes at which an output of `out_size` bytes touches its first and its last byte."""
    return [-((out_size - 1) // align * align), (size - 1) // align * align]


M, K, COLS, NB = 5, 100, 48, 4
BUFFERS = dict(scales=COLS * NB, codes2=COLS * 16 * NB, scales2=COLS * NB, bias=COLS * 2, bias2=COLS * 2, codes=COLS * 16 * NB)


def linear(p, out_dtype=0, ldx=K):
    return N.lib().mv_op_linear_mxfp4(None, M, COLS, K, p["x"], ldx, p["codes"], p["scales"], p["codes2"], p["scales2"], p["bias"], p["bias2"], p["residual"], out_dtype, p["out"])


def gemm(p, out_dtype=0):
    return N.lib().mv_op_gemm_mxfp4(None, M, COLS, K, p["x"], p["xs"], p["codes"], p["scales"], p["codes2"], p["scales2"], p["bias"], p["bias2"], p["residual"], out_dtype, p["out"])


@pytest.mark.parametrize("out_dtype", [0, 1])
@pytest.mark.parametrize("name", list(BUFFERS) + ["x", "xs", "residual"])
def test_products_refuse_an_output_on_an_input(name, out_dtype):
    out = M * COLS * (4 if out_dtype else 2)
    for fn in (linear, gemm):
        if fn is linear and name == "xs":
            continue
        size = {"x": M * K * 2 if fn is linear else M * 16 * NB, "xs": M * NB, "residual": out, **BUFFERS}[name]
        for off in around(size, out, 4):
            p = places("x", "xs", "codes", "scales", "codes2", "scales2", "bias", "bias2", "residual", "out")
            p["out"] = p[name] + off
            refused(fn(p, out_dtype))


def test_linear_refuses_an_output_on_a_row_of_strided_x():
    for row in range(M):
        for at in (0, (K - 1) * 2, -2 * M * COLS + 2):
            p = places("x", "codes", "scales", "codes2", "scales2", "bias", "bias2", "residual", "out")
            p["out"] = p["x"] + row * 2000 + at
            refused(linear(p, ldx=1000))


@pytest.mark.parametrize("dtype", [0, 1])
def test_quantiser_refuses_outputs_on_buffers(dtype):
    esz = 4 if dtype else 2
    sizes = dict(w=M * K * esz, codes=M * 16 * NB, scales=M * NB, deq=M * K * 2)
    for a, align in (("codes", 16), ("scales", 1), ("deq", 2)):
        for b in sizes:
            if a == b:
                continue
            for off in around(sizes[b], sizes[a], align):
                p = places("w", "codes", "scales", "deq")
                p[a] = p[b] + off
                if p["codes"] % 16:
                    continue
                refused(N.lib().mv_op_quantize_mxfp4(None, M, K, dtype, p["w"], K, p["codes"], p["scales"], p["deq"]))


ROWS, V = 6, 100


def controls(p, dtype=0, out_dtype=0, ld=V, ld_out=V, uncond=True):
    c = N.mv_logit_controls(guidance=p["guidance"], repetition=p["repetition"], presence=p["presence"], frequency=p["frequency"], history=p["history"],
                            history_len=p["history_len"], prompt_len=p["prompt_len"], ld_history=9, history_cap=8, n_bias=3, bias_ids=p["bias_ids"], bias=p["bias"],
                            ld_bias=3, masks=p["masks"], mask_index=p["mask_index"], ld_mask=4, n_masks=2)
    return N.lib().mv_op_logit_controls(None, ROWS, V, dtype, p["logits"], p["uncond"] if uncond else None, ld, c, out_dtype, p["out"], ld_out, p["allowed"])


PER_ROW = ("guidance", "repetition", "presence", "frequency", "history_len", "prompt_len", "mask_index")
NAMES = ("logits", "uncond", "out", "allowed", "history", "bias_ids", "bias", "masks") + PER_ROW
SIZES = dict({n: ROWS * 4 for n in PER_ROW}, logits=ROWS * V * 2, uncond=ROWS * V * 2, out=ROWS * V * 2, allowed=ROWS * 4, history=(ROWS - 1) * 36 + 32, bias_ids=ROWS * 12,
             bias=ROWS * 12, masks=2 * 16)


@pytest.mark.parametrize("name", [n for n in NAMES if n not in ("out", "allowed")])
def test_controls_refuse_outputs_on_inputs(name):
    for output in ("out", "allowed"):
        for off in around(SIZES[name], SIZES[output], 4):
            p = places(*NAMES)
            p[output] = p[name] + off
            refused(controls(p))


def test_controls_refuse_outputs_on_each_other_and_rows_that_meet():
    p = places(*NAMES)
    p["allowed"] = p["out"] + ROWS * V * 2 - 4
    refused(controls(p))
    for off in (-2 * (V - 1), 2 * (V - 1), 2 * 300 - 2 * (V - 1), 5 * 600 + 2, -5 * 600 - 2):  # rows 300 apart, both
        p = places(*NAMES)
        p["out"] = p["logits"] + off
        refused(controls(p, ld=300, ld_out=300))
    for other in ("logits", "uncond"):
        p = places(*NAMES)
        p["out"] = p[other]
        refused(controls(p, ld_out=V + 1))
