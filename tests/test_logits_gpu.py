"""mv_op_logit_controls on the GPU against oracle/logits.py (64 bits).

Tolerance: a token passes at most 8 fp32 roundings, each half a step (2^-24) of the magnitudes that enter it (the oracle returns them); the output's
own rounding is half a step of its type (2^-8 bf16, 2^-24 fp32).  Counts, masks and infinities are exact."""
import ctypes as C

import numpy as np
import pytest
import torch

from conftest import load_pkg
from oracle import logits as o_lg
from oracle import mxfp4 as o_mx

pytestmark = pytest.mark.gpu

N = load_pkg("_native")
CODE = {torch.bfloat16: 0, torch.float32: 1}
BF, F = torch.bfloat16, torch.float32


def ptr(t):
    return None if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


def struct(d):
    """d: name -> device tensor, as mv_logit_controls names them."""
    h, b, m = d.get("history"), d.get("bias_ids"), d.get("masks")
    return N.mv_logit_controls(guidance=ptr(d.get("guidance")), repetition=ptr(d.get("repetition")), presence=ptr(d.get("presence")),
                               frequency=ptr(d.get("frequency")), history=ptr(h), history_len=ptr(d.get("history_len")), prompt_len=ptr(d.get("prompt_len")),
                               ld_history=0 if h is None else h.stride(0), history_cap=0 if h is None else h.shape[1],
                               bias_ids=ptr(b), bias=ptr(d.get("bias")), ld_bias=0 if b is None or b.shape[0] == 1 else b.stride(0),
                               n_bias=0 if b is None else b.shape[1], masks=ptr(m), mask_index=ptr(d.get("mask_index")),
                               ld_mask=0 if m is None else m.stride(0), n_masks=0 if m is None else m.shape[0])


def hip(logits, uncond, d, out_dtype, pad=0, in_place=False):
    rows, v = logits.shape
    allowed = torch.full((rows + 1,), -5, dtype=torch.int32, device="cuda")
    buf = logits if in_place else torch.full((rows + 1, v + pad), 7.0, dtype=out_dtype, device="cuda")
    N.check(N.lib().mv_op_logit_controls(stream(), rows, v, CODE[logits.dtype], ptr(logits), ptr(uncond), logits.stride(0), struct(d), CODE[out_dtype], ptr(buf),
                                         buf.stride(0), ptr(allowed)))
    torch.cuda.synchronize()
    assert int(allowed[rows]) == -5
    if in_place:
        return logits, allowed[:rows]
    assert bool((buf[rows] == 7).all()) and bool((buf[:, v:] == 7).all())
    return buf[:rows, :v], allowed[:rows]


def check(logits, uncond, d, out_dtype, **kw):
    host = {k: t.cpu().numpy() for k, t in d.items()}
    if "masks" in host:
        host["masks"] = host["masks"].view(np.uint32)
    want, allowed, size = o_lg.controls(logits.cpu().double().numpy(), None if uncond is None else uncond.cpu().double().numpy(), **host)
    # a result past the range of fp32 is an infinity there: rounding takes what lies half a step or more beyond the largest number to infinity
    # (the lowest fp32 number -3.4028e38 with guidance 2 and repetition 1.5 is about -1.02e39 in 64 bits, three times the largest fp32 number)
    top = float(torch.finfo(out_dtype).max) * (1 + (2.0 ** -9 if out_dtype == BF else 2.0 ** -25))
    want = np.where(np.abs(want) >= top, np.copysign(np.inf, want), want)
    got, n = hip(logits, uncond, d, out_dtype, **kw)
    got = got.cpu().double().numpy()
    assert np.array_equal(n.cpu().numpy(), allowed)
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine], equal_nan=True)
    half = 2.0 ** -8 if out_dtype == BF else 2.0 ** -24
    with np.errstate(invalid="ignore"):
        bad = fine & ~(np.abs(got - want) <= 8 * 2.0 ** -24 * size + half * np.abs(want))
    assert not bad.any(), f"{bad.sum()} off, first at {np.argwhere(bad)[0]}: {got[bad][0]} against {want[bad][0]}"


def controls(rows, v, g, cap=0, n_bias=0, n_masks=0, shared=False, penalties=True):
    d = {}
    if penalties:
        d.update(repetition=torch.rand(rows, generator=g) + 0.6, presence=torch.rand(rows, generator=g), frequency=torch.rand(rows, generator=g) * 0.3 - 0.05)
    if cap:
        d.update(history=(torch.rand(rows, cap, generator=g) ** 2 * (v + 2)).int() - 1, history_len=torch.randint(0, cap + 1, (rows,), generator=g).int(),
                 prompt_len=torch.randint(0, cap + 1, (rows,), generator=g).int())
        d["history_len"][0] = cap
    if n_bias:
        r = 1 if shared else rows
        d.update(bias_ids=torch.randint(-1, v + 1, (r, n_bias), generator=g).int(), bias=torch.randn(r, n_bias, generator=g) * 5)
    if n_masks:
        d.update(masks=torch.randint(-2 ** 31, 2 ** 31, (n_masks, (v + 31) // 32 + 1), generator=g).int(), mask_index=torch.randint(-1, n_masks + 1, (rows,), generator=g).int())
    return {k: t.cuda() for k, t in d.items()}


@pytest.mark.parametrize("rows,v", [(1, 1), (1, 3), (2, 31), (3, 33), (2, 2562), (5, 4095), (3, 4096), (2, 4097), (4, 8193), (2, 32003), (1, 131072)])
@pytest.mark.parametrize("dt,ot", [(BF, BF), (BF, F), (F, BF), (F, F)])
@pytest.mark.parametrize("cap,n_bias,n_masks", [(0, 0, 0), (1, 1, 1), (700, 40, 3), (3000, 700, 5)])
def test_controls(rows, v, dt, ot, cap, n_bias, n_masks):
    g = torch.Generator().manual_seed(rows * 31 + v + cap)
    pair = (torch.randn(rows, 2, v, generator=g) * 4 - 1).to(dt).cuda()
    d = controls(rows, v, g, cap, n_bias, n_masks, shared=n_bias == 40)
    d2 = dict(d, guidance=(torch.rand(rows, generator=g) * 4).cuda())
    check(pair[:, 0], pair[:, 1], d2, ot)           # the engine's layout: pairs of rows
    check(pair[:, 0].contiguous(), None, d, ot, pad=3)
    if dt == ot:
        check(pair[:, 0].contiguous(), None, d, ot, in_place=True)


@pytest.mark.parametrize("offset", [0, 1, 3])
def test_rows_at_any_alignment(offset):
    g = torch.Generator().manual_seed(2)
    for dt in (BF, F):
        big = torch.randn(4, 1000 + 7, generator=g).to(dt).cuda()
        check(big[:, offset:offset + 1000], None, controls(4, 1000, g, 50, 5, 2), dt, pad=offset)


def test_masked_places_hold_anything():
    """NaN, infinities and the type's lowest value in masked places and beside them; a row whose mask leaves nothing; a row with one token left."""
    g = torch.Generator().manual_seed(3)
    v = 100
    for dt in (BF, F):
        x = torch.randn(4, v, generator=g).to(dt)
        x[:, 0], x[:, 1], x[:, 2], x[:, 3] = float("nan"), float("inf"), float("-inf"), torch.finfo(dt).min
        u = torch.randn(4, v, generator=g).to(dt)
        u[:, 2] = float("-inf")
        masks = torch.zeros(3, 4, dtype=torch.int32)
        masks[0] = -1
        masks[0, 0] = -1 - 15  # the first four tokens forbidden
        masks[2, 1] = 1        # token 32 alone
        d = dict(masks=masks.cuda(), mask_index=torch.tensor([0, 1, 2, -1]).int().cuda(), guidance=torch.tensor([3.0, 1.0, 0.0, 2.0]).cuda(),
                 repetition=torch.full((4,), 1.5).cuda(), history=torch.tensor([[0, 1, 2, 3]] * 4).int().cuda())
        check(x.cuda(), u.cuda(), d, F)
        out, allowed = hip(x.cuda(), u.cuda(), d, F)
        assert allowed.tolist() == [v - 4, 0, 1, v]
        assert bool((out[1] == float("-inf")).all()) and int(torch.isfinite(out[2]).sum()) == 1 and float(out[3, 2]) == float("-inf")


def test_history_edges():
    """A history longer than its room, negative lengths, prompts longer than the history, ids that repeat, ids outside the vocabulary."""
    v = 64
    x = torch.linspace(-3, 3, v).repeat(5, 1).cuda()
    hist = torch.full((5, 9), 7).int()
    hist[2] = torch.tensor([-1, 64, 2 ** 31 - 1, -2 ** 31, 63, 0, 0, 0, 5])
    d = dict(history=hist.cuda(), history_len=torch.tensor([100, -3, 9, 9, 0]).int().cuda(), prompt_len=torch.tensor([-2, 0, 6, 100, 0]).int().cuda(),
             repetition=torch.full((5,), 2.0).cuda(), presence=torch.full((5,), 0.5).cuda(), frequency=torch.full((5,), 0.25).cuda())
    check(x, None, d, F)
    check(x, None, {k: d[k] for k in ("history", "frequency")}, F)   # no lengths: the whole room, no prompt
    check(x, None, {k: d[k] for k in ("repetition", "presence", "frequency")}, F)


def test_the_later_bias_entry_holds():
    v = 50
    ids = torch.randint(0, 4, (3, 2000)).int()
    d = dict(bias_ids=ids.cuda(), bias=torch.randn(3, 2000).cuda())
    for _ in range(3):
        check(torch.zeros(3, v).cuda(), None, d, F)
    d["bias"][:, -1] = float("-inf")
    check(torch.zeros(3, v).cuda(), None, d, F)


def test_masks_row_by_row():
    g = torch.Generator().manual_seed(8)
    v = 70
    d = dict(masks=torch.randint(-2 ** 31, 2 ** 31, (4, 3), generator=g).int().cuda())
    check(torch.randn(4, v, generator=g).cuda(), None, d, BF)


@pytest.fixture
def room():
    """Hands back what a test of large buffers took."""
    yield
    torch.cuda.empty_cache()


def test_offsets_past_32_bits(room):
    """20000 rows of 131072 tokens: the first and last rows against 64 bits."""
    rows, v = 20000, 131072
    g = torch.Generator().manual_seed(9)
    x = torch.randn(rows, v, device="cuda")
    d = controls(rows, v, g, 40, 5, 3)
    out, allowed = hip(x, None, d, BF)
    pick = torch.tensor([0, rows // 2, rows - 1])
    host = {k: (t if k == "masks" else t[pick.to(t.device)]).cpu().numpy() for k, t in d.items()}
    host["masks"] = host["masks"].view(np.uint32)
    want, n, size = o_lg.controls(x[pick.cuda()].cpu().double().numpy(), **host)
    got = out[pick.cuda()].cpu().double().numpy()
    fine = np.isfinite(want)
    assert np.array_equal(allowed[pick.cuda()].cpu().numpy(), n) and np.array_equal(got[~fine], want[~fine])
    assert (np.abs(got[fine] - want[fine]) <= (8 * 2.0 ** -24 * size + 2.0 ** -8 * np.abs(want))[fine]).all()


def test_more_workgroups_than_one_grid_dimension_takes(room):
    """Nine million rows of three tokens, two workgroups each: biases of one shared list and one of two masks are exact."""
    rows, v = 9000000, 3
    x = torch.randint(-50, 50, (rows, v), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).float()
    d = dict(bias_ids=torch.tensor([[2, 0]], dtype=torch.int32, device="cuda"), bias=torch.tensor([[4.0, -8.0]], device="cuda"),
             masks=torch.tensor([[0b111], [0b101]], dtype=torch.int32, device="cuda"), mask_index=(torch.arange(rows, device="cuda") % 2).int())
    got, n = hip(x, None, d, F)
    want = x + torch.tensor([-8.0, 0.0, 4.0], device="cuda")
    want[1::2, 1] = -float("inf")
    assert torch.equal(got, want)
    assert torch.equal(n, 3 - d["mask_index"])


def test_no_rows():
    y = torch.full((2, 8), 7.0, device="cuda")
    N.check(N.lib().mv_op_logit_controls(stream(), 0, 8, 1, None, None, 8, struct({}), 1, ptr(y), 8, None))
    torch.cuda.synchronize()
    assert bool((y == 7).all())


def test_decode_steps_together():
    """The operators as a serving loop uses them: an MXFP4 LM head over the conditioned and unconditioned row, the controls with the two-state grammar
    of interleaved codebooks, the sampler; the drawn token joins the history.  Greedy draws equal the 64-bit computation's, a captured step gives the
    tokens of the eager one, and every token obeys its state."""
    dim, v, steps = 256, 2562, 24
    g = torch.Generator().manual_seed(4)
    head = (torch.randn(v, dim, generator=g) / 16).bfloat16().cuda()
    emb = torch.randn(v, 2, dim, generator=g).bfloat16().cuda()
    codes, scales = torch.empty(v, dim // 2, dtype=torch.uint8, device="cuda"), torch.empty(v, dim // 32, dtype=torch.uint8, device="cuda")
    lib = N.lib()
    N.check(lib.mv_op_quantize_mxfp4(stream(), v, dim, 0, ptr(head), dim, ptr(codes), ptr(scales), None))
    torch.cuda.synchronize()
    w64 = o_mx.values(codes.cpu().numpy(), scales.cpu().numpy(), dim)
    masks = torch.zeros(2, (v + 31) // 32, dtype=torch.int32)
    masks[0, :32], masks[1, 32:64] = -1, -1                  # state 0: tokens 0 .. 1023, state 1: 1024 .. 2047
    x, logits, pair = torch.empty(2, dim, dtype=BF, device="cuda"), torch.empty(2, v, dtype=BF, device="cuda"), torch.zeros(2, v, dtype=BF, device="cuda")
    d = dict(guidance=torch.tensor([2.0]).cuda(), repetition=torch.tensor([1.3]).cuda(), presence=torch.tensor([0.2]).cuda(), frequency=torch.tensor([0.1]).cuda(),
             history=torch.zeros(1, steps + 1, dtype=torch.int32, device="cuda"), history_len=torch.zeros(1, dtype=torch.int32, device="cuda"),
             prompt_len=torch.tensor([1]).int().cuda(), bias_ids=torch.tensor([[5, 1030]]).int().cuda(), bias=torch.tensor([[0.5, -0.5]]).cuda(),
             masks=masks.cuda(), mask_index=torch.zeros(1, dtype=torch.int32, device="cuda"))
    allowed, token = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    c = struct(d)

    def step():
        s = stream()
        N.check(lib.mv_op_linear_mxfp4(s, 2, v, dim, ptr(x), dim, ptr(codes), ptr(scales), None, None, None, None, None, 0, ptr(logits)))
        N.check(lib.mv_op_logit_controls(s, 1, v, 0, ptr(logits), ptr(logits[1]), 2 * v, c, 0, ptr(pair), v, ptr(allowed)))

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    sp = N.mv_sampling(guidance_scale=1.0, one_minus_guidance=0.0, temperature=1.0, top_p=-1.0, top_k=1, seed=1)
    for captured in (False, True):
        d["history"].zero_()
        tok, ties = 3, 0
        for i in range(steps):
            d["history"][0, i] = tok
            d["history_len"].fill_(i + 1)
            d["mask_index"].fill_(i % 2)
            x.copy_(emb[tok])
            pair[0].fill_(0)
            torch.cuda.synchronize()
            graph.replay() if captured else step()
            torch.cuda.synchronize()
            N.check(lib.mv_op_sample(stream(), v, ptr(pair), C.byref(sp), i + 1, ptr(token), None))
            raw = x.cpu().double().numpy() @ w64.T
            host = {k: t.cpu().numpy() for k, t in d.items()}
            host["masks"] = host["masks"].view(np.uint32)
            want, n, _ = o_lg.controls(raw[:1], raw[1:], **host)
            tok = int(token.item())
            assert int(allowed.item()) == int(n[0]) == 1024 and 1024 * (i % 2) <= tok < 1024 * (i % 2) + 1024
            best = int(want[0].argmax())
            if tok != best:  # logits are rounded to bf16 twice on the way to the sampler: 3 and 1 half steps of at most |32|
                assert want[0, best] - want[0, tok] <= 2 * 4 * 2.0 ** -8 * 32
                ties += 1
        assert ties <= steps // 3
