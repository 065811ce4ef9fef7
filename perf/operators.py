"""Workloads of the microscaled 4-bit (MXFP4) products and of the logit controls, with their plain forms.

Four operators of the C ABI (include/metavoice_hip.h): `mv_op_quantize_mxfp4`, `mv_op_linear_mxfp4` (bf16 activations), `mv_op_gemm_mxfp4`
(both operands in 4 bits) and `mv_op_logit_controls`.  `run` computes a case either in elementary torch operations (`own` false) or through the
library (`own` true); `exact` computes it in 64 bits, written apart from both.

MXFP4: a row of K values is cut into blocks of 32 (the last one may be short).  A block holds 32 codes of 4 bits (sign, 2 exponent bits, 1 mantissa
bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6) and one scale byte s standing for 2^(s - 127), 255 for NaN.  codes: [rows][16 * ceil(K / 32)] bytes, column 2j in the
low and column 2j + 1 in the high nibble of byte j; scales: [rows][ceil(K / 32)] bytes.
"""
import importlib
import math

import torch

own = False

BF16, F32 = "bf16", "f32"
_TORCH = {BF16: torch.bfloat16, F32: torch.float32}
_SIZE = {BF16: 2, F32: 4}
_CODE = {BF16: 0, F32: 1}  # mv_dtype


# ---- the cases ------------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the LM head of the first-stage model (2562 tokens, width 2048), quantised when the weights are loaded
        dict(name="quantize_head", op="quantize", rows=2562, k=2048, dtype=BF16, pad=0),
        # a large feed-forward matrix of float32 checkpoint weights
        dict(name="quantize_large", op="quantize", rows=28672, k=8192, dtype=F32, pad=0),
        # one utterance's decode step: the LM head over its conditioned and unconditioned row; the smallest call, latency counts
        dict(name="linear_head_m2", op="linear", m=2, n=2562, k=2048, gated=False, bias=False, residual=False, out=BF16, pad=0),
        # eight utterances decoded together: the gated feed-forward pair
        dict(name="linear_gate_m16", op="linear", m=16, n=5632, k=2048, gated=True, bias=False, residual=False, out=BF16, pad=0),
        # a short ragged prompt through an oddly sized layer with a bias, activations cut out of a wider buffer
        dict(name="linear_odd_m77", op="linear", m=77, n=2001, k=1111, gated=False, bias=True, residual=True, out=F32, pad=9),
        # a long batched prompt through a large layer
        dict(name="linear_prefill_m4096", op="linear", m=4096, n=16384, k=8192, gated=False, bias=False, residual=False, out=BF16, pad=0),
        # decode with 4-bit activations: the down projection of eight utterances
        dict(name="gemm_down_m16", op="gemm", m=16, n=2048, k=5632, gated=False, bias=False, residual=True, out=BF16, pad=0),
        # a prompt of 128 tokens in its two rows through the gated pair
        dict(name="gemm_gate_m256", op="gemm", m=256, n=5632, k=2048, gated=True, bias=False, residual=False, out=BF16, pad=0),
        # the same product at the size of a large batched prompt
        dict(name="gemm_large_m8192", op="gemm", m=8192, n=16384, k=8192, gated=False, bias=False, residual=False, out=BF16, pad=0),
        # one utterance near the end of its context: guidance, penalties, and the two-state grammar of interleaved codebooks
        dict(name="controls_one", op="controls", rows=1, vocab=2562, dtype=BF16, out=BF16, guidance=True, history=2016, penalties=True, n_bias=0,
             states=2, empty=False),
        # a serving batch over a text vocabulary of odd size, with user biases and a grammar that leaves one row nothing
        dict(name="controls_batch", op="controls", rows=64, vocab=32003, dtype=BF16, out=F32, guidance=False, history=4096, penalties=True,
             n_bias=300, states=16, empty=True),
        # a large batch over a large vocabulary
        dict(name="controls_large", op="controls", rows=256, vocab=131072, dtype=F32, out=F32, guidance=False, history=1024, penalties=True, n_bias=64,
             states=64, empty=False),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "gemm", "gemm", "controls"])
    if op == "quantize":
        return dict(op=op, rows=_log(rng, 1, 28672), k=_log(rng, 1, 8192), dtype=rng.choice([BF16, F32]), pad=rng.choice([0, 0, 1, 8, 56]))
    if op in ("linear", "gemm"):
        gated = rng.random() < 0.3
        m, n, k = _log(rng, 1, 4096 if op == "linear" else 8192), _log(rng, 16, 16384), _log(rng, 32, 8192)
        if rng.random() < 0.5:  # model widths are usually multiples of 64; the other half stays as odd as it was drawn
            n, k = (n + 63) // 64 * 64, (k + 63) // 64 * 64
        if gated:
            n = (n + 1) // 2
        return dict(op=op, m=m, n=n, k=k, gated=gated, bias=rng.random() < 0.4, residual=rng.random() < 0.4, out=rng.choice([BF16, BF16, F32]),
                    pad=rng.choice([0, 0, 8, 3]) if op == "linear" else 0)
    return dict(op=op, rows=_log(rng, 1, 256), vocab=_log(rng, 257, 131072), dtype=rng.choice([BF16, F32]), out=rng.choice([BF16, F32]),
                guidance=rng.random() < 0.5, history=rng.choice([0, 1, _log(rng, 2, 4096)]), penalties=rng.random() < 0.8,
                n_bias=rng.choice([0, 1, _log(rng, 2, 1000)]), states=rng.choice([0, 2, 17, 64]), empty=rng.random() < 0.3)


# ---- inputs ---------------------------------------------------------------------------------------------------------------------------
def _fp4(x):
    """Plain quantiser: [rows][K] -> codes [rows][nb][32] uint8 (not packed), exponents [rows][nb] int32 (128 = NaN)."""
    rows, k = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -k % 32)).view(rows, -1, 32)
    mag = x.abs()
    top = mag.amax(-1)
    e = (torch.frexp(top).exponent - 3).clamp(-127, 127)
    e = torch.where(top == 0, torch.full_like(e, -127), e)
    y = mag * ((127 - e) << 23).view(torch.float32).unsqueeze(-1)
    q = ((y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0)).to(torch.uint8)
    q = q + torch.signbit(x).to(torch.uint8) * 8
    return q, torch.where(torch.isfinite(top), e, torch.full_like(e, 128))


def _values(q, e):
    """Codes [rows][nb][32] and exponents [rows][nb] -> float32 [rows][32 nb]."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=q.device)
    v = grid[(q & 7).long()]
    v = torch.where(q >= 8, -v, v)
    h = torch.div(e, 2, rounding_mode="floor")  # 2^e in two factors: 2^-127 alone is below the smallest normal number
    v = v * ((h + 127) << 23).view(torch.float32).unsqueeze(-1) * ((e - h + 127) << 23).view(torch.float32).unsqueeze(-1)
    return torch.where(e.unsqueeze(-1) == 128, torch.full_like(v, math.nan), v).flatten(1)


def _pack(x):
    q, e = _fp4(x)
    q = q.flatten(1)
    return (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous(), (e + 127).to(torch.uint8).contiguous()


def _unpack(codes, scales, k):
    rows, nb = scales.shape
    q = torch.stack([codes & 15, codes >> 4], dim=-1).view(rows, nb, 32)
    return _values(q, scales.int() - 127)[:, :k]


def _native():
    return importlib.import_module("metavoice-src_amd._native")


def _p(t):
    return None if t is None else t.data_ptr()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def randint(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device="cuda")

    st = dict(case)
    if case["op"] == "quantize":
        rows, k, dt = case["rows"], case["k"], _TORCH[case["dtype"]]
        nb = (k + 31) // 32
        w = randn(rows, k + case["pad"]).mul_(0.02).to(dt)
        w[:, :: 97] *= 12  # a few columns with larger weights, as checkpoints have them
        st.update(w=w[:, :k], codes=torch.empty(rows, 16 * nb, dtype=torch.uint8, device="cuda"),
                  scales=torch.empty(rows, nb, dtype=torch.uint8, device="cuda"), deq=torch.empty(rows, k, dtype=torch.bfloat16, device="cuda"))
        if own:
            st["args"] = (rows, k, _CODE[case["dtype"]], _p(st["w"]), k + case["pad"], _p(st["codes"]), _p(st["scales"]), _p(st["deq"]))
        return st
    if case["op"] in ("linear", "gemm"):
        m, n, k = case["m"], case["n"], case["k"]
        x = randn(m, k + case["pad"]).to(torch.bfloat16)
        if case["op"] == "gemm":
            st["x"], st["xs"] = _pack(x)
            del x
        else:
            st["x"] = x[:, :k]
        st["w"], st["ws"] = _pack(randn(n, k) / math.sqrt(k))
        st["w2"], st["ws2"] = _pack(randn(n, k) / math.sqrt(k)) if case["gated"] else (None, None)
        st["b"] = randn(n).to(torch.bfloat16) if case["bias"] else None
        st["b2"] = randn(n).to(torch.bfloat16) if case["bias"] and case["gated"] else None
        st["res"] = randn(m, n).to(_TORCH[case["out"]]) if case["residual"] else None
        st["y"] = torch.empty(m, n, dtype=_TORCH[case["out"]], device="cuda")
        if own:
            act = (_p(st["x"]), _p(st["xs"])) if case["op"] == "gemm" else (_p(st["x"]), k + case["pad"])
            st["args"] = (m, n, k) + act + (_p(st["w"]), _p(st["ws"]), _p(st["w2"]), _p(st["ws2"]), _p(st["b"]), _p(st["b2"]), _p(st["res"]),
                                            _CODE[case["out"]], _p(st["y"]))
        return st
    rows, v, h, nbias, states = case["rows"], case["vocab"], case["history"], case["n_bias"], case["states"]
    pair = 2 if case["guidance"] else 1
    st["logits"] = (randn(rows, pair, v) * 3 - 2).to(_TORCH[case["dtype"]])  # as the model leaves them: the unconditioned row behind the conditioned
    st["g"] = torch.rand(rows, generator=g, device="cuda") * 3 + 1 if case["guidance"] else None
    pen = case["penalties"]
    st["rho"] = torch.rand(rows, generator=g, device="cuda") + 0.8 if pen else None
    st["pres"] = torch.rand(rows, generator=g, device="cuda") if pen else None
    st["freq"] = torch.rand(rows, generator=g, device="cuda") * 0.2 if pen else None
    # what a model says repeats itself: squared uniforms crowd the low ids
    st["hist"] = (torch.rand(rows, h, generator=g, device="cuda") ** 2 * v).int().clamp_(max=v - 1) if h else None
    st["hist_len"] = randint(0, h + 1, rows).int() if h else None
    st["prompt_len"] = (st["hist_len"] // 4).int() if h else None
    st["bias_ids"] = randint(0, v, rows, nbias).int() if nbias else None
    if nbias:
        st["bias_ids"][:, nbias - nbias // 8:] = -1  # lists of unequal length, filled up with -1
    st["bias"] = randn(rows, nbias) * 4 if nbias else None
    words = (v + 31) // 32
    st["masks"] = randint(-2 ** 31, 2 ** 31, states, words).int() if states else None
    st["state"] = randint(-1, states, rows).int() if states else None  # -1: the row has no grammar
    if states and case["empty"]:
        st["masks"][states - 1] = 0
        st["state"][rows - 1] = states - 1
    st["y"] = torch.empty(rows, v, dtype=_TORCH[case["out"]], device="cuda")
    st["allowed"] = torch.empty(rows, dtype=torch.int32, device="cuda")
    if own:
        c = _native().mv_logit_controls(guidance=_p(st["g"]), repetition=_p(st["rho"]), presence=_p(st["pres"]), frequency=_p(st["freq"]),
                                        history=_p(st["hist"]), history_len=_p(st["hist_len"]), prompt_len=_p(st["prompt_len"]), ld_history=h,
                                        history_cap=h, bias_ids=_p(st["bias_ids"]), bias=_p(st["bias"]), ld_bias=nbias, n_bias=nbias,
                                        masks=_p(st["masks"]), mask_index=_p(st["state"]), ld_mask=words, n_masks=states)
        uncond = st["logits"][:, 1] if case["guidance"] else None
        st["controls"] = c
        st["args"] = (rows, v, _CODE[case["dtype"]], _p(st["logits"]), _p(uncond), pair * v, c, _CODE[case["out"]], _p(st["y"]), v, _p(st["allowed"]))
    return st


# ---- one pass -------------------------------------------------------------------------------------------------------------------------
def run(st):
    if own:
        return _run_own(st)
    if st["op"] == "quantize":
        return _values(*_fp4(st["w"]))[:, : st["k"]].to(torch.bfloat16)
    if st["op"] in ("linear", "gemm"):
        x = st["x"].float() if st["op"] == "linear" else _unpack(st["x"], st["xs"], st["k"])
        y = x @ _unpack(st["w"], st["ws"], st["k"]).t()
        if st["b"] is not None:
            y = y + st["b"].float()
        if st["w2"] is not None:
            u = x @ _unpack(st["w2"], st["ws2"], st["k"]).t()
            if st["b2"] is not None:
                u = u + st["b2"].float()
            y = y / (1 + torch.exp(-y)) * u
        if st["res"] is not None:
            y = y + st["res"].float()
        return y.to(_TORCH[st["out"]])
    return _plain_controls(st)


def _plain_controls(st):
    rows, v = st["rows"], st["vocab"]
    x = st["logits"][:, 0].float()
    dev = x.device
    if st["g"] is not None:
        gs = st["g"].unsqueeze(1)
        x = torch.where(x == -math.inf, x, gs * x + (1 - gs) * st["logits"][:, 1].float())
    if st["hist"] is not None and st["rho"] is not None:
        at = torch.arange(st["hist"].shape[1], device=dev)
        used = (at < st["hist_len"].unsqueeze(1)).float()
        ids = st["hist"].long()
        n_all = torch.zeros(rows, v, device=dev).scatter_add_(1, ids, used)
        n_out = torch.zeros(rows, v, device=dev).scatter_add_(1, ids, used * (at >= st["prompt_len"].unsqueeze(1)))
        rho = st["rho"].unsqueeze(1)
        x = torch.where(n_all > 0, torch.where(x > 0, x / rho, x * rho), x)
        x = x - (n_out * st["freq"].unsqueeze(1) + (n_out > 0) * st["pres"].unsqueeze(1))
    if st["bias"] is not None:  # an id given twice: the later entry holds; negative ids are no entries
        ids = st["bias_ids"].long()
        order = torch.arange(1, ids.shape[1] + 1, device=dev).expand_as(ids) * (ids >= 0)
        last = torch.zeros(rows, v, dtype=torch.long, device=dev).scatter_reduce_(1, ids.clamp(min=0), order, "amax")
        x = x + torch.where(last > 0, st["bias"].gather(1, (last - 1).clamp(min=0)), torch.zeros_like(x))
    allowed = torch.full((rows,), v, dtype=torch.int32, device=dev)
    if st["masks"] is not None:
        bits = (st["masks"].unsqueeze(-1) >> torch.arange(32, device=dev, dtype=torch.int32)) & 1
        ok = bits.flatten(1)[:, :v].bool()[st["state"].clamp(min=0).long()] | (st["state"] < 0).unsqueeze(1)
        x = torch.where(ok, x, torch.full_like(x, -math.inf))
        allowed = ok.sum(1).int()
    return x.to(_TORCH[st["out"]]), allowed


def _run_own(st):
    native = _native()
    lib, stream = native.lib(), torch.cuda.current_stream().cuda_stream
    if st["op"] == "quantize":
        native.check(lib.mv_op_quantize_mxfp4(stream, *st["args"]))
        return st["deq"]
    if st["op"] == "linear":
        native.check(lib.mv_op_linear_mxfp4(stream, *st["args"]))
        return st["y"]
    if st["op"] == "gemm":
        native.check(lib.mv_op_gemm_mxfp4(stream, *st["args"]))
        return st["y"]
    native.check(lib.mv_op_logit_controls(stream, *st["args"]))
    return st["y"], st["allowed"]


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "quantize":
        n, nb = case["rows"] * case["k"], case["rows"] * ((case["k"] + 31) // 32)
        return dict(bytes=n * _SIZE[case["dtype"]] + nb * 17 + n * 2, flops=3 * n)
    if case["op"] in ("linear", "gemm"):
        m, n, k, mats = case["m"], case["n"], case["k"], 2 if case["gated"] else 1
        nb = (k + 31) // 32
        x = m * k * 2 if case["op"] == "linear" else m * nb * 17
        y = m * n * _SIZE[case["out"]] * (2 if case["residual"] else 1)
        return dict(bytes=x + mats * n * nb * 17 + (mats * n * 2 if case["bias"] else 0) + y, flops=2 * m * n * k * mats)
    rows, v = case["rows"], case["vocab"]
    read = rows * v * _SIZE[case["dtype"]] * (2 if case["guidance"] else 1) + rows * case["n_bias"] * 8 + case["states"] * ((v + 31) // 32) * 4
    if case["penalties"]:
        read += rows * case["history"] * 2  # half of the room on average
    return dict(bytes=read + rows * v * _SIZE[case["out"]] + rows * 4, flops=4 * rows * v)


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------------------
def _exact_matrix(codes, scales, k):
    table = torch.tensor([(1 - 2 * (c >> 3)) * [0, 0.5, 1, 1.5, 2, 3, 4, 6][c & 7] for c in range(16)], dtype=torch.float64, device=codes.device)
    out = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.float64, device=codes.device)
    out[:, 0::2] = table[(codes % 16).long()]
    out[:, 1::2] = table[torch.div(codes, 16, rounding_mode="floor").long()]
    size = torch.tensor([2.0 ** (s - 127) for s in range(255)] + [math.nan], dtype=torch.float64, device=codes.device)
    return (out * size[scales.long()].repeat_interleave(32, dim=1))[:, :k]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "quantize":
        w = st["w"].double()
        rows, k = w.shape
        grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=w.device)
        out = torch.empty_like(w)
        for lo in range(0, rows, 4096):  # the large matrix in slices
            x = torch.zeros(min(4096, rows - lo), -(-k // 32) * 32, dtype=torch.float64, device=w.device)
            x[:, :k] = w[lo:lo + 4096]
            top = x.abs().unflatten(1, (-1, 32)).amax(2).clamp(min=2.0 ** -140)
            mant, ex = torch.frexp(top)
            unit = (((ex - 3).clamp(min=-127).long() + 1023) << 52).view(torch.float64).repeat_interleave(32, dim=1)
            y = (x.abs() / unit).clamp(max=6.0)
            below = torch.bucketize(y, grid, right=True) - 1
            above = (below + 1).clamp(max=7)
            mid = (grid[below] + grid[above]) / 2
            pick = torch.where((y > mid) | ((y == mid) & (below % 2 == 1)), above, below)
            out[lo:lo + 4096] = (torch.sign(x) * grid[pick] * unit)[:, :k]
        return out
    if case["op"] in ("linear", "gemm"):
        x = st["x"].double() if case["op"] == "linear" else _exact_matrix(st["x"], st["xs"], case["k"])
        y = torch.mm(x, _exact_matrix(st["w"], st["ws"], case["k"]).t().contiguous())
        if case["bias"]:
            y += st["b"].double()
        if case["gated"]:
            u = torch.mm(x, _exact_matrix(st["w2"], st["ws2"], case["k"]).t().contiguous())
            if case["bias"]:
                u += st["b2"].double()
            y = y * torch.sigmoid(y) * u
        if case["residual"]:
            y += st["res"].double()
        return y
    rows, v = case["rows"], case["vocab"]
    out = torch.empty(rows, v, dtype=torch.float64, device="cuda")
    allowed = torch.empty(rows, dtype=torch.int32, device="cuda")
    host = {n: t.cpu() if torch.is_tensor(t) else t for n, t in st.items() if n not in ("logits", "y", "allowed", "controls", "args")}
    for r in range(rows):
        x = st["logits"][r, 0].double()
        if case["guidance"]:
            gs = float(host["g"][r])
            x = gs * x + (1 - gs) * st["logits"][r, 1].double()
        if case["history"] and case["penalties"]:
            h = st["hist"][r, : int(host["hist_len"][r])].long()
            seen = torch.bincount(h, minlength=v) > 0
            count = torch.bincount(h[int(host["prompt_len"][r]):], minlength=v).double()
            rho = float(host["rho"][r])
            x[seen & (x <= 0)] *= rho
            x[seen & (x > 0)] /= rho
            x -= count * float(host["freq"][r]) + (count > 0).double() * float(host["pres"][r])
        if case["n_bias"]:
            extra = {i: b for i, b in zip(host["bias_ids"][r].tolist(), host["bias"][r].tolist()) if i >= 0}
            ids = torch.tensor(list(extra), dtype=torch.long, device="cuda")
            x[ids] += torch.tensor(list(extra.values()), dtype=torch.float64, device="cuda")
        allowed[r] = v
        if case["states"] and int(host["state"][r]) >= 0:
            words = host["masks"][int(host["state"][r])].numpy().view("uint8")
            ok = torch.from_numpy(((words[:, None] >> [0, 1, 2, 3, 4, 5, 6, 7]) & 1).reshape(-1)[:v].astype(bool)).cuda()
            x[~ok] = -math.inf
            allowed[r] = int(ok.sum())
        out[r] = x
    return out, allowed
