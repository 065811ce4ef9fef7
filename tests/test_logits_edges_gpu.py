"""mv_op_logit_controls on the GPU where a guidance mix leaves the range of fp32 on its way or meets infinities: against oracle/logits.py (64 bits),
with the tolerance of test_logits_gpu.py."""
import pytest
import torch

from test_logits_gpu import BF, CODE, F, N, check, hip, ptr, stream, struct

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def pairs(dt):
    """Every conditioned value beside every unconditioned one."""
    low = torch.finfo(dt).min
    values = torch.tensor([0.0, -0.0, 1.5, -7.25, 3.0e4, low, -low, low / 2, -low / 4, INF, -INF, NAN], dtype=torch.float64).to(dt)
    n = len(values)
    return values.repeat_interleave(n), values.repeat(n)


@pytest.mark.parametrize("dt,ot", [(BF, BF), (BF, F), (F, BF), (F, F)])
def test_guidance_of_every_pair(dt, ot):
    """The type's lowest value in both rows (how many programs mask) stays that value under every guidance; an infinite logit stays; guidance 1 is the
    conditioned row whatever lies beside it; a token that the unconditioned row alone excludes is not pushed to +inf."""
    x, u = pairs(dt)
    scale = torch.tensor([0.0, 0.5, 0.999, 1.0, 1.001, 1.5, 3.0, 100.0])
    rows = len(scale)
    check(x.repeat(rows, 1).cuda(), u.repeat(rows, 1).cuda(), dict(guidance=scale.cuda()), ot)


@pytest.mark.parametrize("dt", [BF, F])
def test_guidance_of_rows_masked_by_the_lowest_value(dt):
    low = torch.finfo(dt).min
    g = torch.Generator().manual_seed(1)
    x, u = (torch.randn(4, 300, generator=g).to(dt) for _ in range(2))
    x[:, ::3], u[:, ::3] = low, low
    x[3], u[3] = low, low  # nothing left in this row
    scale = torch.tensor([1.0, 1.5, 3.0, 2.0]).cuda()
    out, _ = hip(x.cuda(), u.cuda(), dict(guidance=scale), F)
    assert bool((out[:, ::3] == low).all()) and bool((out[3] == low).all())
    assert bool(torch.isfinite(out).all())


def test_guidance_one_is_the_conditioned_row():
    x, u = pairs(F)
    out, _ = hip(x[None].cuda(), u[None].cuda(), dict(guidance=torch.tensor([1.0]).cuda()), F)
    nan = torch.isnan(x)
    assert torch.equal(out[0].cpu()[~nan], x[~nan]) and bool(torch.isnan(out[0].cpu()[nan]).all())


def test_tokens_that_one_row_excludes():
    x = torch.tensor([[2.0, -INF, 2.0, -INF]] * 3)
    u = torch.tensor([[1.0, 1.0, -INF, -INF]] * 3)
    out, _ = hip(x.cuda(), u.cuda(), dict(guidance=torch.tensor([0.5, 1.0, 3.0]).cuda()), F)
    assert out.tolist() == [[1.5, -INF, -INF, -INF], [2.0, -INF, 2.0, -INF], [4.0, -INF, 2.0, -INF]]


@pytest.mark.parametrize("dt", [BF, F])
def test_outputs_beside_their_inputs(dt):
    """Rows of outputs may lie between rows of inputs, and on top of either row of a pair."""
    g = torch.Generator().manual_seed(4)
    rows, v = 5, 333
    data = torch.randn(rows, 4, v, generator=g).to(dt)
    d = dict(guidance=torch.full((rows,), 1.5).cuda())
    want = hip(data[:, 0].contiguous().cuda(), data[:, 1].contiguous().cuda(), d, dt)[0]
    for place in range(4):
        room = data.cuda()
        c = struct(d)
        N.check(N.lib().mv_op_logit_controls(stream(), rows, v, CODE[dt], ptr(room), ptr(room[:, 1]), 4 * v, c, CODE[dt], ptr(room[:, place]), 4 * v, None))
        torch.cuda.synchronize()
        assert torch.equal(room[:, place], want)
        rest = [i for i in range(4) if i != place]
        assert torch.equal(room[:, rest].cpu(), data[:, rest])
