"""Products of 8-bit integer rows whose scales are so large that a sum (up to 2^31) times its row's scale is no float32 although the result, which has the column's
scale in it too, is one; beside rows of ordinary and of the smallest scales.

A result is the sum's conversion and two factors, three roundings of float32: 3 x 2^-24, and the result's own, 2^-8 for bfloat16.  Moving a power of two from one
scale to the other adds none: the sums here times either scale, however the powers are dealt, are normal numbers or exact."""
import pytest
import torch

from tests.gpu_util import require_gpu
from tests.test_gpu_q8 import PLANS, activation64, integers, near, product64

pytestmark = pytest.mark.gpu


def operands(T, N, K, seed):
    """Integers, and scales whose products are 1e-6 to 1: rows of 1e31 to 2.6e36 (a row's largest value up to 3.3e38), of 1, and columns to suit; a third
    of the columns are for the ordinary rows, whose results with the large rows overflow."""
    g = torch.Generator().manual_seed(seed)
    q, p = (torch.randint(-127, 128, size, generator=g, dtype=torch.int8) for size in ((T, K), (N, K)))
    large = torch.arange(T) % 3 != 1
    sx = torch.where(large, 10.0 ** (31 + 5.4 * torch.rand(T, generator=g)), 10.0 ** (-2 * torch.rand(T, generator=g)))
    small = torch.arange(N) % 3 != 2
    sw = torch.where(small, 10.0 ** (-37 + 2 * torch.rand(N, generator=g)), 10.0 ** (-3 * torch.rand(N, generator=g)))
    if T > 4:
        q[3] = 0                                    # (a sum of zero is zero whatever the scales)
        sx[4] = 1e-42                               # (below the smallest normal number)
    if N > 2:
        sw[2] = 3e38
        sw[1] *= -1
    return q, sx.float(), p, sw.float()


def check(y, want, rel):
    """Numbers near what they should be; infinities where float32 (and so bfloat16) has none."""
    y, want = y.cpu().double(), want.cpu()
    most = float(torch.finfo(torch.float32).max)
    over = want.abs() > most * 1.01
    assert bool((y[over] == torch.sign(want[over]) * float("inf")).all())
    inside = want.abs() < most * 0.99
    assert bool(inside.any()) and bool(torch.isfinite(y[inside]).all())
    near(y[inside], want[inside], rel)


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("plan", [0] + PLANS)
@pytest.mark.parametrize("T,N,K", [(260, 200, 320), (270, 77, 1500)])
def test_product(T, N, K, plan, out, monkeypatch):
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    monkeypatch.setattr(ops, "Q8_PLAN", plan)
    q, sx, p, sw = operands(T, N, K, plan + T)
    x, w = ops.Q8Rows.from_values(q.to(dev), sx.to(dev)), ops.Q8Weight.from_values(p.to(dev), sw.to(dev))
    want, rel = product64(q, sx, p, sw), (2.0 ** -8 if out == torch.bfloat16 else 0.0) + 3.1 * 2.0 ** -24
    check(ops.linear_q8(x, w, out), want, rel)
    # results that begin anywhere
    held = torch.empty((1 + T * N,), dtype=out, device=dev)
    check(ops.linear_q8(x, w, out, out=held[1:].view(T, N)), want, rel)


@pytest.mark.parametrize("plan", [0] + PLANS)
@pytest.mark.parametrize("T,N,K", [(260, 200, 320), (270, 77, 300)])
def test_rows_of_all_scales_side_by_side(T, N, K, plan, monkeypatch):
    """Scales from the smallest numbers to the largest, columns so that float32 holds every result that is not zero as a normal number."""
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    monkeypatch.setattr(ops, "Q8_PLAN", plan)
    g = torch.Generator().manual_seed(plan + T)
    q, p = (torch.randint(-127, 128, size, generator=g, dtype=torch.int8) for size in ((T, K), (N, K)))
    sx = (10.0 ** (-44 + 81 * torch.rand(T, generator=g, dtype=torch.float64))).float()
    order = torch.arange(N) % 2 == 0
    for sw in (torch.where(order, 1e9, 3e8), torch.where(order, 1e-7, 2e-8)):
        x, w = ops.Q8Rows.from_values(q.to(dev), sx.to(dev)), ops.Q8Weight.from_values(p.to(dev), sw.to(dev))
        want, y = product64(q, sx, p, sw).cpu(), ops.linear_q8(x, w, torch.float32).cpu().double()
        held = (want == 0) | ((want.abs() > 2.0 ** -126) & (want.abs() < 3.3e38))
        assert float(held.double().mean()) > 0.5
        assert bool(((y - want).abs() <= want.abs() * (3.1 * 2.0 ** -24))[held].all())


@pytest.mark.parametrize("plan", [0] + [p for p in PLANS if p // 100 % 2 == 0])
@pytest.mark.parametrize("T,I,K", [(260, 200, 320), (270, 77, 1500)])
def test_gated(T, I, K, plan, monkeypatch):
    """Gate and up columns for the large rows alone (products with the others are nearly nothing)."""
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    monkeypatch.setattr(ops, "Q8_PLAN", plan)
    q, sx, p, _ = operands(T, 2 * I, K, plan + T)
    sx[torch.arange(T) % 3 != 1] = 1e33
    sw = 1e-39 * (1 + torch.arange(2 * I) % 5).float()          # (sums below 2^24: |z| below 30)
    x, w = ops.Q8Rows.from_values(q.to(dev), sx.to(dev)), ops.Q8Weight.from_values(p.to(dev), sw.to(dev), gated=True)
    z = product64(q, sx, p, sw)
    assert float(z.abs().max()) < 30 and float(z.abs().max()) > 1
    near(ops.linear_q8_gated(x, w), activation64(z[:, :I], "silu") * z[:, I:], 2.0 ** -8 + 2.0 ** -13)


@pytest.mark.parametrize("T", [1, 40, 600])
def test_from_floats(T):
    """Rows of float32 near its largest numbers and a matrix of tiny ones, brought to 8 bits and multiplied."""
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    g = torch.Generator().manual_seed(T)
    x, w = torch.randn((T, 512), generator=g) * 5e37, torch.randn((96, 512), generator=g) * 1e-34
    y = ops.linear_q8(ops.quantize_rows(x.to(dev)), ops.quantize_weight(w.to(dev)), torch.float32)
    (q, a), (p, b) = integers(x.double()), integers(w.double())
    near(y, product64(q, a / 127, p, b / 127), 5.1 * 2.0 ** -24)          # (and the two scales' roundings)
