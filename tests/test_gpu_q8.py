"""Rows in 8-bit integers and their products (csrc/rows_q8.hip, csrc/gemm_q8.hip) against their definitions in 64 bits: one row and
many, odd widths, rows of a wider tensor, rows of zeros, NaN, infinities, the smallest and the largest numbers, every dtype;
whole feed-forwards, recorded and replayed.

Tolerances.  Integers are equal.  A scale is formed in 64 bits and rounded once: 2^-24 of it.  A product's sum is exact, its conversion and
two factors are three roundings of float32, 3 x 2^-24, beside the result's own, 2^-8 for bfloat16.  A gated result: an error of 4 x 2^-24 in the gate's value z
moves act(z) by at most that times |z act'(z) / act(z)| <= 1 + |z| (silu; 1 + |z| (1.6 + 0.22 z^2) for the tanh form) and the activation itself is off by up to
100 units of 2^-24: below 2^-13 in all for |z| <= 30 (silu) and 8 (the tanh form), where the inputs are held."""
import math

import pytest
import torch

from tests.gpu_util import require_gpu

pytestmark = pytest.mark.gpu

EPS = 1e-6
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def integers(z):
    """(q, a) of rows of float64: 127 z / a rounded half to even."""
    a = z.abs().amax(dim=1)
    return torch.round(z * 127.0 / torch.where(a > 0, a, 1.0)[:, None]).to(torch.int8), a


def scales_near(got, want):
    got, want = got.cpu().double(), want.double()
    assert bool(((got - want).abs() <= want * (2.0 ** -24 * 1.0001) + 1e-45).all())


def near(got, want, rel):
    got, want = got.cpu().double(), want.cpu().double()
    err, lim = (got - want).abs(), want.abs() * rel + 1e-37
    assert bool((err <= lim).all()), (float((err - lim).max()), int((err > lim).sum()), got.numel())


def uneven(shape, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(2.0 * torch.randn((shape[0], 1), generator=g))
    x[:, torch.rand(shape[1], generator=g) < 0.03] *= 20.0
    return x.to(dtype)


SIZES = [(1, 1), (3, 2), (1, 4096), (2, 17), (5, 64), (7, 1001), (61, 250), (9, 1024), (4, 5120), (3, 12288), (2, 20480), (130, 96), (9, 1084), (3, 2830), (700, 1548), (600, 3001), (520, 2050), (2, 6226), (4, 16796), (3, 16398), (600, 5120), (530, 12288), (2, 24576), (1, 32768), (257, 4096), (1025, 128), (300, 2560), (2, 130816)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K", SIZES)
def test_rows(T, K, dtype):
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    x = uneven((T, K), T + K, dtype)
    got = ops.quantize_rows(x.to(dev))
    q, a = integers(x.double())
    assert torch.equal(got.values[:, :K].cpu(), q) and got.shape == (T, K) and got.values.shape[1] == -(-K // 256) * 256
    scales_near(got.scales, a / 127.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K,ld,at", [(5, 64, 192, 64), (3, 100, 333, 7), (1, 96, 400, 16), (40, 2048, 4096, 2048), (6, 1, 5, 3), (17, 4096, 4104, 8)])
def test_rows_of_a_wider_tensor(T, K, ld, at, dtype):
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    wide = uneven((T, ld), T * ld, dtype)
    got = ops.quantize_rows(wide.to(dev)[:, at:at + K])
    q, a = integers(wide[:, at:at + K].double())
    assert torch.equal(got.values[:, :K].cpu(), q)
    scales_near(got.scales, a / 127.0)


@pytest.mark.parametrize("K", [16, 129, 4096])
def test_rows_at_the_border_of_two_integers(K):
    """Multiples of a / 254: quotients that end in a half, which go to the even one."""
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    g = torch.Generator().manual_seed(K)
    for a, dtype in ((127.0, torch.float32), (128.0, torch.bfloat16), (127.0, torch.bfloat16), (1.9375, torch.bfloat16), (3.0e38, torch.float32), (2.0 ** -120, torch.float32)):
        x = torch.randint(-254, 255, (7, K), generator=g).double() * (a / 254.0)
        x[:, 0] = a
        x = x.to(dtype)
        got = ops.quantize_rows(x.to(dev))
        q, top = integers(x.double())
        assert torch.equal(got.values[:, :K].cpu(), q)
        scales_near(got.scales, top / 127.0)


def test_rows_of_zeros_of_nan_and_of_infinities():
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    for dtype in (torch.float32, torch.bfloat16):
        for K in (48, 1000, 8192):
            x = uneven((8, K), K, dtype)
            x[1] = 0.0
            x[2, K - 1] = float("nan")
            x[3, 0] = float("inf")
            x[4, K // 2] = float("-inf")
            x[5] = -0.0
            x[6, 3], x[6, 4] = float("nan"), float("inf")
            got = ops.quantize_rows(x.to(dev))
            q, s = got.values[:, :K].cpu(), got.scales.cpu()
            assert torch.equal(q[[0, 7]], integers(x[[0, 7]].double())[0]) and not q[1:7].any()
            assert torch.equal(s[[1, 5]], torch.zeros(2)) and bool(torch.isnan(s[[2, 3, 4, 6]]).all()) and bool((s[[0, 7]] > 0).all())
            w = ops.quantize_weight(uneven((24, K), 1).to(dev))
            y = ops.linear_q8(got, w, torch.float32).cpu()
            assert bool(torch.isnan(y[[2, 3, 4, 6]]).all()) and not y[[1, 5]].any() and bool(torch.isfinite(y[[0, 7]]).all())


def test_smallest_and_largest_numbers():
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    x = torch.tensor([[1e-45, -1e-45, 0.0, 7e-45], [1e-38, 2e-38, -3e-38, 1e-39], [3.4e38, -3.4e38, 1.0, 2e38], [1e-30, 3e30, 1e10, -1e30]])
    got = ops.quantize_rows(x.to(dev))
    q, a = integers(x.double())
    assert torch.equal(got.values[:, :4].cpu(), q)
    # (scales below the smallest normal number are rounded to a multiple of 2^-149)
    assert bool(((got.scales.cpu().double() - a / 127.0).abs() <= a / 127.0 * 2.0 ** -24 * 1.0001 + 2.0 ** -150).all())


@pytest.mark.parametrize("addend", [None, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("weight", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,H", SIZES[:-1])
def test_norm(T, H, addend, weight):
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    s, w = uneven((T, H), T + H), (1.0 + 0.3 * torch.randn(H, generator=torch.Generator().manual_seed(H))).to(weight)
    d = None if addend is None else uneven((T, H), T - H, addend)
    stream = s.to(dev)
    got = ops.add_rms_norm_q8(stream, None if d is None else d.to(dev), w.to(dev), EPS)
    want = s if d is None else s + d.float()
    assert torch.equal(stream.cpu(), want)
    z = want.double() * w.double()
    q, a = integers(z)
    assert torch.equal(got.values[:, :H].cpu(), q)
    eps = float(torch.tensor(EPS))
    scales_near(got.scales, a / 127.0 / torch.sqrt((want.double() ** 2).mean(dim=1) + eps))


def test_norm_of_zeros_of_nan_and_of_large_numbers():
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    for H in (50, 4096):
        s = uneven((6, H), H)
        s[0], s[1, 5], s[2, 0] = 0.0, float("nan"), float("inf")
        s[3] *= 1e30          # (squares beyond float32)
        w = torch.ones(H)
        got = ops.add_rms_norm_q8(s.to(dev), None, w.to(dev), EPS)
        assert not got.values[:3, :H].any() and got.scales[0] == 0 and bool(torch.isnan(got.scales[1:3]).all())
        q, a = integers(s[3:].double())
        assert torch.equal(got.values[3:, :H].cpu(), q)
        scales_near(got.scales[3:], a / 127.0 / torch.sqrt((s[3:].double() ** 2).mean(dim=1) + float(torch.tensor(EPS))))
        # a weight that is no number spoils every row, as in the norm itself
        w[7] = float("inf")
        assert bool(torch.isnan(ops.add_rms_norm_q8(s[4:].to(dev), None, w.to(dev), EPS).scales).all())


PRODUCTS = [(1, 16, 64), (1, 1, 1), (1, 4096, 4096), (2, 33, 300), (3, 6144, 4096), (8, 4096, 12288), (16, 777, 1023), (17, 256, 512), (31, 1000, 4096), (33, 1040, 2560), (45, 777, 1023), (48, 96, 17408), (49, 4096, 1024),
            (64, 6144, 4096), (65, 16, 256), (65, 1040, 128), (100, 500, 5000), (128, 2048, 2048), (129, 272, 640), (200, 6144, 4096), (255, 257, 259), (256, 256, 256), (300, 2560, 9728), (513, 1024, 768), (700, 5120, 1280), (1100, 1536, 512),
            (2047, 520, 400), (2100, 4096, 4096)]


def drawn(T, N, K, seed):
    """Integers of every size up to the largest, -128 among the given ones, and scales of several sizes."""
    g = torch.Generator().manual_seed(seed)
    q, p = (torch.randint(-128, 128, size, generator=g, dtype=torch.int8) for size in ((T, K), (N, K)))
    if T > 1:
        q[T - 1] = -128
    p[N - 1] = -128
    return q, torch.exp(torch.randn(T, generator=g)) / 500, p, torch.exp(torch.randn(N, generator=g)) / 500 / math.sqrt(K)


def product64(q, sx, p, sw):
    dev = torch.device("cuda:0")
    return (q.to(dev).double() @ p.to(dev).double().T.contiguous()) * (sx.to(dev).double()[:, None] * sw.to(dev).double())


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,N,K", PRODUCTS)
def test_product(T, N, K, out):
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    q, sx, p, sw = drawn(T, N, K, T + N + K)
    x, w = ops.Q8Rows.from_values(q.to(dev), sx.to(dev)), ops.Q8Weight.from_values(p.to(dev), sw.to(dev))
    want = product64(q, sx, p, sw)
    rel = (HALF[out] if out != torch.float32 else 0.0) + 3.1 * 2.0 ** -24
    y = ops.linear_q8(x, w, out)
    assert y.dtype == out and tuple(y.shape) == (T, N)
    near(y, want, rel)
    # into a tensor of the caller's; rows and columns beside it stay as they are
    held = torch.full((T + 2, N), 7.0, dtype=out, device=dev)
    assert ops.linear_q8(x, w, out, out=held[1:T + 1]).data_ptr() == held[1].data_ptr()
    assert torch.equal(held[1:T + 1], y) and bool((held[0] == 7).all()) and bool((held[T + 1] == 7).all())


@pytest.mark.parametrize("T,N,K", [(3, 48, 130816), (80, 32, 130816)])
def test_longest_sums(T, N, K):
    """Every product 2^14, the most terms: a sum just below 2^31."""
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    q, p = torch.full((T, K), -128, dtype=torch.int8, device=dev), torch.full((N, K), -128, dtype=torch.int8, device=dev)
    y = ops.linear_q8(ops.Q8Rows.from_values(q, torch.ones(T, device=dev)), ops.Q8Weight.from_values(p, torch.ones(N, device=dev)), torch.float32)
    near(y, torch.full((T, N), 16384.0 * K, dtype=torch.float64), 2.0 ** -24)


def activation64(z, name):
    if name == "silu":
        return z * torch.sigmoid(z)
    return z * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3))


@pytest.mark.parametrize("name", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("T,I,K", [(T, N, K) for T, N, K in PRODUCTS if T * N * K < 1 << 33])
def test_gated(T, I, K, name):
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    q, sx, p, sw = drawn(T, 2 * I, K, T + I + K)
    x, w = ops.Q8Rows.from_values(q.to(dev), sx.to(dev)), ops.Q8Weight.from_values(p.to(dev), sw.to(dev), gated=True)
    most = 30.0 if name == "silu" else 8.0
    z = product64(q, sx, p, sw)
    big = float(z.abs().max())
    if big > most:         # (scales that hold the gate's values where the tolerance is derived)
        sx = sx * (most / big)
        x, z = ops.Q8Rows.from_values(q.to(dev), sx.to(dev)), product64(q, sx, p, sw)
    y = ops.linear_q8_gated(x, w, name)
    assert y.dtype == torch.bfloat16 and tuple(y.shape) == (T, I)
    near(y, activation64(z[:, :I], name) * z[:, I:], 2.0 ** -8 + 2.0 ** -13)


def test_no_rows():
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    w = ops.quantize_weight(torch.randn(32, 40, device=dev))
    r = ops.quantize_rows(torch.empty((0, 40), device=dev))
    n = ops.add_rms_norm_q8(torch.empty((0, 40), device=dev), None, torch.ones(40, device=dev), EPS)
    assert r.shape == n.shape == (0, 40) and tuple(ops.linear_q8(r, w).shape) == (0, 32)
    assert tuple(ops.linear_q8_gated(r, ops.quantize_weight(torch.randn(32, 40, device=dev), gated=True)).shape) == (0, 16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,K,gated", [(33, 100, False), (64, 512, True), (6, 1, False)])
def test_matrix(N, K, gated, dtype):
    """A matrix brought to 8 bits is within half an integer of what it was."""
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    m = uneven((N, K), N * K, dtype)
    w = ops.quantize_weight(m.to(dev), gated)
    q, a = integers(m.double())
    near(w.to_rows(), q.double() * (a / 127.0)[:, None], 2.0 ** -23)        # (the scale's rounding and the value's)
    # half an integer is a / 254; the scale is rounded, and its product with an integer of up to 127: two of 2^-24 a, which is 2^-15 of a / 254
    assert bool(((w.to_rows().cpu().double() - m.double()).abs() <= (a / 254.0 * (1 + 2.0 ** -15))[:, None]).all())


def feed_forward(ops, stream, delta, weight, gate_up, down):
    rows = ops.add_rms_norm_q8(stream, delta, weight, EPS)
    act = ops.linear_q8_gated(rows, gate_up)
    inner = ops.quantize_rows(act)
    return rows, act, inner, ops.linear_q8(inner, down)


@pytest.mark.parametrize("T", [1, 7, 40, 90, 400])
def test_a_feed_forward(T):
    """The four operators as a layer runs them: every step against its definition on what the step before left, and the whole against
    the same feed-forward of the matrices' values in 64 bits.  There each of two roundings to 8 bits is off by up to half a step of a row's
    largest value, evenly spread: a / 127 / sqrt(12) of a row against its root mean square, a few of which a row's largest value is."""
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    H, I = 256, 688
    g = torch.Generator().manual_seed(T)
    s, d, w = torch.randn((T, H), generator=g), torch.randn((T, H), generator=g).bfloat16(), (1 + 0.1 * torch.randn(H, generator=g)).bfloat16()
    gate_up = ops.quantize_weight((torch.randn((2 * I, H), generator=g) / 16).to(dev), gated=True)
    down = ops.quantize_weight((torch.randn((H, I), generator=g) / math.sqrt(I)).to(dev))
    stream = s.to(dev)
    rows, act, inner, y = feed_forward(ops, stream, d.to(dev), w.to(dev), gate_up, down)
    x64 = s + d.float()
    assert torch.equal(stream.cpu(), x64)
    assert torch.equal(rows.values.cpu(), integers(x64.double() * w.double())[0])
    matrices = [m.to_rows(torch.float64) for m in (gate_up, down)]        # (exact: an integer times a float32)
    def product(x, m):                                                      # (of the integers, so that a sum that is zero is zero)
        p = ops.Q8Weight(m.tiles, torch.ones_like(m.scales), m.shape, m.gated).to_rows(torch.float64)
        sw = (m.to_rows(torch.float64).abs().amax(dim=1) / p.abs().amax(dim=1))
        return product64(x.values[:, :x.width], x.scales, p, sw)
    z = product(rows, gate_up)
    near(act, activation64(z[:, :I], "silu") * z[:, I:], 2.0 ** -8 + 2.0 ** -13)
    q, a = integers(act.cpu().double())
    assert torch.equal(inner.values[:, :I].cpu(), q)
    near(y, product(inner, down), 2.0 ** -8 + 2.0 ** -20)
    normed = x64.double() / torch.sqrt((x64.double() ** 2).mean(dim=1, keepdim=True) + EPS) * w.double()
    z = normed @ matrices[0].cpu().T
    full = (activation64(z[:, :I], "silu") * z[:, I:]) @ matrices[1].cpu().T
    off = float((y.cpu().double() - full).norm() / full.norm())
    # largest values: up to 4.5 root mean squares of the normed row, up to 12 of the activation's; both enter gate and up
    assert off < (2 * 4.5 + 12.0) / 127.0 / math.sqrt(12.0) + 2.0 ** -8, off


@pytest.mark.parametrize("T", [1, 12, 70, 300])
def test_recorded_and_replayed(T):
    """A feed-forward in a HIP graph, replayed with new contents of its inputs and work of its own between the replays: what a call leaves each time."""
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    H, I = 512, 1100
    g = torch.Generator().manual_seed(T)
    w = torch.ones(H, device=dev)
    gate_up, down = ops.quantize_weight(torch.randn((2 * I, H), generator=g).to(dev) / 20, gated=True), ops.quantize_weight(torch.randn((H, I), generator=g).to(dev) / 30)
    stream, delta = torch.zeros((T, H), device=dev), torch.zeros((T, H), dtype=torch.bfloat16, device=dev)
    graphs = []
    side = torch.cuda.Stream()
    for _ in range(2):                      # (two graphs of the same operators, replayed in turn)
        with torch.cuda.stream(side):
            feed_forward(ops, stream, delta, w, gate_up, down)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = feed_forward(ops, stream, delta, w, gate_up, down)
        graphs.append((graph, out))
    for k in range(6):
        s, d = torch.randn((T, H), generator=g).to(dev), torch.randn((T, H), generator=g).bfloat16().to(dev)
        stream.copy_(s)
        delta.copy_(d)
        graph, (rows, act, inner, y) = graphs[k % 2]
        graph.replay()
        eager = s.clone()
        e_rows, e_act, e_inner, e_y = feed_forward(ops, eager, d, w, gate_up, down)
        torch.cuda.synchronize()
        assert torch.equal(stream, eager) and torch.equal(rows.values, e_rows.values) and torch.equal(rows.scales, e_rows.scales)
        assert torch.equal(act, e_act) and torch.equal(inner.values[:, :I], e_inner.values[:, :I]) and torch.equal(y, e_y)


def test_two_streams_at_once():
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    g = torch.Generator().manual_seed(3)
    w = ops.quantize_weight(torch.randn((4096, 2048), generator=g).to(dev))
    few, many = (ops.quantize_rows(torch.randn((T, 2048), generator=g).to(dev)) for T in (5, 200))
    want = [ops.linear_q8(x, w, torch.float32) for x in (few, many)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for k in range(40):
        with torch.cuda.stream(streams[k % 4]):
            got.append(ops.linear_q8((few, many)[k % 2], w, torch.float32))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[k % 2]) for k, y in enumerate(got))


def test_a_result_tensor_of_another_kind_is_turned_away():
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    x, w = ops.quantize_rows(torch.randn((4, 64), device=dev)), ops.quantize_weight(torch.randn((32, 64), device=dev))
    for bad in (torch.empty((4, 31), dtype=torch.bfloat16, device=dev), torch.empty((4, 32), device=dev), torch.empty((32, 4), dtype=torch.bfloat16, device=dev).t(), torch.empty((4, 32), dtype=torch.bfloat16)):
        with pytest.raises(ops.KernelError):
            ops.linear_q8(x, w, out=bad)
    with pytest.raises(ops.KernelError):
        ops.quantize_rows(torch.randn((8, 8), device=dev).t())
    with pytest.raises(ops.KernelError):
        ops.add_rms_norm_q8(torch.randn((8, 8), device=dev), torch.randn((8, 8), device=dev).half(), torch.ones(8, device=dev), EPS)
    with pytest.raises(ops.KernelError):
        ops.add_rms_norm_q8(torch.randn((8, 8), device=dev).t(), None, torch.ones(8, device=dev), EPS)


#: kinds of blocks of a product (csrc/gemm_q8.hip), and row tiles of each
PLANS = [101, 201, 202, 203, 204, 304, 306, 308, 404, 405, 406, 407, 408, 1202, 1404, 8, 10, 12, 14, 16]


@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("T,N,K", [(1, 40, 64), (16, 16, 1), (47, 100, 300), (64, 272, 2300), (130, 70, 1024), (259, 513, 777), (513, 33, 4200), (2100, 550, 200)])
def test_every_kind_of_block(plan, T, N, K, monkeypatch):
    """Fewer rows, columns and chunks of K than a block has, and more of each, with more row blocks than a band; plain and gated, both result types."""
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    monkeypatch.setattr(ops, "Q8_PLAN", plan)
    q, sx, p, sw = drawn(T, 2 * N, K, plan + T)
    sx = sx / 10
    x = ops.Q8Rows.from_values(q.to(dev), sx.to(dev))
    want = product64(q, sx, p, sw)
    w = ops.Q8Weight.from_values(p.to(dev), sw.to(dev))
    if plan <= 16 and T < 16 * plan:              # (tall blocks are for rows that fill one)
        with pytest.raises(ops.KernelError, match="row tiles"):
            ops.linear_q8(x, w)
        return
    for out in (torch.bfloat16, torch.float32):
        near(ops.linear_q8(x, w, out), want, (HALF[out] if out != torch.float32 else 0.0) + 3.1 * 2.0 ** -24)
    narrow = ops.Q8Weight.from_values(p[:N].to(dev), sw[:N].to(dev))
    near(ops.linear_q8(x, narrow, torch.float32), want[:, :N], 3.1 * 2.0 ** -24)
    gated = ops.Q8Weight.from_values(p.to(dev), sw.to(dev), gated=True)
    if plan // 100 % 2:
        with pytest.raises(ops.KernelError, match="gated"):
            ops.linear_q8_gated(x, gated)
        return
    assert float(want.abs().max()) < 30
    near(ops.linear_q8_gated(x, gated), activation64(want[:, :N], "silu") * want[:, N:], 2.0 ** -8 + 2.0 ** -13)


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("plan", PLANS)
def test_results_that_begin_anywhere(plan, out, monkeypatch):
    """A caller's tensor that begins at an odd place, at every second and at every fourth value; what lies around it stays."""
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    monkeypatch.setattr(ops, "Q8_PLAN", plan)
    T, N, K = 260, 200, 320
    q, sx, p, sw = drawn(T, N, K, plan)
    x, w = ops.Q8Rows.from_values(q.to(dev), sx.to(dev)), ops.Q8Weight.from_values(p.to(dev), sw.to(dev))
    y = ops.linear_q8(x, w, out)
    near(y, product64(q, sx, p, sw), (HALF[out] if out != torch.float32 else 0.0) + 3.1 * 2.0 ** -24)
    for at in (1, 2, 4, 7):
        held = torch.full((at + T * N + 9,), 7.0, dtype=out, device=dev)
        ops.linear_q8(x, w, out, out=held[at:at + T * N].view(T, N))
        assert torch.equal(held[at:at + T * N].view(T, N), y) and bool((held[:at] == 7).all()) and bool((held[at + T * N:] == 7).all())


def test_blocks_that_do_not_exist_are_turned_away(monkeypatch):
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    x, w = ops.quantize_rows(torch.randn((4, 64), device=dev)), ops.quantize_weight(torch.randn((32, 64), device=dev))
    for plan in (1, 9, 17, 100, 105, 303, 409, -1):
        monkeypatch.setattr(ops, "Q8_PLAN", plan)
        with pytest.raises(ops.KernelError, match="no blocks|row tiles"):
            ops.linear_q8(x, w)


def test_rows_and_results_beyond_32_bits():
    """More than 2^31 bytes of rows, and more than 2^31 results: the last rows and columns are those of the rows alone."""
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    g = torch.Generator(device=dev).manual_seed(9)
    T, K = 140_000, 17_408
    q = torch.randint(-128, 128, (T, K), device=dev, generator=g, dtype=torch.int8)
    x = ops.Q8Rows(q, torch.rand(T, device=dev, generator=g), K)
    w = ops.Q8Weight.from_values(torch.randint(-128, 128, (24, K), device=dev, generator=g, dtype=torch.int8), torch.rand(24, device=dev, generator=g))
    y = ops.linear_q8(x, w, torch.float32)
    for at in (0, 123_361, 123_370, T - 70):
        assert torch.equal(y[at:at + 70], ops.linear_q8(ops.Q8Rows(q[at:at + 70], x.scales[at:at + 70].clone(), K), w, torch.float32))
    del x, q, y, w
    T, N = 270_001, 8200
    q = torch.randint(-128, 128, (T, 256), device=dev, generator=g, dtype=torch.int8)
    x = ops.Q8Rows(q, torch.rand(T, device=dev, generator=g), 256)
    w = ops.Q8Weight.from_values(torch.randint(-128, 128, (N, 256), device=dev, generator=g, dtype=torch.int8), torch.rand(N, device=dev, generator=g))
    y = ops.linear_q8(x, w)
    for at in (0, 261_890, T - 70):
        assert torch.equal(y[at:at + 70], ops.linear_q8(ops.Q8Rows(q[at:at + 70], x.scales[at:at + 70].clone(), 256), w))
    del y
    T, K = 530_000, 4096
    s = torch.empty((T, K), device=dev)
    s[:100].normal_(generator=g)
    s[100:-100] = 0
    s[-100:].normal_(generator=g)
    weight = torch.ones(K, device=dev)
    last = ops.quantize_rows(s[-100:].clone())
    rows = ops.quantize_rows(s)
    assert torch.equal(rows.values[-100:], last.values) and torch.equal(rows.scales[-100:], last.scales) and not rows.values[100:-100].any()
    last = ops.add_rms_norm_q8(s[-100:].clone(), s[-100:].clone(), weight, EPS)
    rows = ops.add_rms_norm_q8(s, s.clone(), weight, EPS)
    assert torch.equal(rows.values[-100:], last.values) and torch.equal(rows.scales[-100:], last.scales)
