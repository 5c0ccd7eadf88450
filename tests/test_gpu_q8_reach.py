"""Gated products in 8-bit integers on rows that are no numbers and on gates far out; matrices in 8 bits where a model has them in other places than a plain
block: a mixture's shared expert, attention beside another mixer.

Tolerance of the gated products: an error of 4 x 2^-24 in the gate's value z moves act(z) by at most that times |z act'(z) / act(z)| <= 1 + |z| (silu;
1 + |z| (1.6 + 0.22 z^2) for the tanh form; both below 3 for z > 0, where act'(z) nears 1), the activation is off by up to 100 units of 2^-24, the up value by 4, and the result is rounded to bfloat16, 2^-8.  What
exp(-s) below 2^-126 makes of an activation, up to 128 x 2^-126 (and nothing past 2^-128), may be lost whole: 2^-118 of the up value.
Models: as in test_gpu_q8_engine.py, 1.1 % of the layers' part of the logits a product, held to 10 %; every token takes all experts, so that none is chosen otherwise."""
import copy

import pytest
import torch

from tests import meronex_cases, nolatar_cases, tarunex_cases
from tests.gpu_util import require_gpu
from tests.test_gpu_q8 import PLANS, activation64, product64, uneven
from tests.test_gpu_q8_engine import logits, runner_of

pytestmark = pytest.mark.gpu

GATED_PLANS = [p for p in PLANS if p // 100 % 2 == 0]


@pytest.mark.parametrize("plan", [0] + GATED_PLANS)
@pytest.mark.parametrize("I", [64, 75])
def test_gated_rows_that_are_no_numbers(I, plan, monkeypatch):
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    T, K = 260, 300
    x = uneven((T, K), T)
    bad = torch.arange(T) % 7 == 2
    x[bad, 5] = float("nan")
    x[torch.arange(T) % 7 == 5, K - 1] = float("inf")
    bad |= torch.arange(T) % 7 == 5
    x[11] = 0.0
    bad[11] = False
    rows, w = ops.quantize_rows(x.to(dev)), ops.quantize_weight(uneven((2 * I, K), 1).to(dev) / 100, gated=True)
    monkeypatch.setattr(ops, "Q8_PLAN", plan)
    for name in ("silu", "gelu_tanh"):
        y = ops.linear_q8_gated(rows, w, name).cpu()
        assert bool(torch.isnan(y[bad]).all()) and bool(torch.isfinite(y[~bad]).all()) and not y[11].any()


@pytest.mark.parametrize("name,most", [("silu", 85.0), ("silu", 400.0), ("gelu_tanh", 30.0), ("gelu_tanh", 400.0)])
@pytest.mark.parametrize("T,I,K,plan", [(1, 50, 300, 0), (40, 256, 1024, 0), (300, 130, 700, 0), (600, 128, 512, 0), (260, 75, 300, 408), (260, 75, 300, 16)])
def test_gates_far_out(T, I, K, plan, name, most, monkeypatch):
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    monkeypatch.setattr(ops, "Q8_PLAN", plan)
    g = torch.Generator().manual_seed(T + K)
    q, p = torch.randint(-128, 128, (T, K), generator=g, dtype=torch.int8), torch.randint(-128, 128, (2 * I, K), generator=g, dtype=torch.int8)
    sx, sw = torch.ones(T), torch.exp(torch.randn(2 * I, generator=g))
    sw[:I] *= most / float(product64(q, sx, p, sw)[:, :I].abs().max())
    sw[I:] /= float(product64(q, sx, p, sw)[:, I:].abs().max())
    x, w = ops.Q8Rows.from_values(q.to(dev), sx.to(dev)), ops.Q8Weight.from_values(p.to(dev), sw.to(dev), gated=True)
    y = ops.linear_q8_gated(x, w, name).cpu().double()
    z = product64(q, sx, p, sw).cpu()
    up, z = z[:, I:], z[:, :I]
    want, size = activation64(z, name) * up, z.abs()
    moved = torch.where(z > 0, 2.0, size if name == "silu" else size * (1.6 + 0.22 * size ** 2))
    rel = 2.0 ** -8 + (4 * (1 + moved) + 104) * 2.0 ** -24
    # (where that passes one, the activation lies below what may be lost)
    err, lim = (y - want).abs(), want.abs() * rel.clamp(max=1.0) + up.abs() * 2.0 ** -118
    assert bool((err <= lim).all()), (float((err - lim).max()), int((err > lim).sum()))
    assert float(size.max()) > 0.9 * most


def whole_model(write, config, tmp_path, seed, vocab):
    """(model with matrices in 8 bits, worst of some schedules' distance between its logits and those of the stored matrices, over their spread)."""
    folder = write(str(tmp_path / "m"), copy.deepcopy(config), seed)
    g = torch.Generator().manual_seed(seed)
    requests = [torch.randint(0, vocab, (n,), generator=g).tolist() for n in (3, 80, 21)]
    q8 = runner_of(folder, "int8")
    want = torch.cat(logits(runner_of(folder, "stored"), requests, [256])).double()
    spread = (want - want.mean(dim=1, keepdim=True)).norm()
    return q8.model, max(float((torch.cat(logits(q8, requests, cuts)).double() - want).norm() / spread) for cuts in ([256], [1], [5, 40]))


def test_a_mixture_s_shared_expert(tmp_path):
    from spyinfer_amd.kernels import ops
    require_gpu()
    c = tarunex_cases
    config = dict(c.TAR_C, layers=[c._layer("attention", c._attention(4, 2, 64, 32, 0.12, 20.0, 0.25, 32), c._moe(64, 2, 2, 64)),
                                   c._layer("attention", c._attention(8, 2, 32, 48, 0.18, 10.0, 0.2, 64), c._moe(64, 4, 4, 75))])
    model, off = whole_model(c.write_model, config, tmp_path, 31, 400)
    for layer in model.layers:
        shared = layer.ffn.shared
        assert isinstance(shared.w_gate_up, ops.Q8Weight) and isinstance(shared.w_down, ops.Q8Weight) and isinstance(layer.mixer.w_o, ops.Q8Weight)
    assert off < 0.1, off


@pytest.mark.parametrize("design", ["meronex", "nolatar"])
def test_attention_beside_another_mixer(design, tmp_path):
    from spyinfer_amd.kernels import ops
    require_gpu()
    if design == "meronex":
        c = meronex_cases
        config = dict(c.MER_C, layers=[dict(c.MER_C["layers"][1], mlp=c._moe(128, 3.0, 1, 1)), c.MER_C["layers"][3]])
    else:
        c = nolatar_cases
        config = dict(c.NOL_C, layers=[dict(c.NOL_C["layers"][2], mlp=c._moe(128, 2, 2, 96)), dict(c.NOL_C["layers"][2], mlp=None)])
    model, off = whole_model(c.write_model, config, tmp_path, 32, 400)
    assert all(isinstance(layer.mixer.left.w_qkv, ops.Q8Weight) and isinstance(layer.mixer.left.w_o, ops.Q8Weight) for layer in model.layers)
    assert off < 0.1, off
