"""The engine option for matrices in 8 bits, without a GPU."""
import pytest
import torch

from spyinfer_amd.config.engine_config import EngineConfig
from spyinfer_amd.engine.runner import bind_weights
from spyinfer_amd.kernels import ops


def test_option():
    assert EngineConfig().matrix_precision == "stored"
    EngineConfig(matrix_precision="int8").validate()
    for bad in (dict(matrix_precision="int4"), dict(matrix_precision="int8", dtype="float32")):
        with pytest.raises(ValueError, match="matrix_precision"):
            EngineConfig(**bad).validate()


class _Model:
    """Binds one matrix, which asks for 8 bits or does not."""

    def __init__(self, q8):
        self.q8 = q8

    def bind(self, weights, device):
        assert ops.MATRICES_Q8
        if weights is None:
            raise RuntimeError("no weights")
        self.forms = ops.weight_forms(weights["w"], q8=self.q8)


def test_binding(monkeypatch):
    made = []
    monkeypatch.setattr(ops, "quantize_weight", lambda w, gated=False: made.append(gated) or "in 8 bits")
    model = _Model(True)
    bind_weights(model, {"w": torch.zeros(2, 2)}, "cpu", matrix_precision="int8")
    assert model.forms == ("in 8 bits", None) and made == [False] and not ops.MATRICES_Q8
    with pytest.raises(ValueError, match="no matrix"):
        bind_weights(_Model(False), {"w": torch.zeros(2, 2)}, "cpu", matrix_precision="int8")
    with pytest.raises(RuntimeError):
        bind_weights(_Model(True), None, "cpu", matrix_precision="int8")
    assert not ops.MATRICES_Q8
    w = torch.zeros(2, 2)
    assert ops.weight_forms(w, q8=True)[0] is w


def test_products_go_by_the_matrix(monkeypatch):
    """Every product of a part takes a matrix in 8 bits in a matrix' place, and rows in 8 bits or not."""
    rows, w, wg = (ops.Q8Rows(torch.zeros((2, 256), dtype=torch.int8), torch.ones(2), 16), ops.Q8Weight.from_values(torch.zeros((8, 16), dtype=torch.int8), torch.ones(8)),
                   ops.Q8Weight.from_values(torch.zeros((8, 16), dtype=torch.int8), torch.ones(8), gated=True))
    calls = []
    monkeypatch.setattr(ops, "quantize_rows", lambda x: rows)
    monkeypatch.setattr(ops, "linear_q8", lambda x, m, dtype, out=None: calls.append((x, m, dtype, out)) or "y")
    monkeypatch.setattr(ops, "linear_q8_gated", lambda x, m, act: calls.append((x, m, act)) or "g")
    x = torch.zeros(2, 16, dtype=torch.bfloat16)
    for given in (x, rows):
        assert ops.linear(given, w) == ops.linear_few(given, w) == ops.linear_parts(given, w) == "y"
        assert ops.linear(given, w, torch.float32, out="here") == "y"
        assert ops.linear_swiglu(given, wg, activation="gelu_tanh") == "g"
    b = (rows, w, torch.bfloat16, None)
    assert calls == [b, b, b, (rows, w, torch.float32, "here"), (rows, wg, "gelu_tanh")] * 2
    assert ops.linear(x.float(), w) == "y" and calls[-1] == (rows, w, torch.float32, None)
