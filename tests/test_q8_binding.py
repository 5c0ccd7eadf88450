"""Models bound from several threads at once, each with its own forms of the matrices (engine/runner.py, ops.weight_forms), without a GPU."""
import threading

import pytest
import torch

from spyinfer_amd.engine.runner import bind_weights
from spyinfer_amd.kernels import ops


class _Model:
    """Binds one matrix in 8 bits if that is asked for and it can be held so, one that cannot, and a gated feed-forward; ``pause`` is called before each."""

    def __init__(self, pause=lambda: None, q8=True):
        from spyinfer_amd.parts.mlp import GatedMLP
        self.pause, self.q8, self.mlp = pause, q8, GatedMLP(8, 24)

    def bind(self, weights, device):
        self.forms = []
        for q8 in (self.q8, False):
            self.pause()
            self.forms.append(ops.weight_forms(torch.zeros(16, 128), q8=q8))
        self.pause()
        if self.q8:
            self.mlp.bind("mlp", {"mlp.%s_proj.weight" % n: torch.zeros((24, 8) if n != "down" else (8, 24)) for n in ("gate", "up", "down")})


def kinds(model):
    return [m if isinstance(m, str) else type(m).__name__ for m, _ in model.forms] + [m if isinstance(m, str) else "Tensor" for m in (model.mlp.w_gate_up, model.mlp.w_down)]


@pytest.fixture
def forms(monkeypatch):
    """Matrices in 8 bits, tiled copies and tiled copies alone as names of their own."""
    monkeypatch.setattr(ops, "quantize_weight", lambda w, gated=False: "int8")
    monkeypatch.setattr(ops, "tile_weight", lambda w: "tiled")
    monkeypatch.setattr(ops, "TiledOnly", lambda t: "tiles alone")


STORED, INT8, ALONE = ["Tensor"] * 4, ["int8", "Tensor", "int8", "int8"], ["int8", "tiles alone", "int8", "int8"]


def run(*jobs):
    """Each job in a thread of its own; what each raised, or None."""
    raised = [None] * len(jobs)

    def guarded(i):
        try:
            jobs[i]()
        except Exception as e:
            raised[i] = e
    threads = [threading.Thread(target=guarded, args=(i,), daemon=True) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(30)
        assert not t.is_alive()
    return raised


def test_two_models_at_once_have_each_its_own(forms):
    """Both go from matrix to matrix in turn, so that each has entered before the other binds anything, and the one that entered first leaves first."""
    meet = threading.Barrier(2, timeout=20)
    for copies, kinds_of_first in (("both", INT8), ("tiled", ALONE)):
        first, second = _Model(meet.wait), _Model(meet.wait)
        assert run(lambda: bind_weights(first, {}, "cpu", copies, "int8"), lambda: bind_weights(second, {}, "cpu", "both", "stored")) == [None, None]
        assert kinds(first) == kinds_of_first
        assert kinds(second) == STORED
        assert not ops.MATRICES_Q8 and ops.weight_forms(torch.zeros(16, 128), q8=True)[1] == "tiled"


def test_leaving_in_another_order_than_entering(forms):
    """The one that entered last leaves last: nothing of either stays."""
    entered, left = threading.Event(), threading.Event()
    a = _Model(lambda: entered.wait(20))
    b = _Model(lambda: (entered.set(), left.wait(20)))

    def bind_a():
        bind_weights(a, {}, "cpu", "tiled", "int8")
        left.set()
    assert run(bind_a, lambda: bind_weights(b, {}, "cpu", "both", "stored")) == [None, None]
    assert kinds(a) == ALONE and kinds(b) == STORED
    for q8 in (True, False):
        w = torch.zeros(16, 128)
        assert ops.weight_forms(w, q8=q8)[0] is w
    assert not ops.MATRICES_Q8 and ops.ROW_MAJOR_WEIGHTS


def test_a_model_that_keeps_nothing_in_8_bits_says_so_beside_one_that_does(forms):
    meet = threading.Barrier(2, timeout=20)
    some, none = _Model(meet.wait), _Model(meet.wait, q8=False)
    raised = run(lambda: bind_weights(some, {}, "cpu", "both", "int8"), lambda: bind_weights(none, {}, "cpu", "both", "int8"))
    assert raised[0] is None and isinstance(raised[1], ValueError) and "no matrix" in str(raised[1])
    assert kinds(some) == INT8
