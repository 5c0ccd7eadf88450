"""Engines whose attention and feed-forward matrices are held in 8 bits (``matrix_precision="int8"``): logits beside those of the stored
matrices, prompts cut in every way, recorded steps, the entry points, and what is turned away.

A row or matrix in 8 bits is off by a / 127 / sqrt(12) evenly spread, a the largest value of some 100 to 700 of a bell curve, 2.7 to 3.5
times their root mean square: 0.6 to 0.8 % each, 1.1 % a product.  Two or three layers of four products each, one after the other, and all of them
added to a stream: 1.1 % sqrt(12) = 4 % of the layers' part of the logits; held to 10 %, where a wrong scale, order or row gives
errors of the size of the logits."""
import io
import json

import pytest
import torch

from tests.configs import INIT, TINY_C, TINY_D, TINY_E
from tests.gpu_util import require_gpu

pytestmark = pytest.mark.gpu


def folder_of(tmp_path, raw, seed):
    from spyinfer_amd.weights import write_random_model
    return write_random_model(str(tmp_path / "m"), raw, seed, torch.bfloat16, **INIT)


def runner_of(folder, precision, eager=True):
    from spyinfer_amd.engine.runner import ModelRunner, load_model
    model = load_model(folder, "bfloat16", "cuda:0", matrix_precision=precision)
    return ModelRunner(model, "bfloat16", "cuda:0", 16, 64, 8, enforce_eager=eager, max_model_len=256)


def logits(runner, requests, cuts):
    """Logits of every token of the requests, whose tokens run in portions of the sizes ``cuts``, side by side."""
    from spyinfer_amd.engine.batch import StepEntry
    caches = [runner.manager.admit(i) for i in range(len(requests))]
    done, out = [0] * len(requests), [[] for _ in requests]
    k = 0
    while any(d < len(r) for d, r in zip(done, requests)):
        n, k = cuts[k % len(cuts)], k + 1
        entries, live = [], []
        for i, r in enumerate(requests):
            part = r[done[i]:done[i] + n]
            if part:
                runner.manager.reserve(caches[i], len(part))
                entries.append(StepEntry(caches[i], part, list(range(len(part)))))
                live.append((i, len(part)))
        y = runner.step(entries).clone()
        for i, m in live:
            out[i].append(y[:m])
            y = y[m:]
            done[i] += m
    for c in caches:
        runner.manager.release(c)
    return [torch.cat(o) for o in out]


@pytest.mark.parametrize("raw", [TINY_C, TINY_D, TINY_E], ids=["odd", "folded", "wide-heads"])
def test_logits_beside_those_of_the_stored_matrices(raw, tmp_path):
    from spyinfer_amd.kernels import ops
    require_gpu()
    folder = folder_of(tmp_path, raw, 11)
    g = torch.Generator().manual_seed(5)
    requests = [torch.randint(0, raw["vocab_size"], (n,), generator=g).tolist() for n in (1, 17, 90, 33)]
    q8 = runner_of(folder, "int8")
    for layer in q8.model.layers:
        assert all(isinstance(m, ops.Q8Weight) for m in (layer.mixer.w_qkv, layer.mixer.w_o, layer.ffn.w_gate_up, layer.ffn.w_down))
        assert layer.ffn.w_gate_up.gated and layer.mixer.takes_q8_rows and layer.ffn.takes_q8_rows
    want = torch.cat(logits(runner_of(folder, "stored"), requests, [256])).double()
    got = {tuple(cuts): torch.cat(logits(q8, requests, cuts)).double() for cuts in ([256], [1], [7, 64, 2])}
    spread = (want - want.mean(dim=1, keepdim=True)).norm()
    for cuts, y in got.items():
        assert float((y - want).norm() / spread) < 0.1, cuts
    # another cut of the work gives another order of the attention's sums, which may move an activation to the next integer: a step of 8 bits
    # here and there, less than what the roundings themselves cost
    for y in got.values():
        assert float((y - got[(256,)]).norm() / spread) < 0.05


def test_recorded_steps_are_the_steps(tmp_path):
    """Single tokens step by step, kernel by kernel and replayed from graphs: the same bits."""
    require_gpu()
    folder = folder_of(tmp_path, TINY_E, 12)
    g = torch.Generator().manual_seed(6)
    requests = [torch.randint(0, TINY_E["vocab_size"], (24,), generator=g).tolist() for _ in range(3)]
    eager = logits(runner_of(folder, "int8"), requests, [1])
    runner = runner_of(folder, "int8", eager=False)
    for _ in range(2):
        got = logits(runner, requests, [1])
        assert all(torch.equal(a, b) for a, b in zip(eager, got))
    assert runner.graph_replays > 20


def test_entry_points(tmp_path, capsys):
    from spyinfer_amd import __main__ as main
    from spyinfer_amd.engine import replay
    from spyinfer_amd.engine.llm_engine import LLMEngine
    from spyinfer_amd.kernels import ops
    from spyinfer_amd.sampling import SamplingParams
    require_gpu()
    folder = folder_of(tmp_path, TINY_E, 13)
    g = torch.Generator().manual_seed(7)
    prompts = [torch.randint(0, TINY_E["vocab_size"], (n,), generator=g).tolist() for n in (5, 70, 33)]
    kw = dict(dtype="bfloat16", max_model_len=128, num_kvcache_blocks=40, max_num_seqs=8, matrix_precision="int8")
    eng = LLMEngine(folder, **kw)
    assert isinstance(eng.model.layers[1].ffn.w_down, ops.Q8Weight) and isinstance(eng.model.lm_head.weight, torch.Tensor)
    params = SamplingParams(max_new_tokens=12, ignore_eos=True)
    got = eng.generate(prompts, params)
    assert [len(t) for t in got] == [12, 12, 12]
    assert LLMEngine(folder, weight_copies="tiled", **kw).generate(prompts, params) == got
    # the command line and the replay
    alone = eng.generate(prompts[:1], params)[0]
    assert main.main(["-m", folder, "--dtype", "bfloat16", "--matrix-precision", "int8", "--prompt-ids", " ".join(map(str, prompts[0])), "--max-new-tokens", "12", "--ignore-eos",
                      "--max-model-len", "128", "--num-kvcache-blocks", "40", "--max-num-seqs", "8"]) == 0
    assert " ".join(map(str, alone)) in capsys.readouterr().out
    line = json.dumps({"step": 0, "entries": [{"id": 1, "tokens": prompts[0], "want": [len(prompts[0]) - 1]}]})
    assert replay.run(["--model", folder, "--dtype", "bfloat16", "--out", str(tmp_path / "o"), "--max-tokens", "64", "--matrix-precision", "int8"], io.StringIO(line + "\n"), io.StringIO()) == 0
    row = torch.frombuffer(bytearray((tmp_path / "o" / "0.f32").read_bytes()), dtype=torch.float32)
    assert int(row.argmax()) == alone[0]


@pytest.mark.parametrize("name", ["sodedra", "balelorn"])
def test_other_architectures(name, tmp_path):
    """Blocks in which others read the norm too, or whose results are normed: the rows are brought to 8 bits where the product begins."""
    from spyinfer_amd.kernels import ops
    from tests import balelorn_cases, sodedra_cases
    require_gpu()
    if name == "sodedra":
        folder, vocab = sodedra_cases.write_model(str(tmp_path / "m"), sodedra_cases.SOD_FAR, 21), sodedra_cases.SOD_FAR["vocab"]
    else:
        dense = balelorn_cases.BAL_C["layers"][0]
        folder, vocab = balelorn_cases.write_model(str(tmp_path / "m"), dict(balelorn_cases.BAL_C, layers=[dense, dense]), 22), balelorn_cases.BAL_C["vocab"]
    g = torch.Generator().manual_seed(8)
    requests = [torch.randint(0, vocab, (n,), generator=g).tolist() for n in (3, 80, 21)]
    q8 = runner_of(folder, "int8")
    assert isinstance(q8.model.layers[0].ffn.w_gate_up, ops.Q8Weight) and isinstance(q8.model.layers[0].mixer.w_qkv, ops.Q8Weight)
    want = torch.cat(logits(runner_of(folder, "stored"), requests, [256])).double()
    spread = (want - want.mean(dim=1, keepdim=True)).norm()
    for cuts in ([256], [1], [5, 40]):
        assert float((torch.cat(logits(q8, requests, cuts)).double() - want).norm() / spread) < 0.1, cuts


def test_what_is_turned_away(tmp_path):
    """A model without such matrices, a float32 model, a precision that does not exist."""
    from spyinfer_amd.engine.llm_engine import LLMEngine
    from spyinfer_amd.engine.runner import load_model
    from spyinfer_amd.kernels import ops
    from tests import sefevik_cases
    require_gpu()
    folder, other = folder_of(tmp_path, TINY_E, 14), sefevik_cases.write_model(str(tmp_path / "s"), sefevik_cases.SEF_C, 15)
    for call in (lambda: LLMEngine(folder, dtype="float32", matrix_precision="int8"), lambda: load_model(folder, "float32", "cuda:0", matrix_precision="int8"),
                 lambda: LLMEngine(folder, matrix_precision="int4"), lambda: load_model(other, "bfloat16", "cuda:0", matrix_precision="int8")):
        with pytest.raises(ValueError, match="matrix_precision"):
            call()
    assert not ops.MATRICES_Q8
