"""More rows than one launch has threads for (2^32): the rows on both sides of the launches' borders and the last ones are those of the rows alone."""
import pytest
import torch

from tests.gpu_util import require_gpu

pytestmark = pytest.mark.gpu


def places(T):
    return [slice(0, 40)] + [slice(at - 20, at + 20) for at in range(1 << 21, T, 1 << 21)] + [slice(T - 40, T)]


@pytest.mark.parametrize("T,K,ld", [((1 << 21) + 3, 64, 64), ((1 << 22) + 1, 8, 24), ((1 << 24) + 77, 66, 66)])
def test_rows(T, K, ld):
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    g = torch.Generator(device=dev).manual_seed(T)
    x = torch.empty((T, ld), dtype=torch.bfloat16, device=dev).normal_(generator=g)[:, :K]
    got = ops.quantize_rows(x)
    for s in places(T):
        alone = ops.quantize_rows(x[s].clone())
        assert torch.equal(got.values[s, :K], alone.values[:, :K]) and torch.equal(got.scales[s], alone.scales)


@pytest.mark.parametrize("T,H,addend", [((1 << 21) + 3, 64, torch.bfloat16), ((1 << 24) + 77, 66, None), ((1 << 21) + 1, 33, torch.float32)])
def test_norm(T, H, addend):
    from spyinfer_amd.kernels import ops
    dev = require_gpu()
    g = torch.Generator(device=dev).manual_seed(T)
    stream, w = torch.empty((T, H), device=dev).normal_(generator=g), 1 + torch.rand(H, device=dev, generator=g)
    d = None if addend is None else torch.empty((T, H), dtype=addend, device=dev).normal_(generator=g)
    before = [stream[s].clone() for s in places(T)]
    got = ops.add_rms_norm_q8(stream, d, w, 1e-6)
    for s, mine in zip(places(T), before):
        alone = ops.add_rms_norm_q8(mine, None if d is None else d[s].clone(), w, 1e-6)
        assert torch.equal(got.values[s, :H], alone.values[:, :H]) and torch.equal(got.scales[s], alone.scales) and torch.equal(stream[s], mine)
