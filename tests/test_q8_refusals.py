"""What the 8-bit products and the operators that make their rows turn away, before anything is asked of a GPU."""
import pytest
import torch

from spyinfer_amd.kernels import ops
from spyinfer_amd.kernels.ops import KernelError, Q8Rows, Q8Weight


def rows(t=2, k=32):
    return Q8Rows(torch.zeros((t, (k + 255) // 256 * 256), dtype=torch.int8), torch.ones(t), k)


def weight(n=32, k=32, gated=False):
    return Q8Weight(torch.zeros((-(-k // 256), n // 16, 4, 4, 16, 16), dtype=torch.int8), torch.ones(n), (n, k), gated)


@pytest.mark.parametrize("call, says", [
    (lambda: ops.quantize_rows(torch.zeros(2, 8)), "on the GPU"),
    (lambda: ops.quantize_rows(torch.zeros(8)), "rows"),
    (lambda: ops.add_rms_norm_q8(torch.zeros(2, 8), None, torch.ones(8), 1e-6), "GPU only"),
    (lambda: ops.linear_q8(torch.zeros(2, 32), weight()), "Q8Rows"),
    (lambda: ops.linear_q8(rows(), torch.zeros(32, 32)), "Q8Weight"),
    (lambda: ops.linear_q8(rows(), weight(gated=True)), "linear_q8_gated"),
    (lambda: ops.linear_q8(rows(k=31), weight()), "rows of 31"),
    (lambda: ops.linear_q8(rows(), weight(), torch.float16), "output dtype"),
    (lambda: ops.linear_q8(rows(), weight()), "GPU only"),
    (lambda: ops.linear_q8_gated(rows(), weight()), "gate"),
    (lambda: ops.linear_q8_gated(rows(k=48), weight(gated=True)), "rows of 48"),
    (lambda: ops.linear_q8_gated(rows(), weight(gated=True), "relu"), "relu"),
    (lambda: ops.linear_q8_gated(rows(), weight(gated=True)), "GPU only"),
    (lambda: ops.quantize_weight(torch.zeros(4, 8)), "on the GPU"),
    (lambda: Q8Rows(torch.zeros((2, 33), dtype=torch.int8), torch.ones(2), 33), "rounded up to 256"),
    (lambda: Q8Rows(torch.zeros((2, 512), dtype=torch.int8), torch.ones(2), 256), "rounded up to 256"),
    (lambda: Q8Rows(torch.zeros((256, 2), dtype=torch.int8).t(), torch.ones(2), 48), "dense"),
    (lambda: Q8Rows(torch.zeros((2, 256), dtype=torch.int8), torch.ones(4)[::2], 48), "scale"),
    (lambda: Q8Weight(torch.zeros((1, 2, 4, 4, 16, 16), dtype=torch.int8), torch.ones(16), (32, 256), False), "scale"),
    (lambda: Q8Weight(torch.zeros((1, 2, 4, 4, 16, 16), dtype=torch.int8), torch.ones(32), (33, 256), False), "tiles"),
    (lambda: Q8Weight(torch.zeros((1, 2, 4, 4, 16, 16), dtype=torch.int8), torch.ones(32), (31, 256), True), "gate and up"),
    (lambda: Q8Rows.from_values(torch.zeros(2, 8), torch.ones(2)), "int8"),
    (lambda: Q8Rows.from_values(torch.zeros((2, 8), dtype=torch.int8), torch.ones(3)), "scale"),
    (lambda: Q8Weight.from_values(torch.zeros(2, 8), torch.ones(2)), "int8"),
    (lambda: Q8Weight.from_values(torch.zeros((2, 8), dtype=torch.int8), torch.ones(2).double()), "scale"),
    (lambda: Q8Weight.from_values(torch.zeros((3, 8), dtype=torch.int8), torch.ones(3), gated=True), "3 rows"),
    (lambda: Q8Weight.from_values(torch.zeros((2, 8), dtype=torch.int8), torch.tensor([1.0, float("nan")])), "finite"),
    (lambda: Q8Weight.from_values(torch.zeros((1, ops.Q8_MAX_WIDTH + 1), dtype=torch.int8), torch.ones(1)), "sums hold"),
])
def test_turned_away(call, says):
    with pytest.raises(KernelError, match=says):
        call()


@pytest.mark.parametrize("N,K,gated", [(1, 1, False), (16, 256, False), (33, 300, False), (34, 300, True), (96, 64, True), (2, 1, True)])
def test_a_matrix_laid_out_is_the_matrix(N, K, gated):
    g = torch.Generator().manual_seed(N + K)
    p = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8)
    s = torch.rand(N, generator=g) + 0.5
    w = Q8Weight.from_values(p, s, gated)
    assert torch.equal(w.to_rows(), p.float() * s[:, None]) and tuple(w.shape) == (N, K)
    # an element's place: chunk k / 256, tile, step, lane 16 (k / 16 % 4) + row, byte
    half = -(-N // 2 // 16) * 16 if gated else 0
    for n in range(0, N, 5):
        row = n if not gated or n < N // 2 else half + n - N // 2
        for k in range(0, K, 7):
            assert w.tiles[k // 256, row // 16, k // 64 % 4, k // 16 % 4, row % 16, k % 16] == p[n, k]


def test_rows_of_any_width_are_kept_in_pieces_of_256():
    q = torch.arange(-33, 33, dtype=torch.int8).view(2, 33)
    r = Q8Rows(torch.zeros((2, 256), dtype=torch.int8), torch.tensor([2.0, 0.5]), 33)
    r.values[:, :33] = q
    assert torch.equal(r.to_rows(), q.float() * r.scales[:, None]) and r.shape == (2, 33)


def test_a_matrix_from_any_place_in_memory():
    """Values that begin at any byte, rows of a wider tensor, and scales whose sum is no float32."""
    g = torch.Generator().manual_seed(1)
    flat = torch.randint(-128, 128, (3 + 32 * 256,), generator=g, dtype=torch.int8)
    p, s = flat[3:].view(32, 256), torch.full((32,), 3e38)
    assert torch.equal(Q8Weight.from_values(p, s).to_rows(torch.float64), p.double() * s[:, None].double())
    wide = torch.randint(-128, 128, (32, 600), generator=g, dtype=torch.int8)
    assert torch.equal(Q8Weight.from_values(wide[:, 5:261], s).to_rows(torch.float64), wide[:, 5:261].double() * s[:, None].double())
