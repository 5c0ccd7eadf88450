"""Matrices and rows in 8-bit integers made from a caller's tensors: they hold values of their own whatever the size, the place and the order of
the tensors, without a GPU."""
import pytest
import torch

from spyinfer_amd.kernels.ops import Q8Rows, Q8Weight


def drawn(N, K, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8), torch.rand(N, generator=g) + 0.5


@pytest.mark.parametrize("N,K,gated", [(16, 256, False), (32, 256, True), (48, 512, False), (15, 256, False), (32, 255, True), (34, 256, True)])
def test_a_matrix_stays_when_the_tensors_it_came_from_change(N, K, gated):
    p, s = drawn(N, K)
    want = p.double() * s.double()[:, None]
    w = Q8Weight.from_values(p, s, gated)
    s.fill_(7.0)
    p.zero_()
    assert torch.equal(w.to_rows(torch.float64), want)


@pytest.mark.parametrize("K", [256, 512, 255, 40])
def test_rows_stay_when_the_tensors_they_came_from_change(K):
    q, s = drawn(5, K, 1)
    want = q.double() * s.double()[:, None]
    x = Q8Rows.from_values(q, s)
    s.fill_(7.0)
    q.zero_()
    assert torch.equal(x.to_rows(torch.float64), want) and x.shape == (5, K)


@pytest.mark.parametrize("at", range(9))
@pytest.mark.parametrize("N,K,gated", [(16, 256, False), (256, 256, True), (64, 512, False), (17, 40, False)])
def test_a_transposed_matrix_from_any_place_in_memory(N, K, gated, at):
    p, s = drawn(N, K, at)
    flat = torch.empty(at + N * K, dtype=torch.int8)
    there = flat[at:].view(K, N).t()
    there.copy_(p)
    assert there.data_ptr() % 8 == (flat.data_ptr() + at) % 8 and not there.is_contiguous()
    assert torch.equal(Q8Weight.from_values(there, s, gated).to_rows(torch.float64), p.double() * s.double()[:, None])


@pytest.mark.parametrize("at", range(9))
def test_a_matrix_in_a_buffer_that_begins_anywhere(at):
    """The address may be a multiple of eight where the place in the storage is none, and the other way round."""
    p, s = drawn(16, 256)
    held = torch.frombuffer(bytearray(at + 20 + 16 * 256), dtype=torch.int8, offset=at)
    for skip in range(9):
        there = held[skip:skip + 16 * 256].view(16, 256)
        there.copy_(p)
        assert torch.equal(Q8Weight.from_values(there, s).to_rows(torch.float64), p.double() * s.double()[:, None])
