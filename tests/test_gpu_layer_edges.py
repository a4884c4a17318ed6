"""The operators between a layer's projections on the GPU at the ends of what their documentation allows: sequences of more
elements than 31 bits count, and more threads than one launch holds."""
import pytest
import torch

from monarch_muon_amd import rotary, rotary_table
from oracle import layer as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def randn(*shape, seed=0, size=1.0, dtype=torch.bfloat16):
    return (size * torch.randn(shape, generator=torch.Generator().manual_seed(seed))).to(DEV).to(dtype)


def room_for(gigabytes):
    if torch.cuda.get_device_properties(0).total_memory < gigabytes << 30:
        pytest.skip(f"needs {gigabytes} GB")


# ----- rotary ----------------------------------------------------------------------
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_of_a_sequence_of_more_than_31_bits(interleaved):
    """2^31 + 10240 elements of one sequence: the bits of its two halves, and the exact values at its ends."""
    room_for(60)
    T, H, K, D, part = (1 << 20) + 5, 15, 1, 128, 64
    q, k = randn(1, 997, H, D, seed=1).repeat(1, T // 997 + 1, 1, 1)[:, :T], randn(1, 1, K, D, seed=2).expand(1, T, K, D)
    table, at = rotary_table(part, T, device=DEV), torch.arange(T, device=DEV)
    out = rotary(q, k, table, interleaved=interleaved)
    for half in (slice(0, T // 2), slice(T // 2, T)):
        for x, y in zip(out, rotary(q[:, half], k[:, half], table, at[half], interleaved=interleaved)):
            assert torch.equal(x[:, half], y)
    ends = torch.tensor([0, 1, T // 2, T - 1], device=DEV)
    angles = ends.double()[None, :, None] * 10000.0 ** (-torch.arange(0, part, 2, dtype=torch.float64, device=DEV) / part)
    for x, y in zip((q, k), out):
        ref, tol = oracle.rotary(x[:, ends], angles, interleaved=interleaved)
        assert ((y[:, ends].double() - ref).abs() <= tol).all()


def test_rotary_of_a_sequence_of_more_threads_than_a_launch():
    """2^31 + 70 tokens of one chunk: a launch holds 2^31 of them."""
    room_for(90)
    T, cycle = (1 << 31) + 70, 1000
    q, table = randn(1, 1, 1, 2, seed=3), rotary_table(2, cycle, device=DEV)
    at = torch.arange(T, device=DEV).remainder_(cycle)
    out, _ = rotary(q.expand(1, T, 1, 2), q[:, :, :0].expand(1, T, 0, 2), table, at)
    ref, _ = rotary(q.expand(1, cycle, 1, 2), q[:, :, :0].expand(1, cycle, 0, 2), table)
    out, ref = out.view(torch.int32).flatten(), ref.view(torch.int32).flatten()
    whole = T // cycle * cycle
    assert torch.equal(out[:whole].view(-1, cycle), ref.expand(T // cycle, cycle))
    assert torch.equal(out[whole:], ref[:T - whole])
