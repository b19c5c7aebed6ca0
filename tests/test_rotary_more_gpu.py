"""Rotary positions on the GPU: batches of more rows than one launch takes."""
import pytest
import torch

from custom_ops_b200 import ops, rotary_frequencies
from tests.paged_testlib import check_turned, turn_reference

pytestmark = pytest.mark.gpu
DTYPES = (torch.bfloat16, torch.float16)


@pytest.mark.parametrize("B", [65535, 65536, 70000, 131071])
@pytest.mark.parametrize("own_positions", [False, True])
def test_rotary_of_many_rows(B, own_positions):
    """Decoding-shaped calls: one token in each of many rows, strided in, and the same tokens as one row."""
    H, Hk, d = 3, 1, 64
    x = torch.randn(B, 1, H + Hk, d, device="cuda", generator=torch.Generator("cuda").manual_seed(B)).bfloat16()
    q, k = x[:, :, :H].transpose(1, 2), x[:, :, H:].transpose(1, 2)
    freqs, _ = rotary_frequencies(d, 10000.0)
    if own_positions:
        positions = torch.arange(2 * B, dtype=torch.int32, device="cuda").view(B, 2)[:, 1:] % 9001
    else:
        positions = torch.full((1,), 4321, dtype=torch.int64, device="cuda")
    a, b = ops.rotary(q, k, positions, freqs)
    assert a.shape == (B, H, 1, d) and b.shape == (B, Hk, 1, d) and a.is_contiguous() and b.is_contiguous()
    at = positions if own_positions else positions.expand(B, 1)
    for y, z in ((a, q), (b, k)):
        check_turned(y, turn_reference(z, at.unsqueeze(1), freqs))
    one = [t.permute(2, 1, 0, 3) for t in (q, k)]                        # (1, heads, B, d)
    for y, z in zip((a, b), ops.rotary(*one, at[:, 0].contiguous(), freqs)):
        assert torch.equal(y.permute(2, 1, 0, 3), z)


def test_rotary_of_one_row_for_many():
    """A row that is broadcast over the batch, and key heads without a row of their own."""
    d, B = 128, 66000
    freqs, _ = rotary_frequencies(d, 10000.0)
    x = torch.randn(1, 2, 1, d, device="cuda").half()
    a, b = ops.rotary(x.expand(B, -1, -1, -1), x[:, :0].expand(B, -1, -1, -1), torch.tensor([7], device="cuda"), freqs)
    want = ops.rotary(x, x[:, :0], torch.tensor([7], device="cuda"), freqs)[0]
    assert torch.equal(a, want.expand(B, -1, -1, -1)) and b.shape == (B, 0, 1, d)
