"""Table operators refuse operands that share memory with what they write, as far as strides show it."""
import pytest
import torch

from custom_ops_b200 import ops

pytestmark = pytest.mark.gpu
OVERLAP = "memory location"


def test_tables_inside_what_is_written_are_refused():
    i32 = dict(dtype=torch.int32, device="cuda")
    pool = torch.zeros(64, **i32)
    table, lens, n, head = torch.zeros(4, 6, **i32), torch.zeros(4, **i32), torch.ones(4, **i32), torch.zeros(1, **i32)
    free = torch.arange(1, 30, **i32)
    inside = table.view(-1)
    for args in ((table, inside[:4], n, free, head), (table, lens, inside[3:7], free, head), (table, lens, n, inside[5:20], head),
                 (table, lens, n, free, inside[23:])):
        for call in (lambda a: ops.paged_extend(*a, 8, 4), lambda a: ops.paged_extend_(*a, 8, 4), lambda a: ops.paged_shrink_(*a, 8)):
            with pytest.raises(RuntimeError, match=OVERLAP):
                call(args)
    for args in ((table, pool[:4], n, pool[3:40], head), (table, pool[:4], n, free, pool[2:3]), (table, lens, n, pool[:30], pool[:1])):
        for call in (lambda a: ops.paged_extend_(*a, 8, 4), lambda a: ops.paged_shrink_(*a, 8)):
            with pytest.raises(RuntimeError, match=OVERLAP):
                call(args)
    assert not table.any() and not lens.any() and not head.any() and not pool.any()


def test_tables_beside_one_another_in_one_buffer():
    """One buffer for all of the state, and lengths that are doubled: nothing is shared that is written early."""
    i32 = dict(dtype=torch.int32, device="cuda")
    state = torch.zeros(4 + 1 + 29 + 24, **i32)
    lens, head, free, table = state[:4], state[4:5], state[5:34], state[34:].view(4, 6)
    free.copy_(torch.arange(1, 30))
    lens.copy_(torch.tensor([0, 3, 8, 0]))
    head.fill_(2)
    table[1, 0], table[2, 0] = 1, 2
    slots, positions, cu = ops.paged_extend_(table, lens, lens, free, head, 8, 11)
    assert lens.tolist() == [0, 6, 16, 0] and head.item() == 3 and cu.tolist() == [0, 0, 3, 11, 11]
    assert slots.tolist() == [11, 12, 13] + list(range(24, 32)) and positions.tolist() == [3, 4, 5] + list(range(8, 16))
    ops.paged_shrink_(table, lens, torch.tensor([0, 0, 9, 5], **i32), free, head, 8)
    assert lens.tolist() == [0, 0, 9, 0] and head.item() == 2 and free[:4].tolist() == [1, 2, 1, 4]
