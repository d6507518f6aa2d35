"""GPU tests of the paged 8-bit cache's calls at the largest sizes that they take."""
import numpy as np
import pytest
import torch

import dgx_attn as A

pytestmark = pytest.mark.gpu


def i32(a):
    return torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).cuda()


@pytest.mark.parametrize("in_place", [False, True])
def test_a_plan_with_room_for_2_31_rows(in_place):
    """slots [2^31 - 1]: the grid's size is a sum past 32 bits. A few requests take their places, every other row gets none."""
    rows, page = (1 << 31) - 1, 16
    slots = torch.zeros(rows, dtype=torch.int32, device="cuda")
    ctx, add = np.array([5, 0, 40]), np.array([30, 0, 20])
    table = i32([[7, -1, -1, -1], [-1] * 4, [1, 2, 3, -1]])
    count, cu, status = i32([4]), i32([0] * 4), i32([9])
    left = count if in_place else i32([0])
    A.kv8_plan(i32(ctx), i32(add), page, table, i32([10, 11, 12, 13]), count, left, cu, slots, status)
    assert int(status[0]) == 0 and int(left[0]) == 1 and cu.tolist() == [0, 30, 30, 50]
    assert table.tolist() == [[7, 13, 12, -1], [-1] * 4, [1, 2, 3, 11]]
    want = [[7, 13, 12][p // 16] * 16 + p % 16 for p in range(5, 35)] + [[1, 2, 3, 11][p // 16] * 16 + p % 16 for p in range(40, 60)]
    assert slots[:50].tolist() == want
    assert int(slots[50:].min()) == -1 and int(slots[50:].max()) == -1
