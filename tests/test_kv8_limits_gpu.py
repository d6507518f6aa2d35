"""GPU tests of the paged 8-bit cache's calls at the largest sizes that they take."""
import numpy as np
import pytest
import torch

import dgx_attn as A
import kv8_ref as R

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


def attend(heads, page, ctx, add, T, mp, shift=0, window=0, chunk=0):
    """One call at positions shifted by `shift` (a multiple of the page and of the splits), against the 64-bit form."""
    NQ, NKV, HD = heads
    rng = np.random.default_rng(page + T % 1000)
    ctx, add = np.array(ctx), np.array(add)
    lens, cu = ctx + add, np.concatenate([[0], np.cumsum(add)])
    P, rows = int((-(-lens // page)).sum()), int(add.sum())
    table = R.tables(rng, lens, page, P)
    K, V, Ks, Vs = R.make_cache_fast(rng, P, page, NKV, HD)
    R.blank_tail(K, V, table, lens, page)
    t = torch.full((len(ctx), mp // page + 1), -1, dtype=torch.int32, device="cuda")
    t[:, shift // page:shift // page + table.shape[1]] = i32(table)
    Q = torch.from_numpy(rng.standard_normal((rows, NQ, HD))).to(torch.bfloat16)
    O, lse = torch.full((rows, NQ, HD), 7.0, dtype=torch.bfloat16, device="cuda"), torch.empty(rows, NQ, device="cuda")
    A.attn_kv8(Q.cuda(), R.to_cache(A, K, V, Ks, Vs), t, i32(ctx + shift), O, T, mp, cu=i32(cu), window=window, chunk=chunk, lse=lse)
    torch.cuda.synchronize()
    R.check(O, lse, R.attention_rows(Q.double().numpy(), K, V, Ks, Vs, table, ctx, cu, window=window), f"T {T} max_pos {mp}")


@pytest.mark.parametrize("T", [100, 1 << 24, 1 << 27])
@pytest.mark.parametrize("window", [0, 33])
def test_a_bound_on_a_requests_rows_far_past_them(T, window):
    attend((24, 4, 256), 64, [100, 0, 300], [1, 3, 1], T, 400, window=window)
    attend((16, 1, 512), 16, [100, 0], [1, 70], min(T, 1 << 25), 400, window=window, chunk=64)


@pytest.mark.parametrize("heads,add,chunk", [((8, 2, 128), [1, 1], 0), ((8, 2, 128), [1, 1], 64), ((16, 1, 512), [8, 3], 128), ((4, 2, 256), [90, 1], 64),
                                             ((4, 2, 256), [90, 1], 0), ((64, 32, 256), [90, 70], 0), ((64, 32, 256), [90, 70], 64)])
def test_the_last_positions(heads, add, chunk):
    """Windows that end at position 2^30 - 1, the largest max_pos."""
    shift = (1 << 30) - 1024
    attend(heads, 64, [1024 - add[0], 700], add, max(add), (1 << 30) - 1, shift, window=200, chunk=chunk)
