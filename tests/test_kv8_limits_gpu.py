"""GPU: what the operators around an 8-bit KV cache do at the edges of their contract -- indices and lengths out of range, more tokens than rows,
numbers of every size in both attention kernels, negative softmax scales, windows as long as the longest sequence."""
import math

import pytest
import torch

import flash_attn_npu_v3 as fa3
import kv8_util as U
from flash_b200 import lib as L
from kv8_util import BF, E4M3, FP, INT8
from test_kv8_gpu import _cache_for, _gen, _i32, _random_cache, _raw, _status

pytestmark = pytest.mark.gpu


def _reported():
    """Whether the device status word told of an index out of range (and clears it)."""
    torch.cuda.synchronize()
    rc = L.load().fa_b200_check_status(torch.cuda.current_stream().cuda_stream)
    assert rc == 0 or "out of range" in L.load().fa_b200_last_error().decode()
    return rc != 0


# ---------------------------------------------------------------- plan
@pytest.mark.parametrize("have,new,total,after,cu,real", [
    ([5, 0, 16], [4, 10, 3], 12, [9, 0, 16], [0, 4, 12, 12], 4),             # the second is cut, the third has no row at all
    ([5, 0, 16], [4, 8, 0], 12, [9, 8, 16], [0, 4, 12, 12], 12),             # just as many tokens as rows
    ([5, 0, 16], [4, 8, 1], 12, [9, 8, 16], [0, 4, 12, 12], 12),
    ([1, 2], [1, 1], 0, [1, 2], [0, 0, 0], 0),
    ([0, 0, 5], [2 ** 31 - 1, 2 ** 31 - 1, 3], 6, [0, 0, 5], [0, 6, 6, 6], 0),  # sums beyond 32 bits
    ([7, 0, 3], [2, 2 ** 31 - 1, 1], 6, [9, 0, 3], [0, 2, 6, 6], 2)])
def test_plan_of_more_tokens_than_rows(have, new, total, after, cu, real):
    """A request whose tokens end behind the packed batch is left as it was and reported; offsets stay within the batch."""
    page, cols, free = 16, 4, [30, 31, 32, 33, 34]
    rows = torch.arange(len(have) * cols).view(-1, cols) + 100
    table = _i32(rows.tolist())
    slots, cu_got, after_got, positions, taken = fa3.paged_kvcache_plan(_i32(have), _i32(new), table, _i32(free), page, total)
    assert _reported() == (sum(new) > total)
    assert after_got.tolist() == after and cu_got.tolist() == cu
    want_rows, used, want_slots = rows.tolist(), 0, []
    for r, (a, b) in enumerate(zip(have, after)):
        for col in range(-(-a // page), -(-b // page)):
            want_rows[r][col], used = free[used], used + 1
        want_slots += [want_rows[r][t // page] * page + t % page for t in range(a, b)]
    assert taken.tolist() == [used] and table.tolist() == want_rows
    assert len(want_slots) == real and slots.tolist() == want_slots + [-1] * (total - real)


@pytest.mark.parametrize("have,new", [([-1, 4], [3, 2]), ([4, 4], [-3, 2])])
def test_plan_of_negative_lengths(have, new):
    table = torch.full((2, 3), 7, dtype=torch.int32, device="cuda")
    slots, cu, after, _, taken = fa3.paged_kvcache_plan(_i32(have), _i32(new), table, _i32([9, 8]), 4, 6)
    assert _reported()
    assert after.tolist() == [have[0], 6] and taken.tolist() == [1] and table.tolist() == [[7, 7, 7], [7, 9, 7]]
    at = max(new[0], 0)
    assert cu.tolist() == [0, at, at + 2] and slots.tolist() == ([-1] * at + [36, 37] + [-1] * 6)[:6]
