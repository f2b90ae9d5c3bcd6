"""Layouts that no sort made, at the counts whose sums pass 32 bits: the experts'
products touch nothing outside their buffers, whose guard rows keep their values."""
import pytest
import torch

import momiru_b200 as mb
from test_linear_gpu import V, gen, rand, replay

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("cuda_lib")]
MOST = 2 ** 31 - 1
COUNTS = {
    "all the largest": lambda e: [MOST] * e,
    "sixteen of them": lambda e: [MOST] * min(e, 16) + [5] * max(e - 16, 0),  # 16 (2^31 - 1 + 15) wraps to 0 in 32 bits
    "all 2^30": lambda e: [2 ** 30] * e,
    "large and negative": lambda e: [MOST if i % 2 else -MOST for i in range(e)],
    "small, then large": lambda e: [1] * (e - e // 2) + [MOST] * (e // 2),
}


@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("tokens,experts,align,kernel", [
    (64, 64, 16, "mmr_linear_strip_kernel"), (40, 17, 1, "mmr_linear_strip_kernel"), (4000, 4, 64, "mmr_linear_pair_kernel"),
    (6000, 40, 128, "mmr_linear")])
def test_counts_whose_sums_pass_32_bits(counts, tokens, experts, align, kernel):
    t, k, n, guard = torch.bfloat16, 64, 136, 256
    g = gen(31)
    rows_n = mb.ExpertLayout.capacity(tokens, 2, experts, align)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for offsets in ([0] * (experts + 1), [rows_n - 1] * experts + [MOST]):
        lay = mb.ExpertLayout(tokens, 2, experts, align, V(i32([[-1, -1]] * tokens)), V(i32([-1] * rows_n)), V(i32(offsets)),
                              V(i32(COUNTS[counts](experts))))
        rows, w = rand(g, rows_n, k, dtype=t), rand(g, experts, k, n, dtype=t)
        buf = torch.full((rows_n + 2 * guard, n), 7.0, dtype=t, device="cuda")
        op = mb.BoundExpertLinear(mb.LinearNode(), lay, V(rows), V(w), V(buf[guard:guard + rows_n]))
        assert kernel in op.plan, op.plan
        replay(op)
        assert bool((buf[:guard] == 7).all()) and bool((buf[guard + rows_n:] == 7).all())
