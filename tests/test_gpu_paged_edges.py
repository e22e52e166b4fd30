"""Calls of the batched-cache operators at the edges of their arguments, in the kernel each names: the sizes are ones that the cost model sends there."""
import pytest
import torch

import _ragged_ref as ref
from test_gpu_paged import i32, ops, paged_case, rnd  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu


def test_blocks_whose_products_leave_fp32_with_both_signs(ops):
    """Two keys outweigh a row's first ones by 2^80 each and carry values of 2^60 of opposite sign: against the first keys' maximum their products are +inf and
    -inf, their sum NaN in EVERY column and never plain infinity, while the row's sum stays in range and the result is finite.  R = 4, 16 heads of 260 rows
    each: the block kernel.  Tolerance: the scores' own fp32 error as for scores up to 60 (128 products of one rounding), the rest as everywhere."""
    R, H, page, new = 4, 16, 32, 260
    q, kp, vp, table, lens, cq = paged_case(21, [new] * R, [200] * R, H, H, page, poison=False)
    direction = rnd(79, 128).float()
    direction /= direction.norm()
    q = (q.float() * 0.2 + 8 * direction).bfloat16()
    vp *= 2.0**60
    for r in range(R):
        a, b = 150 + r, 330 + r
        ka = kp[table[r][a // page], a % page] + (direction * 80).bfloat16()
        for j, sign in ((a, 1), (b, -1)):
            kp[table[r][j // page], j % page] = ka
            vp[table[r][j // page], j % page] = sign * (1.0 + torch.arange(128, device="cuda") / 256) * 2.0**60
    o, lse = ops.attn_paged(q, kp, vp, i32(table), i32(lens), i32(cq), max_q=new, max_kv=max(lens), return_lse=True)
    want, tol, want_lse = ref.paged(q, kp, vp, table, lens, cq, 128**-0.5)
    assert torch.isfinite(o).all()
    assert ((o.double().cpu() - want).abs() <= tol + 128 * 2.0**-24 * 60 * 2 * vp.abs().max().item()).all()
    assert ((lse.double().cpu() - want_lse).abs() <= ref.LSE_TOL + 128 * 2.0**-24 * 60 * 2).all()
