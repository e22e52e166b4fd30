"""Calls of the batched-cache operators at the edges of their arguments, in the kernel each names: the sizes are ones that the cost model sends there."""
import random

import pytest
import torch

import _ragged_ref as ref
from test_gpu_paged import DEV, NAN, cu, i32, ops, paged_case, plan_case, rnd  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ plan: more tokens than rows
@pytest.mark.parametrize("R,W,page,new_hi,window,sink,causal,tight", [(1, 40, 16, 300, 0, 0, False, False), (5, 33, 16, 90, 200, 40, True, False),
                                                                      (9, 12, 32, 200, 90, 0, False, True), (300, 20, 16, 60, 0, 0, False, False),
                                                                      (700, 9, 16, 40, 50, 7, True, True), (1030, 70, 16, 30, 100, 0, False, False)])
@pytest.mark.parametrize("share", [0.0, 0.3, 0.999])
def test_plan_counts_only_tokens_that_have_a_row(ops, R, W, page, new_hi, window, sink, causal, tight, share):
    """A batch that holds a share of the new tokens: the plan is that of the tokens it holds, in lengths, pages, slots and dead pages alike."""
    starts, new, table, held, free, count = plan_case(random.Random(R), R, W, page, new_hi, tight)
    new[0] = max(new[0], 3)
    n_tokens = int(share * sum(new))
    ends = [min(c, n_tokens) for c in cu(new)]
    kept = [b - a for a, b in zip(ends, ends[1:])]
    p = ops.paged_plan(i32(starts), i32(new), i32(table), i32(held), i32(free), i32([count]), page_size=page, n_tokens=n_tokens, grid_hw=(2, 3), window=window,
                       sink=sink, causal=causal)
    want = ref.plan(starts, kept, table, held, free, count, page, n_tokens, 2, 3, window, sink, causal)
    for name, value in want.items():
        assert getattr(p, name).tolist() == value, name


def test_rows_of_a_cut_request_stand_behind_its_cache(ops):
    """A causal request of 9 new tokens of which 4 have a row: they see their own place and what lies before it, no row that nobody wrote (NaN here)."""
    H, page = 2, 16
    kp, vp = (torch.full((6, page, H, 128), NAN, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    kp[2, :7], vp[2, :7] = rnd(1, 7, H, 128), rnd(2, 7, H, 128)    # request 1 has cached 7 tokens
    x = rnd(3, 10, 3 * H * 128)
    p = ops.paged_plan(i32([0, 7]), i32([6, 9]), i32([[-1] * 4, [2, -1, -1, -1]]), i32([0, 1]), i32([0, 1, 3, 4, 5]), i32([5]), page_size=page, n_tokens=10, causal=True)
    assert p.kv_lens.tolist() == [6, 11] and p.pages_held.tolist() == [1, 1] and p.free_count.item() == 4 and p.granted.tolist() == [1, 1]
    assert p.slot_map.tolist() == [5 * page + i for i in range(6)] + [2 * page + 7 + i for i in range(4)]
    q = ops.rmsnorm_rope_paged(x[:, :256], x[:, 256:512], x[:, 512:], None, None, None, None, p.slot_map, kp, vp)
    o = ops.attn_paged(q.view(10, H, 128), kp, vp, p.block_table, p.kv_lens, p.cu_q, max_q=6, max_kv=16, causal=True)
    want, tol, _ = ref.paged(q.view(10, H, 128), kp, vp, p.block_table.tolist(), [6, 11], [0, 6, 10], 128**-0.5, True)
    assert ((o.double().cpu() - want).abs() <= tol).all()


# ------------------------------------------------------------------ attention


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


# ------------------------------------------------------------------ the model's batched forward
def test_a_cache_of_another_frame_size_is_refused(golden_dir):
    """A cache's window and sinks are counted in tokens of one frame size; frames of another would be cut in their middle.  Nothing has changed then."""
    import os
    from fastvideo_amd.wan_causal import CausalWanTransformer3DModelHip
    fx = torch.load(os.path.join(golden_dir, "wan_causal.pt"), weights_only=True)
    case, fs = fx["cases"][1], fx["frame_seqlen"]
    model = CausalWanTransformer3DModelHip(fx["state_dict"], num_heads=fx["config"]["num_heads"], local_attn_size=case["local_attn_size"],
                                           sink_size=case["sink_size"], rope_cache_policy="absolute", num_frames_per_block=2)
    c = case["calls"][0]
    lat, t, text = c["latent"].cuda(), c["timestep"].cuda(), model.text_kv([case["ctx"]])
    for size in (fs // 2, 2 * fs):
        cache = model.init_paged_cache(1, 20, 8 * fs, size, 16)
        with pytest.raises(ValueError, match=f"frames of {fs} tokens"):
            model.forward_paged(lat, text, t, cache, [0])
        assert cache.tokens == [0] and cache.free_page_count() == 20
    assert torch.isfinite(model.forward_paged(lat, text, t, model.init_paged_cache(1, 20, 8 * fs, fs, 16), [0])).all()
