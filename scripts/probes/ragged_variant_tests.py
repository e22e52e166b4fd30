"""Both kernels of the ragged attention with every tile and several splits, on the same cases: the measurement build's `attn_ragged` tunable names the choice
that the product's cost model makes by itself.  Run by tests/test_gpu_ragged_variants.py in a process of its own (FVK_PROBE_LIB=1)."""
import ctypes as C
import os
import random
import sys

assert os.environ.get("FVK_PROBE_LIB") == "1", "run with FVK_PROBE_LIB=1 (see the module docstring)"
ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path[:0] = [ROOT, os.path.join(ROOT, "tests")]

import pytest
import torch

import _ragged_ref as ref
from test_paged_host import attn_args
from test_gpu_paged import BLOCKS, DEV, NAN, TOKENS, check_paged, cu, i32, paged_case, rnd

pytestmark = pytest.mark.gpu
VARIANTS = [(16, 1), (16, 3), (32, 1), (32, 12), (64, 1), (64, 5), (256, 1), (256, 2), (256, 5), (256, 16)]


@pytest.fixture(params=VARIANTS, ids=lambda v: f"tile{v[0]}x{v[1]}")
def ops(request):
    from fastvideo_amd import ops as o
    tile, parts = request.param
    o.set_tunable("attn_ragged", tile + 1024 * parts)
    got = C.c_int(), C.c_int()
    o._lib.call("fvk_attn_ragged_choice", C.byref(attn_args(o._lib)), *map(C.byref, got))
    assert (got[0].value, got[1].value) == request.param
    yield o
    o.set_tunable("attn_ragged", 0)


@pytest.mark.parametrize("causal", [False, True])
def test_tokens_and_blocks(ops, causal):
    for n, case in enumerate(TOKENS + BLOCKS):
        check_paged(ops, 10 + n, *case, causal, layout="hpd" if n % 2 else "phd")


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("causal,window,sink", [(False, 0, 0), (True, 0, 0), (False, 700, 333), (True, 300, 130), (True, 1, 0), (False, 1100, 1600)])
def test_long_walks(ops, page, causal, window, sink):
    """More than eight stages of the block kernel (1024 keys), more than sixteen with the second request; windows and sinks that end inside a stage, a page and
    a 16-key group; rows nobody sees are Inf / NaN."""
    check_paged(ops, page + window, [70, 0, 300, 5], [1190, 40, 1953, 700], 4, 2, page, causal, window, sink, layout="hpd" if page == 64 else "phd")


@pytest.mark.parametrize("R,H,Hkv", [(9, 5, 1), (65, 3, 3), (140, 2, 2), (7, 40, 8), (3, 13, 13)])
@pytest.mark.parametrize("causal,window,sink", [(False, 0, 0), (True, 150, 9)])
def test_many_requests(ops, R, H, Hkv, causal, window, sink):
    rng = random.Random(R + window)
    new = [rng.choice([0, 1, 65, 256, 257]) if R < 30 else rng.choice([0, 1, 3, 66]) for _ in range(R)]
    new[R // 2] = 520 if R < 30 else 258
    check_paged(ops, R, new, [rng.choice([0, 1, 100, 240]) for _ in range(R)], H, Hkv, 16, causal, window, sink)


def test_rows_that_see_nothing(ops):
    """kv_len below the number of rows, and none at all: zeros and -inf, whole blocks of 256 rows among them."""
    q, kp, vp, table, lens, cq = paged_case(3, [20, 9, 4, 600], [0, 0, 0, 0], 4, 2, 16)
    lens = [7, 0, 4, 150]
    for causal in (False, True):
        o, lse = ops.attn_paged(q, kp, vp, i32(table), i32(lens), i32(cq), causal=causal, return_lse=True)
        want, tol, want_lse = ref.paged(q, kp, vp, table, lens, cq, 128**-0.5, causal)
        assert ((o.double().cpu() - want).abs() <= tol).all()
        assert torch.equal(lse.cpu() == float("-inf"), want_lse == float("-inf"))
        assert (not causal) or (o[33:33 + 450] == 0).all()


@pytest.mark.parametrize("new", [1, 40, 260])
def test_large_scores_and_rising_maximum(ops, new):
    """test_gpu_paged.py's case: a fixed softmax reference leaves its range in nearly every row, the exact pass follows.  Its tolerance."""
    H, page = 2, 32
    q, kp, vp, table, lens, cq = paged_case(9, [new], [1000], H, H, page, poison=False)
    direction = rnd(77, 128).float()
    direction /= direction.norm()
    q = (q.float() * 0.2 + 8 * direction).bfloat16()
    for j in range(lens[0]):
        kp[table[0][j // page], j % page] += (direction * (j * 0.6)).bfloat16()
    want, tol, _ = ref.paged(q, kp, vp, table, lens, cq, 128**-0.5)
    o = ops.attn_paged(q, kp, vp, i32(table), i32(lens), i32(cq), max_q=new)
    assert torch.isfinite(o).all() and ((o.double().cpu() - want).abs() <= tol + 128 * 2.0**-24 * 600 * 2 * vp.abs().max().item()).all()
    # a falling maximum: the reference stays, the later keys' weights vanish
    flip = torch.flip(torch.arange(lens[0]), [0]).tolist()
    kf, vf = kp.clone(), vp.clone()
    for j, i in enumerate(flip):
        kf[table[0][j // page], j % page], vf[table[0][j // page], j % page] = kp[table[0][i // page], i % page], vp[table[0][i // page], i % page]
    want, tol, _ = ref.paged(q, kf, vf, table, lens, cq, 128**-0.5)
    o = ops.attn_paged(q, kf, vf, i32(table), i32(lens), i32(cq), max_q=new)
    assert torch.isfinite(o).all() and ((o.double().cpu() - want).abs() <= tol + 128 * 2.0**-24 * 600 * 2 * vp.abs().max().item()).all()


@pytest.mark.parametrize("both_signs", [False, True])
@pytest.mark.parametrize("causal,window,sink", [(False, 0, 0), (True, 260, 40)])
def test_products_beyond_fp32(ops, both_signs, causal, window, sink):
    """A key that outweighs the first ones by 2^80 (a second one with the opposite value), values of 2^60: the exact pass, for every part that meets one."""
    H, page, new = 2, 32, 260
    q, kp, vp, table, lens, cq = paged_case(14, [new, 70], [200, 250], H, H, page, poison=False)
    direction = rnd(78, 128).float()
    direction /= direction.norm()
    q = (q.float() * 0.2 + 8 * direction).bfloat16()
    vp *= 2.0**60
    for t in table[:2]:
        at = lambda x, j: x[t[j // page], j % page]
        at(kp, 150)[:] += (direction * 80).bfloat16()
        if both_signs:
            at(kp, 230)[:] = at(kp, 150)
            at(vp, 230)[:] = -at(vp, 150)
    o = ops.attn_paged(q, kp, vp, i32(table), i32(lens), i32(cq), causal=causal, window=window, sink=sink)
    want, tol, _ = ref.paged(q, kp, vp, table, lens, cq, 128**-0.5, causal, window, sink)
    assert torch.isfinite(o).all() and ((o.double().cpu() - want).abs() <= tol + 128 * 2.0**-24 * 60 * 2 * vp.abs().max().item()).all()


@pytest.mark.parametrize("new,window,sink", [(300, 2**31 - 1, 0), (300, 2**31 - 1, 2**31 - 1), (300, 70, 2**31 - 1), (4, 9, 2**31 - 1)])
def test_windows_and_sinks_of_31_bits(ops, new, window, sink):
    q, kp, vp, table, lens, cq = paged_case(12, [new] * 2, [40] * 2, 2, 2, 32)
    lens = [3, min(lens[1], 290)]
    o = ops.attn_paged(q, kp, vp, i32(table), i32(lens), i32(cq), causal=True, window=window, sink=sink)
    want, tol, _ = ref.paged(q, kp, vp, table, lens, cq, 128**-0.5, True, window, sink)
    assert ((o.double().cpu() - want).abs() <= tol).all()


def test_bad_pages_and_metadata(ops):
    """Pages outside the pool read as zero rows; wrong lengths are clamped (the addresses: tests/ragged_bounds.cpp)."""
    q, kp, vp, table, lens, cq = paged_case(4, [3, 300], [50, 90], 4, 4, 16, poison=False)
    table[0][1], table[1][0], table[1][5] = -1, kp.shape[0], 2**31 - 1
    bad = [[p if 0 <= p < kp.shape[0] else -1 for p in t] for t in table]
    want, tol, _ = ref.paged(q, kp, vp, bad, lens, cq, 128**-0.5)
    o = ops.attn_paged(q, kp, vp, i32(table), i32(lens), i32(cq))
    assert ((o.double().cpu() - want).abs() <= tol).all()


def test_rows_behind_the_batch_stay(ops):
    for new in ([1, 2], [300, 5]):
        q, kp, vp, table, lens, cq = paged_case(6, new, [900, 30], 4, 2, 32)
        T = q.shape[0]
        out = torch.full((T + 9, 6, 128), 5.0, dtype=torch.bfloat16, device=DEV)
        o = ops.attn_paged(torch.cat([q, rnd(1, 9, 4, 128)]), kp, vp, i32(table), i32(lens), i32(cq), out=out[:, 1:5])
        want, tol, _ = ref.paged(q, kp, vp, table, lens, cq, 128**-0.5)
        assert ((o[:T].double().cpu() - want).abs() <= tol).all()
        assert (out[T:] == 5).all() and (out[:, 0] == 5).all() and (out[:, 5] == 5).all()


def test_pool_beyond_32_bit_offsets(ops):
    """A pool of 5 GiB per tensor: page offsets pass 2^32 bytes."""
    page, Hkv, new = 64, 8, 300
    n_pages = 5 * 2**30 // (page * Hkv * 256)
    kp, vp = (torch.empty((n_pages, page, Hkv, 128), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    ids = [n_pages - 1, 0, n_pages - 2, n_pages // 2 + 7, n_pages - 9]
    for i, p in enumerate(ids):
        kp[p], vp[p] = rnd(i, page, Hkv, 128), rnd(i + 50, page, Hkv, 128)
    q, length = rnd(99, new, Hkv, 128, scale=1.5), 4 * page + 11
    o = ops.attn_paged(q, kp, vp, i32([ids]), i32([length]), i32([0, new]))
    want, tol, _ = ref.paged(q, kp, vp, [ids], [length], [0, new], 128**-0.5)
    assert ((o.double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("new,keys,H,Hkv", [([1], [1], 2, 2), ([5, 1, 9], [3, 0, 40], 4, 2), ([64, 100], [512, 77], 6, 6), ([300, 2, 17], [1, 33, 129], 3, 1),
                                            ([270, 0, 31], [16, 5, 0], 12, 12), ([1, 1, 1, 1], [2000, 1, 0, 64], 40, 8), ([257, 520], [1100, 2100], 2, 1),
                                            ([3] * 69 + [260], [20] * 69 + [400], 2, 2)])
def test_packed_keys(ops, new, keys, H, Hkv):
    S = sum(keys)
    q, kv = rnd(1, sum(new), H, 128, scale=1.5), rnd(2, S + 4, 2, Hkv, 128)
    k, v = kv[2:S + 2, 0], kv[2:S + 2, 1]        # a fused projection's views with neighbours on both sides
    kv[:2], kv[S + 2:] = NAN, NAN
    cq, ck = cu(new), cu(keys)
    o, lse = ops.attn_varlen(q, k, v, i32(cq), i32(ck), return_lse=True)
    for r in range(len(new)):
        a, b = cq[r], cq[r + 1]
        want, tol, want_lse = ref.attention(q[a:b], k[ck[r]:ck[r + 1]], v[ck[r]:ck[r + 1]], 128**-0.5)
        assert ((o[a:b].double().cpu() - want).abs() <= tol).all(), r
        if keys[r]:
            assert ((lse[:, a:b].double().cpu() - want_lse).abs() <= ref.LSE_TOL).all()
        else:
            assert (lse[:, a:b] == float("-inf")).all() and (o[a:b] == 0).all()
