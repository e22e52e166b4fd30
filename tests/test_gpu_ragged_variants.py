"""Which kernel a call of the ragged attention takes is a cost model's choice, so a test's sizes say nothing about the kernel it runs.  Two ways round that:
scripts/probes/ragged_variant_tests.py runs the edge cases through every tile and split that the measurement build can be told to take, and the calls below
have sizes that the product's own choice sends to the form they name, which they ask it for first."""
import ctypes as C
import os
import subprocess
import sys

import pytest
import torch

import _ragged_ref as ref
import test_paged_host as host
from test_gpu_paged import check_paged, cu, i32, ops, rnd  # noqa: F401  (ops: the fixture)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def choice(**kw):
    """(rows of a workgroup, parts of the key axis) of a call, from the library (no GPU needed)."""
    from fastvideo_amd import _lib
    heads = kw["H"], kw["Hkv"]
    strides = dict(q_ts=heads[0] * 128, o_ts=heads[0] * 128, k_rs=heads[1] * 128, v_rs=heads[1] * 128)
    tile, parts = C.c_int(), C.c_int()
    _lib.call("fvk_attn_ragged_choice", C.byref(host.attn_args(_lib, **{**strides, **kw})), C.byref(tile), C.byref(parts))
    return tile.value, parts.value


def paged_choice(new, before, H, Hkv, page, causal, window=0, sink=0):
    lens = [b + n for b, n in zip(before, new)]
    width = -(-max(lens) // page) + 1
    return choice(T=sum(new), R=len(new), H=H, Hkv=Hkv, max_q=max(new), max_kv=max(lens), table_width=width, page_shift=page.bit_length() - 1,
                  n_pages=sum(-(-x // page) for x in lens) + 3, k_ps=page * Hkv * 128, v_ps=page * Hkv * 128, causal=int(causal), window=window, sink=sink)


# (new tokens, cached before, heads, key heads, page, causal, window, sink), the kernel, split or not
PAGED = [(([600, 300], [1200, 40], 12, 12, 64, False), 256, True), (([600, 300], [1200, 40], 12, 4, 128, True), 256, True),
         (([300], [5000], 12, 12, 64, False), 256, True), (([1200, 700, 900], [100, 1500, 0], 12, 12, 32, False, 900, 160), 256, False),
         (([900, 37, 512, 1100], [300, 10, 0, 900], 16, 4, 16, True), 256, False), (([700, 700, 700, 700], [650] * 4, 12, 12, 256, False), 256, False),
         (([1], [900], 12, 12, 64, True), 16, True), (([1] * 32, [300] * 32, 40, 8, 64, True), 16, False)]


@pytest.mark.gpu
@pytest.mark.parametrize("case,tile,split", PAGED)
def test_paged_takes_the_kernel_and_is_right(ops, case, tile, split):
    got = paged_choice(*case)
    assert got[0] == tile and (got[1] > 1) == split, got
    check_paged(ops, 5, *case)


@pytest.mark.gpu
@pytest.mark.parametrize("new,keys", [([1500, 1400, 1600], [512, 512, 512]), ([2000, 1, 1500, 700], [0, 77, 1300, 130])])
def test_cross_takes_the_block_kernel_and_is_right(ops, new, keys):
    H, S = 12, sum(keys)
    assert choice(T=sum(new), R=len(new), H=H, Hkv=H, max_q=max(new), max_kv=max(keys), block_table=None, total_k=S)[0] == 256
    q, kv = rnd(1, sum(new), H, 128, scale=1.5), rnd(2, S, 2, H, 128)
    cq, ck = cu(new), cu(keys)
    o, lse = ops.attn_varlen(q, kv[:, 0], kv[:, 1], i32(cq), i32(ck), max_q=max(new), max_k=max(keys), return_lse=True)
    for r in range(len(new)):
        a, b = cq[r], cq[r + 1]
        want, tol, want_lse = ref.attention(q[a:b], kv[ck[r]:ck[r + 1], 0], kv[ck[r]:ck[r + 1], 1], 128**-0.5)
        assert ((o[a:b].double().cpu() - want).abs() <= tol).all(), r
        assert keys[r] == 0 or ((lse[:, a:b].double().cpu() - want_lse).abs() <= ref.LSE_TOL).all()


@pytest.mark.gpu
def test_every_kernel_tile_and_split():
    env = dict(os.environ, FVK_PROBE_LIB="1")
    r = subprocess.run([sys.executable, "-m", "pytest", os.path.join(ROOT, "scripts", "probes", "ragged_variant_tests.py"), "-x", "-q", "-p", "no:cacheprovider"],
                       cwd=ROOT, env=env, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=600)
    print(r.stdout[-3000:])
    assert r.returncode == 0 and " passed" in r.stdout and "skipped" not in r.stdout.splitlines()[-1], r.stdout[-3000:]


# ------------------------------------------------------------------ the query itself
def test_choice_refuses_what_the_call_refuses():
    from fastvideo_amd import _lib
    t, p = C.c_int(), C.c_int()
    with pytest.raises(RuntimeError, match="R=0"):
        choice(H=2, Hkv=2, R=0)
    with pytest.raises(RuntimeError, match="null pointer"):
        _lib.call("fvk_attn_ragged_choice", None, C.byref(t), C.byref(p))
    with pytest.raises(RuntimeError, match="null pointer"):
        _lib.call("fvk_attn_ragged_choice", C.byref(host.attn_args(_lib)), None, C.byref(p))


@pytest.mark.parametrize("kw", [dict(T=1, R=1, max_q=1, max_kv=900), dict(T=300, R=1, max_q=300, max_kv=8000), dict(T=4680, R=1, max_q=4680, max_kv=32760)])
def test_choice_is_the_workspace_s(kw):
    """The workspace holds the parts that the choice names: 129 numbers for each row and head."""
    from fastvideo_amd import _lib
    kw = dict(H=12, Hkv=12, table_width=600, page_shift=6, n_pages=700, k_ps=64 * 1536, v_ps=64 * 1536, q_ts=1536, o_ts=1536, k_rs=1536, v_rs=1536, **kw)
    need = _lib.load().fvk_attn_ragged_workspace_bytes(C.byref(host.attn_args(_lib, **kw)))
    parts = choice(**kw)[1]
    assert need == (parts * kw["T"] * 12 * 129 * 4 if parts > 1 else 0)


@pytest.mark.parametrize("case,tile,split", PAGED)
def test_the_named_cases_still_take_their_kernel(case, tile, split):
    got = paged_choice(*case)
    assert got[0] == tile and (got[1] > 1) == split, got
