#!/bin/bash
# GPU test files under the guard-page device allocator (scripts/probes/guard_alloc.cpp, tests/_guard.py): one process per file, an unmapped page behind
# every tensor.  Every file is expected to pass; the sweep ends at the first that does not, and what it printed and the code are read then.
# Earlier runs: profiles/r06d_guard_page_runs.md.
set -u
cd "${GRAFT_REPO_ROOT:-/root/repo}"
OUT=gpurun_out/guard_sweep; mkdir -p $OUT
timeout -k 10 300 python scripts/guard_selftest.py > $OUT/selftest.log 2>&1; rc=$?; echo "selftest rc=$rc $(tail -1 $OUT/selftest.log)"; [ $rc -eq 0 ] || exit $rc
for T in tests/test_gpu_kernels.py tests/test_gpu_model.py tests/test_gpu_sp.py tests/test_gpu_fullgeom.py tests/test_gpu_fp8.py tests/test_gpu_sched.py \
         tests/test_gpu_causal.py tests/test_gpu_loader.py tests/test_gpu_reference_model.py tests/test_gpu_vae.py tests/test_gpu_vae_tiled.py \
         tests/test_gpu_vae_real.py tests/test_gpu_boundary.py tests/test_gpu_ref_triton.py tests/test_gpu_fullsize.py tests/test_gpu_rccl_single_rank.py; do
  [ -f $T ] || continue
  N=$(basename $T .py)
  FVK_GUARD_ALLOC=1 timeout -k 10 1500 python -m pytest $T -x -q > $OUT/$N.log 2>&1; rc=$?; echo "guard $T rc=$rc $(tail -1 $OUT/$N.log | cut -c1-150)"; [ $rc -eq 0 ] || exit $rc
done
FVK_GUARD_ALLOC=1 FVK_GUARD_MODE=front timeout -k 10 900 python -m pytest tests/test_gpu_kernels.py tests/test_gpu_ref_triton.py -x -q > $OUT/front.log 2>&1
rc=$?; echo "front placement rc=$rc $(tail -1 $OUT/front.log | cut -c1-150)"; exit $rc
