#!/bin/bash
# Session Q (PDMB_EXPERIMENTS=1 build in the tree): the lean exact-fp32
# W4 K-loop (x_f32_w4_lean2), the settled A/B against the auto kernel
# (f32_t128x2) and hipBLASLt on the full grids, two sessions; then PMC at 16k.
# (The streamed kernel this session also ran is not launched any more.)
set -o pipefail
cd "$GRAFT_REPO_ROOT" || exit 1
export TMPDIR=/tmp PDMB_EXPERIMENTS=1
OUT=gpurun_out/r8q; mkdir -p $OUT
timeout -k 10 900 python -m pytorch_distributed_matmul_benchmark_amd.ops.build --no-bench -v > $OUT/build.log 2>&1 || exit $?
KS=x_f32_w4_lean2,f32_t128x2
echo "== fp32 lean A/B $(date +%T)"
timeout -k 10 900 python scripts/ab_kernels.py --dtype float32 --rounds 3 --iters 5 --settle 1 --sessions 2 \
  --kernels $KS,torch --shapes 16384,16384,16384 8192,8192,8192 4096,4096,4096 \
  > $OUT/ab_f32_lean2.jsonl 2> $OUT/ab_f32_lean2.err || exit $?
grep '"summary"' $OUT/ab_f32_lean2.jsonl | cut -c1-200
echo "== pmc $(date +%T)"
DT=float32 N=16384 KS=$KS REPS=3 OUT=$OUT/pmc \
  timeout -k 10 900 bash scripts/gpu_pmc.sh > $OUT/pmc.log 2>&1 || exit $?
python scripts/pmc_summary.py $OUT/pmc --cycle $KS,torch
echo "exit 0"
