#!/bin/bash
# Round-5 GPU sessions (one gpurun call each): tools/gpu_r5.sh <stage> [budget seconds]
cd "$(dirname "$0")/.."
mkdir -p gpurun_out
STAGE=${1:-perf1}
BUDGET=${2:-780}
export TMPDIR=/tmp
T0=$(date +%s)
left() { echo $(( BUDGET - ($(date +%s) - T0) )); }
PYT="python -m pytest -q --no-header --tb=short -p no:cacheprovider --timeout=900 --maxfail=30 -m gpu"
run() { # name, timeout, command...
  local name=$1 to=$2; shift 2
  echo "=== $name ===" | tee -a gpurun_out/session.log
  local t0=$(date +%s)
  timeout $to "$@" > gpurun_out/$name.log 2>&1
  echo "exit=$? $(( $(date +%s) - t0 ))s $(tail -n 1 gpurun_out/$name.log | cut -c1-300)" | tee -a gpurun_out/session.log
}
rm -f gpurun_out/parity.jsonl gpurun_out/session.log
rocminfo 2>/dev/null | grep -E "gfx|Compute Unit" | head -2 >> gpurun_out/session.log
case $STAGE in
perf1)  # round-5 norm kernels (LayerNorm lane groups, GroupNorm two-pass merge): parity first, then per-op and whole-step A/B; the default
  # bench line with the SDXL child (first run of that path); the self-attention mask and the refusal tests
  run t_norm 900 $PYT tests/test_ops_gpu.py -k "group_norm or layer_norm or gn_ or gnstats or stats or fused_groupnorm"
  run t_reftriton 900 $PYT tests/test_ref_triton_gpu.py -k "group_norm or layer_norm"
  run t_unet 900 $PYT tests/test_unet_gpu.py -k "tiny or sd15_unet_parity or attention_mask or isolation or controlnet"
  run micro_new 200 python tools/micro_norm.py
  SFAST_GN_MERGE=chain SFAST_LN_GROUP=0 run micro_old 200 python tools/micro_norm.py
  AB="python bench.py --steps 100 --warmup 10 --no-cpu-baseline --no-end-to-end --no-variants --no-roofline"
  for i in 1 2; do
    run ab_new$i 300 $AB
    SFAST_GN_MERGE=chain SFAST_LN_GROUP=0 run ab_old$i 300 $AB
  done
  for f in ab_new1 ab_old1 ab_new2 ab_old2; do echo "$f $(grep -a -o '"value": [0-9.]*' gpurun_out/$f.log | head -1) $(grep -a -o '"ms_per_step": [0-9.]*' gpurun_out/$f.log | head -1)" >> gpurun_out/session.log; done
  [ $(left) -gt 200 ] && run bench_default 400 python bench.py
  ;;
final3)  # the default bench line FIRST on a fresh box (two final2 sessions in a row measured 150 it/s where every other session of the round
  # measured 180 - 184: is it the box, or what ran before?), then --kernel-trace-only passes (no counters) for the per-symbol durations
  run bench_default 300 python bench.py --dump-kernels gpurun_out/kernels.json
  for cfg in sd15 sdxl; do
    [ $(left) -lt 60 ] && break
    ( cd /tmp && timeout 200 rocprofv3 --kernel-trace -d $OLDPWD/gpurun_out/prof_$cfg -o trace -- python $OLDPWD/bench.py --config $cfg --steps 8 --warmup 2 --no-cpu-baseline --no-roofline --no-end-to-end --no-variants > $OLDPWD/gpurun_out/trace_$cfg.log 2>&1 )
    for db in $(find gpurun_out/prof_$cfg -name "*.db"); do python tools/rocpd_summary.py $db --csv gpurun_out/trace_$cfg.csv --top 200 --step-marker cfg_ddim --steps 6 > gpurun_out/trace_$cfg.txt; done
    rm -rf gpurun_out/prof_$cfg
    echo "trace $cfg: $(head -1 gpurun_out/trace_$cfg.txt)" >> gpurun_out/session.log
  done
  [ $(left) -gt 40 ] && run bench_sdxl 200 python bench.py --config sdxl --no-cpu-baseline --no-variants --dump-kernels gpurun_out/kernels_sdxl.json
  [ $(left) -gt 30 ] && run bench_images8 200 python bench.py --images 8 --steps 50 --warmup 10 --no-cpu-baseline --no-end-to-end --no-variants --no-roofline
  [ $(left) -gt 130 ] && run bench_svd 300 python bench.py --config svd --no-cpu-baseline
  ;;
final2)  # the PMC passes again without the variants (first attempt: B = 1 autotuning under counters), then the lines that did not fit
  run pmc_sd15 400 bash tools/gpu_pmc_bench.sh sd15 6
  cp gpurun_out/pmcb/traffic_by_symbol.json profiles/r05_pmc_traffic_by_symbol.json && cp gpurun_out/pmcb/traffic_by_symbol.json gpurun_out/r05_pmc_traffic_by_symbol.json
  run bench_default 400 python bench.py --dump-kernels gpurun_out/kernels.json
  run pmc_sdxl 330 bash tools/gpu_pmc_bench.sh sdxl 4
  cp gpurun_out/pmcb/traffic_by_symbol_sdxl.json profiles/r05_pmc_traffic_by_symbol_sdxl.json && cp gpurun_out/pmcb/traffic_by_symbol_sdxl.json gpurun_out/r05_pmc_traffic_by_symbol_sdxl.json
  rm -rf gpurun_out/pmcb
  [ $(left) -gt 60 ] && run bench_sdxl 300 python bench.py --config sdxl --no-cpu-baseline --no-variants --dump-kernels gpurun_out/kernels_sdxl.json
  [ $(left) -gt 150 ] && run bench_svd 400 python bench.py --config svd --no-cpu-baseline
  [ $(left) -gt 60 ] && run bench_torchrun 300 python -m torch.distributed.run --nnodes=1 --nproc-per-node 1 --master-addr 127.0.0.1 --master-port 29544 bench.py --gpus 1 --steps 50 --warmup 10 --no-cpu-baseline --no-roofline --no-end-to-end --no-variants
  [ $(left) -gt 50 ] && run bench_images8 300 python bench.py --images 8 --steps 50 --warmup 10 --no-cpu-baseline --no-end-to-end --no-variants --no-roofline
  ;;
final)  # the round's evidence set on HEAD, most important first; SFAST_COMMIT=<sha> in the environment names the commit in the PMC files
  run pytest_full 1500 $PYT tests
  cp gpurun_out/parity.jsonl gpurun_out/parity_full.jsonl 2>/dev/null
  run smoke 300 python __graft_entry__.py smoke
  # PMC traffic by symbol (separate --pmc passes, packaged kernel choices): copied into profiles/ on this box so that the bench lines of this
  # session already quote them (the same files come back through gpurun_out/)
  run pmc_sd15 900 bash tools/gpu_pmc_bench.sh sd15 6
  cp gpurun_out/pmcb/traffic_by_symbol.json profiles/r05_pmc_traffic_by_symbol.json && cp gpurun_out/pmcb/traffic_by_symbol.json gpurun_out/r05_pmc_traffic_by_symbol.json
  for f in fetch write; do cp gpurun_out/pmcb/$f.log gpurun_out/pmc_sd15_$f.log 2>/dev/null; done
  if [ $(left) -gt 700 ]; then
    run pmc_sdxl 900 bash tools/gpu_pmc_bench.sh sdxl 4
    cp gpurun_out/pmcb/traffic_by_symbol_sdxl.json profiles/r05_pmc_traffic_by_symbol_sdxl.json && cp gpurun_out/pmcb/traffic_by_symbol_sdxl.json gpurun_out/r05_pmc_traffic_by_symbol_sdxl.json
  fi
  rm -rf gpurun_out/pmcb
  run bench_default 600 python bench.py --dump-kernels gpurun_out/kernels.json
  ( cd /tmp && timeout 600 rocprofv3 --kernel-trace --stats -d $OLDPWD/gpurun_out/prof -o bench -- python $OLDPWD/bench.py --steps 20 --warmup 5 --no-cpu-baseline --no-roofline --no-end-to-end --no-variants > $OLDPWD/gpurun_out/rocprof.log 2>&1 )
  echo "rocprof exit=$?" >> gpurun_out/session.log
  for db in $(find gpurun_out/prof -name "*.db"); do python tools/rocpd_summary.py $db --csv gpurun_out/kernel_stats.csv --top 60 --step-marker cfg_ddim --steps 12 > gpurun_out/kernel_stats.txt; done
  rm -rf gpurun_out/prof
  [ $(left) -gt 300 ] && run bench_sdxl 600 python bench.py --config sdxl --no-cpu-baseline --dump-kernels gpurun_out/kernels_sdxl.json
  [ $(left) -gt 300 ] && run bench_svd 900 python bench.py --config svd --no-cpu-baseline
  [ $(left) -gt 150 ] && run bench_torchrun 600 python -m torch.distributed.run --nnodes=1 --nproc-per-node 1 --master-addr 127.0.0.1 --master-port 29544 bench.py --gpus 1 --steps 50 --warmup 10 --no-cpu-baseline --no-roofline --no-end-to-end --no-variants
  [ $(left) -gt 120 ] && run bench_images8 600 python bench.py --images 8 --steps 50 --warmup 10 --no-cpu-baseline --no-end-to-end --no-variants --no-roofline
  ;;
esac
cat gpurun_out/session.log
