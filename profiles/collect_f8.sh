#!/bin/bash
# Kernel times and counters of the 8-bit row operators (tools/prof_f8.py), each in a run of its own; raw output under $1,
# profiles/summarize_f8.py writes profiles/f8_kernels.json from it.
set -e
export TMPDIR=/tmp
OUT=${1:?folder for the raw output}
mkdir -p $OUT
stats() { timeout -s KILL 120 rocprofv3 --output-format csv --kernel-trace --stats -d $OUT/stats_$1 -o k -- python3 tools/prof_f8.py ${@:2} > $OUT/stats_$1.log 2>&1; echo "$1"; }
pmc() { for C in "FETCH_SIZE" "WRITE_SIZE" "SQ_VALU_MFMA_BUSY_CYCLES GRBM_GUI_ACTIVE"; do
  timeout -s KILL 120 rocprofv3 --output-format csv --pmc $C -d $OUT/pmc_$1_${C%% *} -o k -- python3 tools/prof_f8.py ${@:2} > $OUT/pmc_$1.log 2>&1; done; echo "$1 counters"; }
stats norm_32768x4096 norm 32768 4096 bf16 1 0
stats norm_200000x2048 norm 200000 2048 f32 0 1
stats quantise_200000x2048 quantise 200000 2048 f32
stats product_1x4096x4096 product 1 4096 4096
stats product_48x12288x4096 product 48 12288 4096
stats product_512x4096x4096 product 512 4096 4096
stats product_8192x8192x8192 product 8192 8192 8192
stats search_10000x4096_1 search 10000 4096 1 10
stats search_10000x4096_64 search 10000 4096 64 10
stats search_1000000x4096_1 search 1000000 4096 1 10
stats search_1000000x4096_64 search 1000000 4096 64 10
stats search_1000000x4096_1024 search 1000000 4096 1024 10
stats search_1000000x4096_1024_k100 search 1000000 4096 1024 100
stats search_1000000x4096_1024_strong search 1000000 4096 1024 10 0.98
pmc product_8192x8192x8192 product 8192 8192 8192
pmc search_1000000x4096_1 search 1000000 4096 1 10
pmc search_1000000x4096_1024 search 1000000 4096 1024 10
echo done
