#!/usr/bin/env bash
# Build libgwn.so (HIP, gfx950) in-tree.  Used by __graft_entry__.build() and by hand.
#   OUT=<path> EXTRA="-DFOO=1" ./build.sh    builds an experiment variant elsewhere
# Each source compiles to its own object in parallel (JOBS, default 8), then one link.
set -euo pipefail
ROOT="$(cd "$(dirname "$0")" && pwd)"
SRC="$ROOT/graph-wavenet_amd/csrc"
OUT="${OUT:-$ROOT/graph-wavenet_amd/gwn_amd/libgwn.so}"
HIPCC="${HIPCC:-/opt/rocm/bin/hipcc}"
# No packed fp32 VALU ops (v_pk_mul_f32 / v_pk_add_f32 / v_pk_fma_f32) in any kernel: with them, hipcc 7.2's gfx950
# code for the bf16 pair backward's gate epilogue overwrote a packed op's source register while the
# op still read it (lanes 48-63), and some dfg values came out wrong, different run to run
# (tools/exp/bwd_pair_probe.py: 30-330 of 34M elements per run; none without packed ops).  The flag
# reaches the host compile too, which ignores it (its warning is filtered below).
NOPK="-Xclang -target-feature -Xclang -packed-fp32-ops"
FLAGS="--offload-arch=gfx950 -O3 -std=c++17 -fPIC -Wall -Wno-unused-result $NOPK ${EXTRA:-} -I$ROOT/include"
OBJ="$(mktemp -d)"
trap 'rm -rf "$OBJ"' EXIT
pids=()
for f in gemm gemm_nt ops gcn_fused gcn_slice supports rowgemm gram wgrad wgrad_group infer bigdiff linear layernorm dropout; do
  ( "$HIPCC" $FLAGS -c -o "$OBJ/$f.o" "$SRC/$f.hip" 2>&1 | { grep -v "packed-fp32-ops' is not a recognized feature" || true; } ) &
  pids+=($!)
  while [ "$(jobs -rp | wc -l)" -ge "${JOBS:-8}" ]; do sleep 0.2; done
done
for p in "${pids[@]}"; do wait "$p"; done
"$HIPCC" --offload-arch=gfx950 -shared -fPIC -o "$OUT.tmp" "$OBJ"/*.o
mv "$OUT.tmp" "$OUT"
echo "built $OUT"
