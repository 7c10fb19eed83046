#!/bin/bash
# Builds libligdiff.so for gfx950 next to the sources (in-tree, travels to the GPU box).
set -e
cd "$(dirname "$0")"
# no packed fp32 arithmetic (v_pk_add / mul / fma_f32, which -O3 makes from ordinary float code): some of its forms have given
# wrong results on this hardware.  (The host pass does not know the feature and says so.)
FLAGS="--offload-arch=gfx950 -O3 -std=c++17 -fPIC -Wall -Wno-unused-function -Xclang -target-feature -Xclang -packed-fp32-ops"
pids=()
for f in chain_dit_mol_heads chain_dit_mol chain_dit_row_heads chain_dit_row forward backward chain_e3 sampler api pack loss consistency optim embed tokens; do
  if [ -f $f.hip ]; then
    MORE=""
    # constants of the per-row 64-bit part are not hoisted into registers for the whole row loop (k_token_rows: 20 to 30
    # registers, two waves a SIMD)
    case $f in embed|tokens) MORE="-mllvm -disable-machine-licm" ;; esac
    hipcc $FLAGS $MORE -c $f.hip -o $f.o &
    pids+=($!)
  fi
done
for p in "${pids[@]}"; do wait $p; done
hipcc --offload-arch=gfx950 -shared -fPIC -o ../libligdiff.so *.o
echo built ../libligdiff.so
