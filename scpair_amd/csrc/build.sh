#!/bin/bash
# Builds libscpair_hip.so and _trunk.so for gfx950 in-tree (cross-compiles without a GPU): what is older than its sources, its
# flags or (for _trunk.so) the torch it was compiled against.  --all: everything; --stale: only names what would be built.
set -e
ALL=; STALE=
case "$1" in --all) ALL=1;; --stale) STALE=1;; "") ;; *) echo "usage: build.sh [--all | --stale]" >&2; exit 2;; esac
HERE="$(cd "$(dirname "$0")" && pwd)"
ROOT="$(cd "$HERE/../.." && pwd)"
OUT="$HERE/../libscpair_hip.so"
HIPCC=${HIPCC:-/opt/rocm/bin/hipcc}
# -packed-fp32-ops: no v_pk_{add,mul,fma}_f32, some of whose forms have given wrong results now and then on this hardware
FLAGS="--offload-arch=gfx950 -O3 -fPIC -std=c++17 -Xclang -target-feature -Xclang -packed-fp32-ops -Wno-unused-result $EXTRA_FLAGS"
HOW="$HIPCC $FLAGS"
FLAGS="$FLAGS -I$ROOT/include -I$HERE"
OBJ="$HERE/build"
mkdir -p "$OBJ"
# older TARGET SOURCE...: the target is missing or older than one of its sources
older() {
  local t="$1" s
  shift
  [ -n "$ALL" ] && return 0
  for s in "$@"; do [ "$s" -nt "$t" ] && return 0; done
  return 1
}
# differs FILE TEXT: the file does not hold the text
differs() { [ "$(cat "$1" 2>/dev/null)" != "$2" ]; }
differs "$OBJ/flags" "$HOW" && [ -z "$STALE" ] && ALL=1
pids=()
for f in capi gemm wgemm spmm_bf16 tiles norm_act enc_tail adamw elementwise raw_rows residual_norm ckpt8 linear8 eval_metrics decoder decoder_ber_ns1 decoder_ber_ns3 decoder_nb_ns1 decoder_nb_ns3; do
  if older "$OBJ/$f.o" "$HERE/$f.hip" "$HERE/build.sh" "$HERE/common.h" "$HERE/ckpt8.h" "$HERE/decoder_kernel.h" "$ROOT/include/scpair_hip.h" ||
     differs "$OBJ/flags" "$HOW"; then
    if [ -n "$STALE" ]; then echo "$f.o"; continue; fi
    $HIPCC $FLAGS -c "$HERE/$f.hip" -o "$OBJ/$f.o" &
    pids+=($!)
  fi
done
for p in "${pids[@]}"; do wait $p; done
if [ -z "$STALE" ]; then
  echo "$HOW" > "$OBJ/flags"
  rm -f "$OBJ/libgemm.o"
  $HIPCC --offload-arch=gfx950 -shared -fPIC -o "$OUT" "$OBJ"/*.o
  echo "built $OUT"
fi
# autograd nodes of the residual-trunk operators: host code against torch's headers, launches through the library above
EXT="$HERE/../_trunk.so"
read -r TORCH VERSION PYINC <<< "$(python3 -c 'import os, sysconfig, torch; print(os.path.dirname(torch.__file__), torch.__version__, sysconfig.get_paths()["include"])')"
AGAINST="$TORCH $VERSION $PYINC"
if older "$EXT" "$HERE/trunk_binding.cpp" "$HERE/build.sh" "$ROOT/include/scpair_hip.h" || differs "$OBJ/torch" "$AGAINST"; then
  if [ -n "$STALE" ]; then echo "_trunk.so"; exit 0; fi
  g++ -O2 -std=c++17 -fPIC -shared -D__HIP_PLATFORM_AMD__=1 -DUSE_ROCM=1 -I"$ROOT/include" -isystem "$TORCH/include" \
    -isystem "$TORCH/include/torch/csrc/api/include" -isystem /opt/rocm/include -isystem "$PYINC" "$HERE/trunk_binding.cpp" -o "$EXT" \
    -L"$HERE/.." -l:libscpair_hip.so -L"$TORCH/lib" -ltorch_python -ltorch -ltorch_cpu -lc10 -lc10_hip -Wl,-rpath,'$ORIGIN'
  echo "$AGAINST" > "$OBJ/torch"
  echo "built $EXT"
fi
[ -n "$STALE" ] && exit 0
# benchmark-only comparison library (rocBLAS bf16 GEMM beside the hand-written wide GEMM): not part of the product
CMP="$ROOT/benchmarks/rocblas_cmp"
if [ "$CMP/rocblas_cmp.hip" -nt "$CMP/librocblas_cmp.so" ]; then
  $HIPCC --offload-arch=gfx950 -O2 -fPIC -shared -o "$CMP/librocblas_cmp.so" "$CMP/rocblas_cmp.hip" -L/opt/rocm/lib -lrocblas -Wl,-rpath,/opt/rocm/lib
  echo "built $CMP/librocblas_cmp.so"
fi
