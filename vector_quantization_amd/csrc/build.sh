#!/bin/bash
# Builds libvqhip.so for gfx950 (MI355X) in-tree.  hipcc cross-compiles without a GPU.  Extra arguments go to hipcc.
# (The packed fp32 instructions are switched off for all device code: some of their forms are not reliable.)
set -e
HERE="$(cd "$(dirname "$0")" && pwd)"
LIB="$HERE/../lib"
mkdir -p "$LIB"
FLAGS=(-O3 -std=c++17 --offload-arch=gfx950 -fPIC -ffp-contract=off -Xclang -target-feature -Xclang -packed-fp32-ops
       -I"$HERE/../../include" "$@")
# objects of this run only, so that two builds at once do not mix
OBJ="$(mktemp -d)"
trap 'rm -rf "$OBJ"' EXIT
/opt/rocm/bin/hipcc "${FLAGS[@]}" -c "$HERE/vq_hip.hip" -o "$OBJ/vq_hip.o" &
FIRST=$!
/opt/rocm/bin/hipcc "${FLAGS[@]}" -c "$HERE/vq_cache.hip" -o "$OBJ/vq_cache.o"
wait $FIRST
/opt/rocm/bin/hipcc --offload-arch=gfx950 -shared -fPIC "$OBJ/vq_hip.o" "$OBJ/vq_cache.o" -o "$LIB/libvqhip.so"
