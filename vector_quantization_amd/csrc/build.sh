#!/bin/bash
# Builds libvqhip.so for gfx950 (MI355X) in-tree.  hipcc cross-compiles without a GPU.  Extra arguments go to hipcc.
# (The packed fp32 instructions are switched off for all device code: some of their forms are not reliable.)
set -e
HERE="$(cd "$(dirname "$0")" && pwd)"
LIB="$HERE/../lib"
mkdir -p "$LIB"
FLAGS=(-O3 -std=c++17 --offload-arch=gfx950 -fPIC -ffp-contract=off -Xclang -target-feature -Xclang -packed-fp32-ops
       -I"$HERE/../../include" "$@")
# objects of this run only, so that two builds at once do not mix; by relative names, so that the same sources give the same library
OBJ="$(mktemp -d)"
cd "$OBJ"
trap 'rm -rf "$OBJ"' EXIT
PIDS=()
compile() {  # source, object, further flags.  (The host pass says of the device's feature that it does not know it; the rest is shown.)
    /opt/rocm/bin/hipcc "${FLAGS[@]}" "${@:3}" -c "$HERE/$1" -o "$2" 2> >(grep -vF "'-packed-fp32-ops' is not a recognized feature" >&2) &
    PIDS+=($!)
}
compile vq_hip.hip vq_hip.o
compile vq_cache.hip vq_cache.o
compile vq_cache_search.hip vq_cache_search.o
compile vq_cache_attend.hip vq_cache_attend_bf16.o -DVQ_CACHE_TYPE=__bf16 -DVQ_CACHE_ATTEND=vq_internal_attend_bf16
compile vq_cache_attend.hip vq_cache_attend_f16.o -DVQ_CACHE_TYPE=_Float16 -DVQ_CACHE_ATTEND=vq_internal_attend_f16
for pid in "${PIDS[@]}"; do wait "$pid"; done
/opt/rocm/bin/hipcc --offload-arch=gfx950 -shared -fPIC *.o -o "$LIB/libvqhip.so"
