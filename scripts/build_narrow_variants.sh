#!/bin/bash
# usage: scripts/build_narrow_variants.sh NAME "-DFLAG=1 ..." [NAME "-D..."]...  -> build/variants/librag_hip_NAME.so
# (only narrow_topk.hip is rebuilt; the other objects come from rag_amd/csrc as built by the Makefile)
set -e
cd "$(dirname "$0")/.."
mkdir -p build/variants
while [ $# -ge 2 ]; do
  name=$1; flags=$2; shift 2
  (
    /opt/rocm/bin/hipcc -O3 -std=c++17 -fPIC --offload-arch=gfx950 -ffp-contract=off -Xclang -target-feature -Xclang -packed-fp32-ops $flags -c rag_amd/csrc/narrow_topk.hip -o build/variants/narrow_$name.o
    objs=$(ls rag_amd/csrc/*.o | grep -v narrow_topk.o)
    /opt/rocm/bin/hipcc --offload-arch=gfx950 -shared -fPIC $objs build/variants/narrow_$name.o -o build/variants/librag_hip_$name.so
    echo built $name
  ) &
done
wait
