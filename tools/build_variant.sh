#!/bin/bash
# build_variant.sh <name> <source.hip> "<extra flags>": libmgnet_hip.so with ONE source compiled with extra flags -> ablib/libmgnet_hip_<name>.so
set -e
cd "$(dirname "$0")/.."
name=$1; src=$2; flags=$3
HIPCC=${HIPCC:-/opt/rocm/bin/hipcc}
mkdir -p ablib/obj_$name
base=$(basename $src .hip)
CF=$(python3 -m mgnet_amd.build --flags)   # (the library's own: no packed fp32, launches through the recorder)
$HIPCC $CF $flags -c mgnet_amd/csrc/$base.hip -o ablib/obj_$name/$base.o
objs=""
for o in mgnet_amd/lib/obj/*.o; do
  b=$(basename $o)
  if [ "$b" == "$base.o" ]; then objs="$objs ablib/obj_$name/$base.o"; elif [ "$b" == "${base}_f16.o" ] && [ -f mgnet_amd/csrc/${base}_f16.hip ]; then
    $HIPCC $CF $flags -c mgnet_amd/csrc/${base}_f16.hip -o ablib/obj_$name/${base}_f16.o; objs="$objs ablib/obj_$name/${base}_f16.o"
  else objs="$objs $o"; fi
done
$HIPCC --offload-arch=gfx950 -shared -fPIC $objs -o ablib/libmgnet_hip_$name.so
echo ablib/libmgnet_hip_$name.so
