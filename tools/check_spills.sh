#!/bin/bash
# Lists VGPR count, scratch bytes and spill count of every kernel in magvit2_pytorch_amd/csrc (gfx950 ISA, no GPU
# needed), and how many 64-bit shifts by an amount in a vector register a file holds.  A non-zero scratch / spill column on a hot kernel is a bug,
# and so is such a shift: with its amount in a wave's last register it has given wrong results on these chips.
# usage: tools/check_spills.sh [file.hip ...]        (default: the product sources)
cd "$(dirname "$0")/../magvit2_pytorch_amd/csrc" || exit 1
T=$(mktemp -d)
for f in ${@:-conv3p.hip conv3.hip convin.hip convout.hip pwse.hip ff.hip conv.hip misc.hip attn.hip quant.hip gateloop.hip blocknorm.hip}; do
  b=$(basename "$f" .hip)
  hipcc -O3 -std=c++17 -Xclang -target-feature -Xclang -packed-fp32-ops --offload-arch=gfx950 --cuda-device-only -S -I../../include "$b.hip" -o "$T/$b.s" 2>/dev/null || { echo "$b: compile failed"; continue; }
  grep "\.name: \+_Z\|private_segment_fixed_size\|\.vgpr_count\|vgpr_spill" "$T/$b.s" |
    awk -v F="$b" '/\.name:/{n=$2} /private_segment_fixed_size/{p=$2} /\.vgpr_count/{v=$2} /vgpr_spill/{printf "%-12s %-105s vgpr=%-4s scratch=%-6s spills=%s\n", F, substr(n,1,105), v, p, $2}'
  echo "$b: $(grep -cE 'v_(lsh[lr]|ash?r)rev_[bi]64 v\[[0-9:]+\], v[0-9]' "$T/$b.s") variable 64-bit shifts"
done
rm -rf "$T"
