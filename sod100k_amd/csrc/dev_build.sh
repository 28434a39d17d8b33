#!/bin/bash
# Developer build: libcsnet_hip.so for gfx950 with per-kernel resource usage and ISA kept in $OUT (default /tmp/csn_build).
# The product build recipe is sod100k_amd/_native.py:build() (same flags without the diagnostics).
set -e
HERE="$(cd "$(dirname "$0")" && pwd)"
OUT="${OUT:-/tmp/csn_build}"
mkdir -p "$OUT"
cd "$OUT"
# the build id the loader checks (csn_build_sources_sha16, include/csnet_hip.h): the unit sod100k_amd/_native.py generates
python3 -c "import sys; sys.path.insert(0, '$HERE/../..'); from sod100k_amd import _native as N; N.write_build_id_object(N.hipcc_path(), N.sources_sha16(), '$OUT')"
# sources and flags of the product build; linked aside, so that a failed build leaves the library in the tree alone
py() { python3 -c "import sys; sys.path.insert(0, '$HERE/../..'); from sod100k_amd import _native as N; print(*$1)"; }
FLAGS=$(py N.HIPCC_FLAGS)
objs=""; jobs=""
for s in $(py N.SOURCES); do
  hipcc $FLAGS -Rpass-analysis=kernel-resource-usage -save-temps=obj -I"$HERE" -c "$HERE/$s" -o "$OUT/${s%.hip}.o" > "$OUT/${s%.hip}.log" 2>&1 &
  jobs="$jobs $!"; objs="$objs $OUT/${s%.hip}.o"
done
failed=0
for j in $jobs; do wait $j || failed=1; done
cat "$OUT"/*.log > "$OUT/build.log.new"; mv "$OUT/build.log.new" "$OUT/build.log"
if [ $failed = 0 ]; then
  hipcc --offload-arch=gfx950 -shared -Wl,--no-undefined -o "$OUT/libcsnet_hip.so" $objs "$OUT/csn_build_id.o" >> "$OUT/build.log" 2>&1 || failed=1
fi
[ $failed = 0 ] || { grep -E "error|undefined" -A3 "$OUT/build.log" | head -40; exit 1; }
cp "$OUT/libcsnet_hip.so" "$HERE/libcsnet_hip.so.new" && mv "$HERE/libcsnet_hip.so.new" "$HERE/libcsnet_hip.so"
python3 - "$OUT/build.log" <<'PY'
import re, sys
txt = open(sys.argv[1]).read()
rows = []
cur = {}
for line in txt.splitlines():
    m = re.search(r"Function Name: (\S+)", line)
    if m:
        cur = {"name": m.group(1)}
        rows.append(cur)
    for key, pat in (("sgpr", r"TotalSGPRs: (\d+)"), ("vgpr", r" VGPRs: (\d+)"), ("scratch", r"ScratchSize \[bytes/lane\]: (\d+)"),
                     ("occ", r"Occupancy \[waves/SIMD\]: (\d+)"), ("lds", r"LDS Size \[bytes/block\]: (\d+)")):
        m = re.search(pat, line)
        if m and cur is not None:
            cur[key] = m.group(1)
print(f"{'kernel':60s} {'sgpr':>5s} {'vgpr':>5s} {'scr':>5s} {'occ':>4s}")
for r in rows:
    print(f"{r['name'][:60]:60s} {r.get('sgpr','?'):>5s} {r.get('vgpr','?'):>5s} {r.get('scratch','?'):>5s} {r.get('occ','?'):>4s}")
PY
