#!/bin/bash
# Build libvid2seq_hip.so for gfx950 (cross-compiles without a GPU).  Usage: build.sh [-B]   (-B: compile every source again)
set -e
cd "$(dirname "$0")"
[ "$1" = "-B" ] && rm -rf build
HIPCC=${HIPCC:-/opt/rocm/bin/hipcc}
# -munsafe-fp-atomics: hardware float atomics (global_atomic_add_f32 / ds_add_f32) instead of CAS loops; all our
# atomics target ordinary (coarse-grained) device memory, where they are exact fp32 adds
FLAGS="--offload-arch=gfx950 -O3 -std=c++17 -fPIC -Wno-unused-result -munsafe-fp-atomics"
# no packed fp32 arithmetic (v_pk_{add,mul,fma}_f32), which the compiler would form from ordinary float code; the one-lane instructions round the same way, so
# results do not depend on it (the host pass warns that it does not know the feature)
FLAGS="$FLAGS -Xclang -target-feature -Xclang -packed-fp32-ops"
SRCS="v2s_api v2s_gemm v2s_norm v2s_attn v2s_misc v2s_optim v2s_decode v2s_memattn v2s_data v2s_q8 v2s_gemm_q8 v2s_sample"
mkdir -p build
# the hand-scheduled K loop of gemm_a4_kernel is generated (scoreboarded s_waitcnt counts, MFMA-gap placement): see gen_gemm_a4.py
if [ ! -f v2s_gemm_a4.inc ] || [ gen_gemm_a4.py -nt v2s_gemm_a4.inc ]; then
  python3 gen_gemm_a4.py v2s_gemm_a4.inc
fi
pids=()
for s in $SRCS; do
  if [ ! -f build/$s.o ] || [ $s.hip -nt build/$s.o ] || [ v2s_common.h -nt build/$s.o ] || [ ../../include/vid2seq_hip.h -nt build/$s.o ] ||
     { [ $s = v2s_gemm ] && { [ v2s_gemm_a4.h -nt build/$s.o ] || [ v2s_gemm_a4.inc -nt build/$s.o ]; }; }; then
    ( $HIPCC $FLAGS -c $s.hip -o build/$s.o ) &
    pids+=($!)
  fi
done
for p in "${pids[@]}"; do wait $p; done
# The persistent deferred-epilogue GEMM counts its VMEM operations by hand (s_waitcnt vmcnt(N) across barriers): a register spill would
# add scratch loads/stores to that queue.  Fail the build if the compiler ever needs scratch for it.
if [ build/v2s_gemm.o -nt build/v2s_gemm.usage ] || [ ! -f build/v2s_gemm.usage ]; then
  $HIPCC $FLAGS -c v2s_gemm.hip -o /dev/null -Rpass-analysis=kernel-resource-usage 2> build/v2s_gemm.usage.raw || true
  grep -A8 "Function Name: .*gemm_p8d_kernel" build/v2s_gemm.usage.raw | grep -E "Function Name|ScratchSize" > build/v2s_gemm.usage || true
  if grep -E "ScratchSize \[bytes/lane\]: [1-9]" build/v2s_gemm.usage; then
    echo "ERROR: gemm_p8d_kernel spills to scratch (see build/v2s_gemm.usage): its hand-counted vmcnt waits would be wrong" >&2
    rm -f build/v2s_gemm.o; exit 1
  fi
  # no GEMM kernel is meant to touch scratch (an accumulator array indexed by a rolled loop, a pointer select between a register
  # value and memory: both have happened) -- say so loudly, the kernels stay correct but lose 10-30 %
  grep -E "Function Name|ScratchSize" build/v2s_gemm.usage.raw | paste - - | grep -vE "lane\]: 0 " | sed 's/.*Function Name: \([^ ]*\).*lane\]: \([0-9]*\).*/WARNING: \1 uses \2 bytes of scratch per lane/' >&2 || true
fi
# gemm_a4_kernel keeps its 256 accumulators in LITERAL AGPRs across asm statements: any v_accvgpr_* / scratch access the compiler
# emits on its own inside that kernel could only be a spill into them.  Audit the ISA (everything outside ;;#ASMSTART .. ;;#ASMEND).
if [ build/v2s_gemm.o -nt build/v2s_gemm_a4.audit ] || [ ! -f build/v2s_gemm_a4.audit ]; then
  ( cd build && $HIPCC $FLAGS -S --cuda-device-only ../v2s_gemm.hip -o v2s_gemm.s 2>/dev/null ) || true
  python3 - <<'PYEOF' > build/v2s_gemm_a4.audit
import re, sys
txt = open("build/v2s_gemm.s").read()
bad = nk = 0
for m in re.finditer(r"^(_ZN\S*gemm_a4p?_kernel\S*):[^\n]*\n(.*?)\n\s*s_endpgm", txt, re.S | re.M):
    body = re.sub(r";;#ASMSTART.*?;;#ASMEND", "", m.group(2), flags=re.S)
    hits = [l for l in body.splitlines() if re.search(r"v_accvgpr|scratch_|buffer_(load|store).*offen.*s\[0:3\]", l)]
    print(m.group(1), "compiler-emitted AGPR/scratch instructions:", len(hits))
    bad += len(hits); nk += 1
print("BAD" if bad else ("CLEAN" if nk == 8 else "NOT-FOUND"))
PYEOF
  cat build/v2s_gemm_a4.audit
  if grep -q BAD build/v2s_gemm_a4.audit; then echo "ERROR: the compiler touched AGPRs / scratch inside gemm_a4_kernel" >&2; rm -f build/v2s_gemm.o; exit 1; fi
  grep -q CLEAN build/v2s_gemm_a4.audit || { echo "ERROR: gemm_a4 ISA audit did not run" >&2; exit 1; }
fi
# Registers spilled to scratch cost what these two are built on, so say so loudly.  The decode memory-attention kernel keeps 192 accumulators in AGPRs and ~200 VGPRs:
# a spill puts scratch reloads (and their vmcnt(0) waits) into every iteration of its loop -- measured 5 us per 16-key group instead of 0.7.  The int8 product counts
# its VMEM operations by hand (s_waitcnt vmcnt(N)): reloads among them stay correct, as more operations in flight only make a counted wait longer, but a reload waits
# for all of them.  Its two 256 x 256 kernels are known to spill (64 and 48 bytes per lane).
for s in v2s_memattn v2s_gemm_q8; do
  if [ build/$s.o -nt build/$s.usage ] || [ ! -f build/$s.usage ]; then
    $HIPCC $FLAGS -c $s.hip -o /dev/null -Rpass-analysis=kernel-resource-usage 2> build/$s.usage.raw || true
    grep -E "Function Name|ScratchSize" build/$s.usage.raw | paste - - > build/$s.usage || true
    grep -vE "lane\]: 0 " build/$s.usage | sed 's/.*Function Name: \([^ ]*\).*lane\]: \([0-9]*\).*/WARNING: \1 uses \2 bytes of scratch per lane/' >&2 || true
  fi
done
OBJS=""; for s in $SRCS; do OBJS="$OBJS build/$s.o"; done
$HIPCC --offload-arch=gfx950 -shared -fPIC -o ../libvid2seq_hip.so $OBJS
echo "built $(realpath ../libvid2seq_hip.so)"
# the Python module that takes tensors apart for the 8-bit decoding calls (host code only; torch's libraries are loaded when it is imported)
if [ ! -f ../_bind.so ] || [ ! -f build/bind.done ] || [ v2s_bind.cpp -nt build/bind.done ] || [ ../../include/vid2seq_hip.h -nt build/bind.done ]; then
  TORCH=$(python3 -c 'import importlib.util as u, os; print(os.path.dirname(u.find_spec("torch").origin))')
  PYINC=$(python3 -c 'import sysconfig; print(sysconfig.get_paths()["include"])')
  g++ -O2 -std=c++17 -fPIC -shared -fvisibility=hidden -Wall -I"$TORCH/include" -I"$PYINC" v2s_bind.cpp -o ../_bind.so -L"$TORCH/lib" -ltorch_python -ltorch_cpu -lc10
  touch build/bind.done
  echo "built $(realpath ../_bind.so)"
fi
