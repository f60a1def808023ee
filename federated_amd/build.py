"""Build recipe for libfedcodec.so (hipcc, gfx950 only, in-tree)."""
import os
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
SRC = os.path.join(HERE, "csrc", "fedcodec.hip")
HDR = os.path.join(os.path.dirname(HERE), "include", "fedcodec.h")
# the clients' local step: ordinary float32 arithmetic (denormals kept, contraction on)
CLIENT_SRCS = [os.path.join(HERE, "csrc", f) for f in ("client_rows.hip", "client_linear.hip")]
CLIENT_HDRS = [os.path.join(HERE, "csrc", "client_common.h")]
OUT = os.path.join(HERE, "libfedcodec.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
# no packed float32 instructions, in any file: some of their forms are not reliable
NO_PACKED_F32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-shared",
         # TF-CPU numerics: FTZ/DAZ on float32, no FMA contraction
         "-fgpu-flush-denormals-to-zero", "-ffp-contract=off",
         # no SLP packing into v_pk_* f32 ops: on gfx950 a v_pk_mul/add costs about two
         # scalar ops plus the register moves it needs (k_encode -2.6 % without it)
         "-fno-slp-vectorize",
         # no atomic optimizer: its expansion (mbcnt, readfirstlane of the result right
         # after the atomic) made k_encode wait for each ticket atomic -- and every
         # vector memory operation before it -- where it is issued instead of where
         # the ticket is used, a tile later
         "-mllvm", "-amdgpu-atomic-optimizer-strategy=None"] + NO_PACKED_F32


CLIENT_FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-shared"] + NO_PACKED_F32


def build(force=False, verbose=False):
  sources = [SRC, HDR] + CLIENT_SRCS + CLIENT_HDRS
  if not force and os.path.exists(OUT) and os.path.getmtime(OUT) >= max(os.path.getmtime(s) for s in sources):
    return OUT
  tmp = OUT + ".tmp.%d" % os.getpid()
  with tempfile.TemporaryDirectory() as d:
    objs, running = [], []
    for src, flags in [(SRC, FLAGS)] + [(s, CLIENT_FLAGS) for s in CLIENT_SRCS]:
      objs.append(os.path.join(d, os.path.basename(src) + ".o"))
      cmd = [HIPCC, "-c"] + [f for f in flags if f != "-shared"] + ["-o", objs[-1], src]
      if verbose:
        print(" ".join(cmd), flush=True)
      running.append((cmd, subprocess.Popen(cmd)))  # pylint: disable=consider-using-with
    codes = [p.wait() for _, p in running]
    for (cmd, _), rc in zip(running, codes):
      if rc:
        raise subprocess.CalledProcessError(rc, cmd)
    subprocess.check_call([HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", tmp] + objs)
  os.replace(tmp, OUT)
  return OUT


if __name__ == "__main__":
  build(force="--force" in sys.argv, verbose=True)
