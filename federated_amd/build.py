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


def _run(commands, verbose):
  """The commands, at most as many at once as there are processors."""
  running, at_once = [], max(1, os.cpu_count() or 1)

  def wait(left):
    while len(running) > left:
      cmd, process = running.pop(0)
      if process.wait():
        for _, other in running:
          other.wait()
        raise subprocess.CalledProcessError(process.returncode, cmd)

  for cmd in commands:
    wait(at_once - 1)
    if verbose:
      print(" ".join(cmd), flush=True)
    running.append((cmd, subprocess.Popen(cmd)))  # pylint: disable=consider-using-with
  wait(0)


def build_libraries(libraries, verbose=False):
  """Libraries {path: macros of the codec's file}: all files each, compiled once where alike."""
  with tempfile.TemporaryDirectory() as d:
    def compiling(src, flags, defines, name):
      obj = os.path.join(d, name + ".o")
      return obj, [HIPCC, "-c"] + [f for f in flags if f != "-shared"] + ["-D" + m for m in defines] + ["-o", obj, src]

    client = [compiling(s, CLIENT_FLAGS, [], os.path.basename(s)) for s in CLIENT_SRCS]
    codec = [compiling(SRC, FLAGS, defines, "codec%d" % i) for i, defines in enumerate(libraries.values())]
    _run([cmd for _, cmd in codec + client], verbose)
    for out, (obj, _) in zip(libraries, codec):
      tmp = out + ".tmp.%d" % os.getpid()
      _run([[HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", tmp, obj] + [o for o, _ in client]], verbose)
      os.replace(tmp, out)


def build(force=False, verbose=False):
  sources = [SRC, HDR] + CLIENT_SRCS + CLIENT_HDRS
  if force or not os.path.exists(OUT) or os.path.getmtime(OUT) < max(os.path.getmtime(s) for s in sources):
    build_libraries({OUT: []}, verbose)
  return OUT


def main(argv):
  """[--force], or diagnostic libraries libfedcodec_NAME.so: NAME=MACRO[=VALUE][,MACRO...] ..."""
  variants = {}
  for arg in argv:
    name, _, macros = arg.partition("=")
    if not arg.startswith("--"):
      variants[os.path.join(HERE, "libfedcodec_%s.so" % name)] = [m for m in macros.split(",") if m]
  if variants:
    build_libraries(variants, verbose=True)
  else:
    build(force="--force" in argv, verbose=True)


if __name__ == "__main__":
  main(sys.argv[1:])
