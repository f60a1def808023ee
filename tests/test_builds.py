"""Every library that the build makes, diagnostic ones too, holds what _lib binds: all of the
sources, compiled with the shipped flags.  The compiler is a stand-in that notes its
arguments."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def commands(tmp_path, *argv, env=()):
  """The compiler's command lines when `argv` runs in a copy of the tree."""
  for part in ("federated_amd/__init__.py", "federated_amd/build.py", "include", "federated_amd/csrc", "tools"):
    src, dst = os.path.join(ROOT, part), tmp_path / part
    if os.path.isdir(src):
      shutil.copytree(src, dst, ignore=shutil.ignore_patterns("__pycache__"))
    else:
      dst.parent.mkdir(parents=True, exist_ok=True)
      shutil.copy(src, dst)
  log, stub = tmp_path / "log", tmp_path / "hipcc"
  stub.write_text("#!%s\nimport sys\nopen(%r, 'a').write('\\t'.join(sys.argv[1:]) + '\\n')\n"
                  "open(sys.argv[sys.argv.index('-o') + 1], 'w').close()\n" % (sys.executable, str(log)))
  stub.chmod(0o755)
  subprocess.check_call(argv, cwd=tmp_path, stdout=subprocess.DEVNULL,
                        env=dict(os.environ, HIPCC=str(stub), PATH=os.path.dirname(sys.executable) + ":" +
                                 os.environ["PATH"], PYTHONPATH="", **dict(env)))
  return [line.split("\t") for line in log.read_text().splitlines()]


def libraries(lines):
  """{library: [compile commands of its objects]}."""
  objects = {c[c.index("-o") + 1]: c for c in lines if "-c" in c}
  made = {}
  for c in lines:
    if "-c" not in c:
      made[os.path.basename(c[c.index("-o") + 1]).split(".tmp")[0]] = [objects[a] for a in c if a in objects]
  return made


def check_whole(compiles, sources):
  assert sorted(os.path.basename(c[-1]) for c in compiles) == sources
  for c in compiles:
    assert "--offload-arch=gfx950" in c and c[c.index("-packed-fp32-ops") - 1] == "-Xclang", c
    if c[-1].endswith("fedcodec.hip"):
      assert "-ffp-contract=off" in c and "-fgpu-flush-denormals-to-zero" in c
    else:
      assert not any(a.startswith("-D") for a in c)


@pytest.mark.parametrize("script,names", [
    (None, {"libfedcodec.so": set()}),
    ("build_variants.sh", {"libfedcodec_stamps.so": {"-DFC_STAMPS"}, "libfedcodec_abl1.so": {"-DFC_ABL=1"},
                           "libfedcodec_abl4.so": {"-DFC_ABL=4"}, "libfedcodec_w6.so": {"-DFC_ENC_WAVES=6"}}),
    ("build_copy_variants.sh", {"libfedcodec_cpu8.so": {"-DFC_COPY_U=8"}, "libfedcodec_cpnt.so": {"-DFC_COPY_NT=1"},
                                "libfedcodec_cpu8nt.so": {"-DFC_COPY_U=8", "-DFC_COPY_NT=1"},
                                "libfedcodec_cpu2.so": {"-DFC_COPY_U=2", "-DFC_COPY_WG=16"}}),
], ids=["library", "variants", "copies"])
def test_libraries_are_whole(tmp_path, script, names):
  argv = ["bash", "tools/" + script] if script else [sys.executable, "-m", "federated_amd.build", "--force"]
  lines = commands(tmp_path, *argv, env=dict(ABL="1 4", WAVES="6"))
  sources = sorted(f for f in os.listdir(os.path.join(ROOT, "federated_amd", "csrc")) if f.endswith(".hip"))
  made = libraries(lines)
  assert set(made) == set(names)
  for name, compiles in made.items():
    check_whole(compiles, sources)
    assert {a for c in compiles for a in c if a.startswith("-D")} == names[name]
    assert (tmp_path / "federated_amd" / name).exists()
  assert len([c for c in lines if "-c" in c]) == len(sources) - 1 + len(names)  # alike files once


def test_a_failed_compile_leaves_no_library(tmp_path):
  with pytest.raises(subprocess.CalledProcessError):
    commands(tmp_path, "bash", "-c", "printf '#!/bin/sh\\nexit 3\\n' > hipcc; %s -m federated_amd.build --force 2>/dev/null" %
             sys.executable)
  assert not list((tmp_path / "federated_amd").glob("*.so*"))
