"""The build script with a stand-in for the compiler: which objects a library is linked from."""
import importlib.util
import os
import stat

import pytest
from conftest import PKG_NAME, ROOT

# writes its own arguments to the output; linking puts the objects' texts together
FAKE = """#!/bin/sh
out=; inputs=; compile=; d=
while [ $# -gt 0 ]; do
  case "$1" in
    -o) out=$2; shift;;
    -c) compile=1;;
    -D*) d="$d $1";;
    *.o) inputs="$inputs $1";;
    *.cu) src=$1;;
  esac
  shift
done
[ -n "$FAIL" ] && case "$src" in *"$FAIL"*) exit 3;; esac
[ -n "$FAIL" ] && sleep 0.5
if [ -n "$compile" ]; then echo "$(basename $src)$d" > "$out"; else cat $inputs > "$out"; fi
"""


@pytest.fixture
def build(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("build_under_test", os.path.join(ROOT, PKG_NAME, "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    nvcc = tmp_path / "nvcc"
    nvcc.write_text(FAKE)
    nvcc.chmod(nvcc.stat().st_mode | stat.S_IEXEC)
    pkg = tmp_path / "pkg"
    pkg.mkdir()
    monkeypatch.setattr(mod, "NVCC", str(nvcc))
    monkeypatch.setattr(mod, "PKG", str(pkg))
    monkeypatch.setattr(mod, "LIB", str(pkg / "libdsd_b200.so"))
    return mod


def test_objects_with_defines_stay_out_of_other_libraries(build, tmp_path):
    other = tmp_path / "experiment"
    other.mkdir()
    lib = str(other / os.path.basename(build.LIB))       # the same file name in another place
    assert "-DX=1" in open(build.build_library(out=lib, defines=("X=1",))).read()
    assert "-D" not in open(build.build_library(out=build.LIB)).read()
    assert "-DX=2" in open(build.build_library(out=lib, defines=("X=2",))).read()
    assert "-D" not in open(build.build_library(out=build.LIB)).read()
    # experiments under the library's own name are not taken for it afterwards
    build.build_library(out=build.LIB, defines=("X=3",))
    assert "-D" not in open(build.build_library(out=build.LIB, force=True)).read()


def test_a_build_that_fails_ends_its_other_compilers_first(build, monkeypatch):
    import subprocess
    monkeypatch.setenv("FAIL", build.SOURCES[0])
    with pytest.raises(subprocess.CalledProcessError):
        build.build_library(out=build.LIB)
    objects = os.path.join(build.PKG, "build", os.path.basename(build.LIB) + "." + build.SOURCES[1] + ".o")
    assert os.path.exists(objects) and not os.path.exists(build.LIB)
