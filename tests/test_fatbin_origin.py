"""Only libraries built here from source are taken apart by strip_fatbin."""

import os
import shutil
import subprocess

import pytest
from click.testing import CliRunner

from lambdipy_amd import recipes
from lambdipy_amd.cli import main
from lambdipy_amd.packager import fatbin

HIPCC = "/opt/rocm/bin/hipcc"

needs_rocm = pytest.mark.skipif(
    not (os.path.exists(HIPCC) and os.path.exists(fatbin.BUNDLER)),
    reason="ROCm toolchain not available")

SRC = r"""
#include <hip/hip_runtime.h>
extern "C" __global__ void lpx_origin_kernel(float* x) { x[threadIdx.x] += 1.0f; }
extern "C" int lpx_origin_launch(float* x) {
  lpx_origin_kernel<<<1, 64>>>(x);
  return (int)hipGetLastError();
}
"""


@pytest.fixture(scope="module")
def built(tmp_path_factory):
    d = tmp_path_factory.mktemp("origin")
    (d / "origin.hip").write_text(SRC)
    so = d / "liborigin.so"
    subprocess.run([HIPCC, "-fPIC", "-shared", str(d / "origin.hip"), "-o", str(so),
                    "-O1", "--offload-arch=gfx950", "--offload-arch=gfx942"],
                   check=True, capture_output=True)
    return so


@needs_rocm
def test_a_library_next_to_its_source_is_stripped(built, tmp_path):
    out = tmp_path / "out.so"
    assert fatbin.strip_fatbin(str(built), str(out))["stripped"] == 1


@needs_rocm
def test_a_library_of_another_origin_is_refused_untouched(built, tmp_path):
    # as it would lie in an installed package: no source anywhere near
    foreign = tmp_path / "liborigin.so"
    shutil.copyfile(built, foreign)
    before = foreign.read_bytes()
    with pytest.raises(fatbin.ForeignLibrary, match="no source next to it"):
        fatbin.strip_fatbin(str(foreign))
    with pytest.raises(fatbin.ForeignLibrary):
        fatbin.strip_fatbin(str(foreign), str(tmp_path / "out.so"))
    r = CliRunner().invoke(main, ["strip-archs", str(foreign)])
    assert r.exit_code != 0 and "no source next to it" in r.output
    # nor through a link from beside a source
    (tmp_path / "src").mkdir()
    shutil.copyfile(built.parent / "origin.hip", tmp_path / "src" / "origin.hip")
    link = tmp_path / "src" / "liborigin.so"
    link.symlink_to(foreign)
    with pytest.raises(fatbin.ForeignLibrary):
        fatbin.strip_fatbin(str(link), str(tmp_path / "out.so"))
    assert foreign.read_bytes() == before and not (tmp_path / "out.so").exists()


@needs_rocm
def test_a_source_newer_than_the_library_is_not_its_source(built, tmp_path):
    so, src = tmp_path / "liborigin.so", tmp_path / "origin.hip"
    shutil.copyfile(built, so)
    src.write_text(SRC)
    os.utime(src, (os.path.getmtime(so) + 10,) * 2)
    with pytest.raises(fatbin.ForeignLibrary):
        fatbin.strip_fatbin(str(so))
    os.utime(src, (os.path.getmtime(so) - 10,) * 2)
    assert fatbin.strip_fatbin(str(so))["stripped"] == 1


def test_what_is_no_library_is_said_to_be_none(tmp_path):
    text = tmp_path / "notes.so"
    text.write_text("no library")
    with pytest.raises(ValueError, match="not an ELF file"):
        fatbin.strip_fatbin(str(text))
    assert text.read_text() == "no library"


def test_a_recipe_that_asks_for_it_is_told(monkeypatch):
    # a layer's libraries come out of wheels
    told = []
    monkeypatch.setattr(recipes.log, "warning", lambda text, *a: told.append(text % a))
    d = {"recipe_format": 1, "name": "x", "versions": ">=1", "kind": "native"}
    recipes.BuildRecipe.from_dict(d)
    assert not told
    recipe = recipes.BuildRecipe.from_dict(dict(d, strip_archs=True))
    assert not hasattr(recipe, "strip_archs")
    assert len(told) == 1 and "no effect" in told[0]
