"""Built code is reused only if it was built with the flags of now."""

import os
import runpy

import pytest

from lambdipy_amd.builder import flags, wheel_builder as wb


class _Compiler:
    """In place of hipcc and setup.py: writes what it is asked for."""

    def __init__(self):
        self.calls = []
        self.returncode = 0

    def run(self, cmd, **_):
        self.calls.append(cmd)
        if "-o" in cmd:
            with open(cmd[cmd.index("-o") + 1], "w") as f:
                f.write("code")
        return self

    def Popen(self, cmd, **_):
        return self.run(cmd)

    def communicate(self):
        return b"", b"failed"

    PIPE = None


@pytest.fixture()
def tree(tmp_path, monkeypatch):
    csrc = tmp_path / "csrc"
    csrc.mkdir()
    for f in ("a.hip", "b.hip", "rmsnorm.hip", "nn_capi.cpp", "kernels.h", "lpx_common.h",
              "standalone.hip"):
        (csrc / f).write_text(f)
        os.utime(csrc / f, (1, 1))  # older than all that is built
    hipcc = _Compiler()
    monkeypatch.setattr(wb, "subprocess", hipcc)
    monkeypatch.setattr(wb, "OPS_DIR", str(tmp_path))
    monkeypatch.setattr(wb, "HSACO_PATH", str(tmp_path / "s.hsaco"))
    monkeypatch.setattr(wb, "HSACO_SRC", str(csrc / "standalone.hip"))
    monkeypatch.setattr(wb, "NN_LIB_PATH", str(tmp_path / "libnn.so"))
    return tmp_path, hipcc, monkeypatch


def test_hsaco_of_other_flags_is_built_again(tree):
    tmp, hipcc, monkeypatch = tree
    (tmp / "s.hsaco").write_text("of a time without records")
    wb.ensure_standalone_hsaco()
    assert len(hipcc.calls) == 1 and set(flags.NO_PACKED_F32) <= set(hipcc.calls[0])
    wb.ensure_standalone_hsaco()
    assert len(hipcc.calls) == 1
    monkeypatch.setattr(flags, "NO_PACKED_F32", ["-other"])
    with pytest.raises(RuntimeError, match="stale"):
        wb.ensure_standalone_hsaco(allow_build=False)
    wb.ensure_standalone_hsaco()
    assert len(hipcc.calls) == 2 and "-other" in hipcc.calls[1]
    os.utime(tmp / "csrc" / "standalone.hip")  # and of an older source, as before
    os.utime(tmp / "s.hsaco", (2, 2))
    wb.ensure_standalone_hsaco()
    assert len(hipcc.calls) == 3


def test_nn_lib_and_its_objects_of_other_flags_are_built_again(tree):
    tmp, hipcc, monkeypatch = tree
    wb.ensure_nn_lib()
    assert len(hipcc.calls) == 4  # a, b, nn_capi and the link
    assert all(set(flags.NO_PACKED_F32) <= set(c) for c in hipcc.calls[:3])
    wb.ensure_nn_lib()
    assert len(hipcc.calls) == 4
    monkeypatch.setattr(wb, "TORCH_ONLY", {"rmsnorm.hip", "b.hip"})
    wb.ensure_nn_lib()
    assert len(hipcc.calls) == 5  # other members: a link of what is there
    monkeypatch.setattr(flags, "NO_PACKED_F32", ["-other"])
    with pytest.raises(RuntimeError, match="stale"):
        wb.ensure_nn_lib(allow_build=False)
    wb.ensure_nn_lib()
    assert len(hipcc.calls) == 8 and all("-other" in c for c in hipcc.calls[5:7])


def test_what_a_failed_build_left_is_not_reused(tree):
    tmp, hipcc, monkeypatch = tree
    hipcc.returncode = 1
    with pytest.raises(RuntimeError, match="hipcc failed"):
        wb.ensure_nn_lib()
    assert (tmp / "csrc" / ".nnobj" / "a.hip.o").exists()
    hipcc.returncode = 0
    hipcc.calls.clear()
    wb.ensure_nn_lib()
    assert len(hipcc.calls) == 4


def test_extension_of_other_flags_is_built_again(tree):
    tmp, hipcc, monkeypatch = tree
    so = str(tmp / "_lpx_ops.so")
    with open(so, "w") as f:
        f.write("code")
    with pytest.raises(RuntimeError, match="as it is now"):
        wb.ensure_ops_extension(allow_build=False)
    assert wb.ensure_ops_extension() == so
    assert len(hipcc.calls) == 1 and "setup.py" in hipcc.calls[0]
    flags.record(so, flags.OPS_HIP)  # as setup.py does
    assert wb.ensure_ops_extension(allow_build=False) == so
    assert len(hipcc.calls) == 1


def test_one_list_of_flags():
    assert set(flags.NO_PACKED_F32) <= set(flags.OPS_HIP)
    # setup.py takes them from the file, without importing the package
    again = runpy.run_path(flags.__file__)
    assert again["OPS_HIP"] == flags.OPS_HIP
