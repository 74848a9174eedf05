"""What the device code is compiled with, and which artefacts were.

An artefact is reused if its sources are older and it was built with the same
flags; those stand in a file of text next to it. setup.py runs this file by its
path, so it imports nothing but the standard library.
"""

from __future__ import annotations

import os
from typing import Sequence

# Device code is compiled without packed f32 instructions: some forms of
# v_pk_{add,mul,fma}_f32 gave wrong results on MI355X.
NO_PACKED_F32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]

# the torch extension: host code, device code
OPS_CXX = ["-O3", "-std=c++17"]
OPS_HIP = [*OPS_CXX, *NO_PACKED_F32]


def _record_of(artefact: str) -> str:
    return artefact + ".flags"


def built_with(artefact: str, flags: Sequence[str]) -> bool:
    """Whether the artefact is there and was built with these flags."""
    try:
        with open(_record_of(artefact)) as f:
            return os.path.exists(artefact) and f.read() == "\n".join(flags)
    except OSError:
        return False


def forget(artefact: str) -> None:
    """Before a build: whatever it leaves behind if it fails is not reused."""
    try:
        os.unlink(_record_of(artefact))
    except FileNotFoundError:
        pass


def record(artefact: str, flags: Sequence[str]) -> None:
    with open(_record_of(artefact), "w") as f:
        f.write("\n".join(flags))
