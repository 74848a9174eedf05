"""Build the lambdipy_amd gfx950 kernel extension in-tree.

    PYTORCH_ROCM_ARCH=gfx950 python setup.py build_ext --inplace

The extension is AOT-compiled for gfx950 only (no JIT at cold start, no
multi-arch fat binaries): the built .so ships inside recipe wheels / the
repo tree and travels to the GPU box with the source snapshot.
"""

import os
import runpy

from setuptools import setup

os.environ.setdefault("PYTORCH_ROCM_ARCH", "gfx950")

from torch.utils.cpp_extension import BuildExtension, CUDAExtension  # noqa: E402

ROOT = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(ROOT, "lambdipy_amd", "ops", "csrc")
FLAGS = runpy.run_path(os.path.join(ROOT, "lambdipy_amd", "builder", "flags.py"))

sources = [
    os.path.join(CSRC, f)
    for f in sorted(os.listdir(CSRC))
    if f.endswith((".cpp", ".hip")) and not f.endswith(("_hip.cpp", "_hip.hip"))
    and f != "standalone.hip"  # --genco code object, built by the builder
    and f != "nn_capi.cpp"  # liblpx_nn C API, built by builder.ensure_nn_lib
]



class BuildOps(BuildExtension):
    """Builds again, too, what was built with other flags."""

    def run(self):
        paths = [self.get_ext_fullpath(ext.name) for ext in self.extensions]
        for path in paths:
            if not FLAGS["built_with"](path, FLAGS["OPS_HIP"]):
                self.force = True
                FLAGS["forget"](path)
        super().run()
        for path in paths:
            FLAGS["record"](path, FLAGS["OPS_HIP"])


setup(
    name="lambdipy-amd",
    version="0.1.0",
    description="MI355X-native scientific-Python packager + runtime",
    packages=[
        "lambdipy_amd",
        "lambdipy_amd.resolver",
        "lambdipy_amd.recipes",
        "lambdipy_amd.builder",
        "lambdipy_amd.packager",
        "lambdipy_amd.ops",
        "lambdipy_amd.runtime",
        "lambdipy_amd.models",
        "lambdipy_amd.parallel",
        "lambdipy_amd.utils",
    ],
    package_data={"lambdipy_amd.recipes": ["data/*.json"]},
    ext_modules=[
        CUDAExtension(
            name="lambdipy_amd.ops._lpx_ops",
            sources=sources,
            depends=[os.path.join(CSRC, h) for h in ("kernels.h", "lpx_common.h")],
            extra_compile_args={"cxx": FLAGS["OPS_CXX"], "nvcc": FLAGS["OPS_HIP"]},
        )
    ],
    cmdclass={"build_ext": BuildOps},
    entry_points={"console_scripts": ["lpx = lambdipy_amd.cli:main"]},
)
