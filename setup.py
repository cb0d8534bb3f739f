"""In-tree build of the HIP/CDNA4 extension (gfx950 only).

    PYTORCH_ROCM_ARCH=gfx950 python setup.py build_ext --inplace

The built .so lands next to the package (deepreduce_amd/_hip_ops*.so) so it
travels with the repo snapshot to GPU boxes.
"""
import glob
import os
import zlib

from setuptools import setup

os.environ.setdefault("PYTORCH_ROCM_ARCH", "gfx950")

from torch.utils.cpp_extension import BuildExtension, CUDAExtension  # noqa: E402

# The compiler's dependency files do not cover HIP sources: a changed header
# has to make the extension be built, and each object's command another one.
headers = sorted(glob.glob("deepreduce_amd/ops/src/*.h"))
version = zlib.crc32(b"".join(open(h, "rb").read() for h in headers))

setup(
    name="deepreduce_amd",
    version="0.1.0",
    packages=["deepreduce_amd"],
    ext_modules=[
        CUDAExtension(
            name="deepreduce_amd._hip_ops",
            sources=[
                "deepreduce_amd/ops/src/hip_ops.hip",
                "deepreduce_amd/ops/src/attention.hip",
                "deepreduce_amd/ops/src/grad_norm.hip",
                "deepreduce_amd/ops/src/rotary.hip",
            ],
            depends=headers,
            extra_compile_args={
                "cxx": ["-O3"],
                # packed float adds and products have given wrong results
                # now and then: the compiler makes none
                "nvcc": ["-O3", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                         f"-DHEADERS={version}"],
            },
        )
    ],
    cmdclass={"build_ext": BuildExtension},
)
