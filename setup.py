"""In-tree build of the MI355X-native extension (_C).

  PYTORCH_ROCM_ARCH=gfx950 python setup.py build_ext --inplace

hipcc cross-compiles gfx950 without a GPU; the built .so lives inside the
package (anand_mxnet_amd/_C*.so) so gpurun snapshots ship it.
"""
import glob
import os
import re

os.environ.setdefault("PYTORCH_ROCM_ARCH", "gfx950")

from setuptools import setup
from torch.utils.cpp_extension import BuildExtension, CUDAExtension

ROOT = os.path.dirname(os.path.abspath(__file__))
SRC = os.path.join(ROOT, "anand_mxnet_amd", "src")

sources = [os.path.join(SRC, "bindings.hip")] + \
    sorted(glob.glob(os.path.join(SRC, "kernels", "*.hip")))


def stale_objects(objects, src):
    """Those of the compiled objects that are older than a header their
    source includes: hipcc is run without dependency files, so ninja knows
    of the sources alone."""
    def headers(path, seen):
        for name in re.findall(r'^\s*#\s*include\s+"([^"]+)"',
                               open(path).read(), re.M):
            h = os.path.join(os.path.dirname(path), name)
            if os.path.exists(h) and h not in seen:
                seen.add(h)
                headers(h, seen)
        return seen

    stale = []
    for obj in objects:
        base = re.sub(r"(_hip)?\.o$", ".hip", os.path.basename(obj))
        for path in glob.glob(os.path.join(src, "**", base), recursive=True):
            if any(os.path.getmtime(h) > os.path.getmtime(obj)
                   for h in headers(path, set())):
                stale.append(obj)
                break
    return stale


if __name__ == "__main__":
    for obj in stale_objects(
            glob.glob(os.path.join(ROOT, "build", "temp*", "**", "*.o"),
                      recursive=True), SRC):
        os.remove(obj)
    setup(
        name="anand_mxnet_amd_native",
        ext_modules=[
            CUDAExtension(
                name="anand_mxnet_amd._C",
                sources=sources,
                extra_compile_args={
                    "cxx": ["-O3", "-std=c++17"],
                    # packed fp32 instructions stay off: some of their forms
                    # have given wrong results on this hardware
                    # and assembly that names M0, which the compiler does
                    # not allocate, is no cause for a remark
                    "nvcc": ["-O3", "-std=c++17", "-Xclang", "-target-feature",
                             "-Xclang", "-packed-fp32-ops",
                             "-Wno-inline-asm"],
                },
            )
        ],
        cmdclass={"build_ext": BuildExtension.with_options(use_ninja=True)},
    )
