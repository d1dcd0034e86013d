"""Prints the compiler flags of a PyTorch extension for this interpreter (used by the Makefile); fails, with the
reason, where there is no PyTorch with CUDA or no Python headers. With --stamp: what they depend on, without importing it."""
import os
import sys
import sysconfig

if sys.argv[1:] == ["--stamp"]:
    import importlib.metadata
    import importlib.util
    try:
        torch = importlib.metadata.version("torch"), importlib.util.find_spec("torch").origin
    except (importlib.metadata.PackageNotFoundError, AttributeError):
        torch = ("none",)
    print(sys.executable, sys.version.split()[0], "torch", *torch)
    sys.exit(0)

try:
    import torch
    from torch.utils import cpp_extension
except ImportError as e:
    sys.exit(str(e))

lib = os.path.join(os.path.dirname(torch.__file__), "lib")
python = sysconfig.get_paths()["include"]
for f in (os.path.join(python, "Python.h"), os.path.join(lib, "libc10_cuda.so")):
    if not os.path.exists(f):
        sys.exit("no " + f)
print(" ".join(["-isystem " + p for p in cpp_extension.include_paths("cuda") + [python]]
               + ["-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI, "-L" + lib, "-Wl,-rpath," + lib,
                  "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python"]))
