"""Prints the compiler flags of a PyTorch extension for this interpreter (used by the Makefile)."""
import os
import sysconfig

import torch
from torch.utils import cpp_extension

lib = os.path.join(os.path.dirname(torch.__file__), "lib")
print(" ".join(["-I" + p for p in cpp_extension.include_paths("cuda") + [sysconfig.get_paths()["include"]]]
               + ["-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI, "-L" + lib, "-Wl,-rpath," + lib,
                  "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python"]))
