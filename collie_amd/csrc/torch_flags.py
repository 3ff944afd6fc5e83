"""Prints the compiler flags for an extension of the installed torch (used by the Makefile)."""
import sysconfig

import torch
from torch.utils import cpp_extension

print('-D_GLIBCXX_USE_CXX11_ABI=%d' % torch._C._GLIBCXX_USE_CXX11_ABI,
      *('-isystem' + p for p in [*cpp_extension.include_paths(), sysconfig.get_paths()['include'],
                                 '/opt/rocm/include']),
      *('-L' + p for p in cpp_extension.library_paths()),
      '-ltorch -ltorch_cpu -ltorch_python -lc10 -lc10_hip')
