"""Build libcpde_b200.so and bin/cpde_server in-tree for sm_100a.

    python -m cpde_b200.build

nvcc cross-compiles without a GPU. The library is five translation units
compiled in parallel (csrc/library.cu: engine core, C ABI, allocation-free
entry; fast_forward.cu, fast_backward.cu, fast_head.cu: the fast-tier
dispatch and the kernels it instantiates; operators.cu: the device-tensor
operators); the server is a host program
linked against it with an $ORIGIN-relative rpath so the pair can be moved
together. The operators' Python binding (csrc/binding.cpp) is an extension module
over torch's C++ interface.
"""
import os
import subprocess
import sys
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
CSRC = PACKAGE / 'csrc'
BINDING = PACKAGE / '_operators.so'
LIBRARY = PACKAGE / 'libcpde_b200.so'
SERVER = PACKAGE / 'bin' / 'cpde_server'
BUILD = PACKAGE / '_build'
ARCH = ['-gencode', 'arch=compute_100a,code=sm_100a']
UNITS = ['library', 'fast_forward', 'fast_backward', 'fast_head', 'operators']


def _run(cmd):
    print(' '.join(str(c) for c in cmd), flush=True)
    subprocess.run([str(c) for c in cmd], check=True)


def _stale(target, sources):
    if not target.exists():
        return True
    mtime = target.stat().st_mtime
    return any(s.stat().st_mtime > mtime for s in sources)


def build(force=False, verbose_ptxas=False):
    from . import codegen
    codegen.write()
    nvcc = os.environ.get('NVCC', 'nvcc')
    sources = sorted(CSRC.glob('*.cu')) + sorted(CSRC.glob('*.cuh')) + sorted(CSRC.glob('*.hpp'))
    sources += sorted((CSRC / 'generated').glob('*.cuh'))
    sources.append(PACKAGE.parent / 'include' / 'cpde_b200.h')
    if force or _stale(LIBRARY, sources):
        # One object per translation unit, compiled in parallel; each unit is
        # compiled whole (no --split-compile, whose partitioning changed the
        # code of unrelated kernels from one build to the next).
        BUILD.mkdir(exist_ok=True)
        procs, objects = [], []
        for unit in UNITS:
            obj = BUILD / (unit + '.o')
            cmd = [nvcc, *ARCH, '-lineinfo', '-O3', '-std=c++17', '-Xcompiler', '-fPIC', '-c',
                   '--expt-relaxed-constexpr', '-o', obj, CSRC / (unit + '.cu')]
            if verbose_ptxas:
                cmd.insert(1, '-Xptxas=-v')
            print(' '.join(map(str, cmd)), flush=True)
            procs.append(subprocess.Popen([str(c) for c in cmd]))
            objects.append(obj)
        failed = [unit for unit, proc in zip(UNITS, procs) if proc.wait() != 0]
        if failed:
            raise RuntimeError(f'nvcc failed on {", ".join(failed)}')
        _run([nvcc, *ARCH, '-shared', '-o', LIBRARY, *objects, '-lnvrtc'])
    SERVER.parent.mkdir(exist_ok=True)
    server_sources = [CSRC / 'server_main.cpp', CSRC / 'wire.hpp', CSRC / 'common.hpp', LIBRARY]
    if force or _stale(SERVER, server_sources):
        cuda = Path(os.environ.get('CUDA_HOME', '/usr/local/cuda'))
        _run(['g++', '-std=c++17', '-O2', '-pthread', f'-I{cuda / "include"}', '-o', SERVER,
              CSRC / 'server_main.cpp', f'-L{PACKAGE}', '-lcpde_b200', f'-L{cuda / "lib64"}', '-lcudart',
              "-Wl,-rpath,$ORIGIN/..", f'-Wl,-rpath,{cuda / "lib64"}',
              '-Wl,--allow-shlib-undefined'])
    _build_binding(force)
    return LIBRARY, SERVER


def _build_binding(force):
    sources = [CSRC / 'binding.cpp', PACKAGE.parent / 'include' / 'cpde_b200.h']
    if not (force or _stale(BINDING, sources)):
        return
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    cuda = Path(os.environ.get('CUDA_HOME', '/usr/local/cuda'))
    includes = [*cpp_extension.include_paths(), sysconfig.get_path('include'), cuda / 'include']
    lib = Path(torch.__file__).parent / 'lib'
    _run(['g++', '-std=c++17', '-O2', '-fPIC', '-shared', f'-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}',
          *[f'-isystem{p}' for p in includes], '-o', BINDING, CSRC / 'binding.cpp', f'-L{lib}', '-ltorch_python', '-ltorch',
          '-ltorch_cpu', '-lc10', '-lc10_cuda', f'-L{cuda / "lib64"}', '-lcudart'])


if __name__ == '__main__':
    build(force='--force' in sys.argv, verbose_ptxas='--ptxas' in sys.argv)
