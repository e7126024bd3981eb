"""Build recipe for the in-tree drop-in library ``libgroupconv.so``.

nvcc compiles the C ABI (``csrc/common.cpp``), the shared host helpers and the
sm_100a CUDA engines (``csrc/conv_cuda.cu``, ``csrc/norm_cuda.cu``), each source
to an object of its own (only those older than what they include, in parallel),
and links them into a shared library that sits next to this file.  The CUDA runtime is linked as a shared library so that, inside a
process that already loaded PyTorch's CUDA runtime, both use one runtime
instance (one current device per thread, one primary context).

    python -m groupconv_atlas_b200.build          # build if stale
    python -m groupconv_atlas_b200.build --force  # always rebuild
"""
from __future__ import annotations

import argparse
import concurrent.futures
import os
import re
import shutil
import subprocess
import sys
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
ROOT = PACKAGE.parent
CSRC = PACKAGE / 'csrc'
INCLUDE = ROOT / 'include'
LIBRARY = PACKAGE / 'libgroupconv.so'
OBJECTS = PACKAGE / '_build'
ARCH = ['-gencode', 'arch=compute_100a,code=sm_100a']


def nvcc() -> str:
    for candidate in (os.environ.get('NVCC'), '/usr/local/cuda/bin/nvcc', shutil.which('nvcc')):
        if candidate and Path(candidate).exists():
            return candidate
    raise FileNotFoundError('nvcc not found: the B200 library needs the CUDA 12.9 toolkit')


def sources() -> list[Path]:
    return sorted(CSRC.glob('*.cu')) + sorted(CSRC.glob('*.cpp'))


def dependencies() -> list[Path]:
    return sources() + sorted(CSRC.glob('*.cuh')) + sorted(CSRC.glob('*.h')) + [INCLUDE / 'groupconv.h', Path(__file__)]


def stale(target: Path = LIBRARY) -> bool:
    if not target.exists():
        return True
    built = target.stat().st_mtime
    return any(p.stat().st_mtime > built for p in dependencies())


def includes(source: Path) -> list[Path]:
    """The source and every file of this library that it includes."""
    found, todo = [], [source]
    while todo:
        path = todo.pop()
        found.append(path)
        for name in re.findall(r'^#include "([^"]+)"', path.read_text(), flags=re.M):
            todo += [d / name for d in (CSRC, INCLUDE) if (d / name).exists() and d / name not in found]
    return found


def compile_command(source: Path, output: Path, extra: list[str] | None = None) -> list[str]:
    return [nvcc(), *ARCH, '-O3', '-lineinfo', '-std=c++17', '-Xcompiler', '-fPIC,-Wall', '-Xptxas', '-warn-spills',
            f'-I{INCLUDE}', f'-I{CSRC}', *(extra or []), '-c', str(source), '-o', str(output)]


def link_command(objects: list[Path], output: Path) -> list[str]:
    cuda_lib = Path(nvcc()).resolve().parent.parent / 'lib64'
    return [nvcc(), *ARCH, '-shared', '-cudart', 'shared', '-Xlinker', f'-rpath,{cuda_lib}', '-o', str(output),
            *map(str, objects)]


def run_tool(cmd: list[str], verbose: bool) -> None:
    if verbose:
        print(' '.join(cmd), flush=True)
    result = subprocess.run(cmd, capture_output=True, text=True)
    if result.returncode != 0:
        sys.stderr.write(result.stdout + result.stderr)
        raise RuntimeError(f'{Path(cmd[0]).name} failed with exit code {result.returncode}')
    if verbose and (result.stdout or result.stderr):
        sys.stderr.write(result.stdout + result.stderr)


def build(force: bool = False, verbose: bool = False, extra: list[str] | None = None) -> Path:
    """Compile the library when a source is newer than it (or when forced)."""
    if not force and not stale():
        return LIBRARY
    OBJECTS.mkdir(exist_ok=True)
    todo, objects = [], []
    for source in sources():
        target = OBJECTS / (source.name + '.o')
        objects.append(target)
        deps = [*includes(source), Path(__file__)]
        if force or not target.exists() or any(d.stat().st_mtime > target.stat().st_mtime for d in deps):
            todo.append((source, target))

    def compile_one(item):
        source, target = item
        part = target.with_suffix('.part')
        run_tool(compile_command(source, part, extra), verbose)
        part.replace(target)

    with concurrent.futures.ThreadPoolExecutor() as pool:
        list(pool.map(compile_one, todo))
    part = LIBRARY.with_suffix('.so.part')
    run_tool(link_command(objects, part), verbose)
    part.replace(LIBRARY)
    return LIBRARY


TORCH_EXT_SOURCE = PACKAGE / 'torch_ext' / 'conv_op.cpp'


def torch_ext_path() -> Path:
    """The PyTorch binding's extension module next to this file."""
    import sysconfig
    return PACKAGE / ('_gcb_torch' + sysconfig.get_config_var('EXT_SUFFIX'))


def build_torch_ext(force: bool = False, verbose: bool = False) -> Path:
    """Compile the PyTorch front end (torch_ext/conv_op.cpp, a thin C++ caller
    of gc_cuda_conv that allocates the output with PyTorch) against the
    in-tree library, when it is older than its sources."""
    import sysconfig
    import torch
    from torch.utils import cpp_extension
    target = torch_ext_path()
    deps = [TORCH_EXT_SOURCE, INCLUDE / 'groupconv.h', LIBRARY, Path(__file__)]
    if not force and target.exists() and all(d.stat().st_mtime <= target.stat().st_mtime for d in deps):
        return target
    cuda_include = Path(nvcc()).resolve().parent.parent / 'include'
    torch_lib = cpp_extension.library_paths()[0]
    abi = int(torch.compiled_with_cxx11_abi())
    cmd = ['g++', '-O2', '-std=c++17', '-shared', '-fPIC', f'-D_GLIBCXX_USE_CXX11_ABI={abi}',
           '-DTORCH_EXTENSION_NAME=_gcb_torch', '-DTORCH_API_INCLUDE_EXTENSION_H',
           *[f'-I{d}' for d in cpp_extension.include_paths()], f'-I{sysconfig.get_paths()["include"]}',
           f'-I{cuda_include}', f'-I{INCLUDE}', str(TORCH_EXT_SOURCE),
           f'-L{PACKAGE}', '-lgroupconv', f'-L{torch_lib}', '-lc10', '-lc10_cuda', '-ltorch', '-ltorch_cpu',
           '-ltorch_cuda', '-ltorch_python', f'-Wl,-rpath,$ORIGIN', f'-Wl,-rpath,{torch_lib}', '-o', str(target) + '.part']
    run_tool(cmd, verbose)
    Path(str(target) + '.part').replace(target)
    return target


def main(argv=None) -> int:
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument('--force', action='store_true')
    parser.add_argument('--verbose', action='store_true')
    parser.add_argument('--ptxas-info', action='store_true', help='print registers/spills per kernel')
    args = parser.parse_args(argv)
    extra = ['-Xptxas', '-v'] if args.ptxas_info else None
    path = build(force=args.force or args.ptxas_info, verbose=args.verbose or args.ptxas_info, extra=extra)
    print(path)
    return 0


if __name__ == '__main__':
    raise SystemExit(main())
