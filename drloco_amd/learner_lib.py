"""The learner's operators: drloco_amd/csrc/libdrloco_learner.so (the C-ABI in include/drloco_learner.h) through ctypes, and
dl_learner_torch.so, which calls it on torch tensors for drloco_amd.memory and drloco_amd.muon.

A library of its own next to libdrloco_hip.so: its kernels need neither the step kernels' compiler flags nor their two code
objects.  There is no CPU fallback: the functions refuse tensors that are not on a HIP device."""
import ctypes as C
import os
import subprocess
import sysconfig

import torch

from . import lib

CSRC = os.path.join(lib.CSRC, 'learner')
LIB_PATH = os.path.join(lib.CSRC, 'libdrloco_learner.so')
TORCH_PATH = os.path.join(lib.CSRC, 'dl_learner_torch.so')
ABI_VERSION = 1
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}          # DL_F32, DL_BF16, DL_F16
MARK = 16                                                                 # DL_MEMORY_MARK
# hipcc turns pairs of float operations into packed ones by itself; some forms of those are not trusted on this hardware
EXTRA_FLAGS = ['-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']

_I64, _I32, _P = C.c_int64, C.c_int32, C.c_void_p


class MemoryShape(C.Structure):
    """dl_memory_shape"""
    _fields_ = [(n, _I64) for n in ('T', 'N', 'D', 'x_t', 'x_n', 'gate_t', 'gate_n', 'starts_t', 'starts_n', 'grad_t', 'grad_n')] + [('dtype', _I32), ('reserved', _I32)]


class OrthShape(C.Structure):
    """dl_orth_shape"""
    _fields_ = [(n, _I64) for n in ('batch', 'rows', 'cols', 'grad_b', 'grad_r', 'momentum_b', 'momentum_r', 'momentum_out_b', 'momentum_out_r', 'weight_b', 'weight_r', 'out_b', 'out_r')] + \
               [(n, C.c_double) for n in ('a', 'b', 'c', 'beta', 'weight_keep', 'gain')] + [(n, _I32) for n in ('steps', 'nesterov', 'grad_type', 'weight_type', 'out_type', 'reserved')]


_SIGNATURES = {
    # name: (restype, argtypes)       -- every symbol include/drloco_learner.h declares
    'dl_learner_last_error': (C.c_char_p, []),
    'dl_learner_abi_version': (C.c_int, []),
    'dl_memory_workspace_bytes': (_I64, [C.POINTER(MemoryShape)]),
    'dl_memory_forward': (C.c_int, [C.POINTER(MemoryShape), _P, _P, _P, _P, _P, _P, _P, _P, _P]),
    'dl_memory_backward': (C.c_int, [C.POINTER(MemoryShape), _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P]),
    'dl_memory_step': (C.c_int, [C.POINTER(MemoryShape), _P, _P, _P, _P, _P, _P, _P]),
    'dl_orth_check_coefficients': (C.c_int, [_I32, C.c_double, C.c_double, C.c_double]),
    'dl_orth_workspace_bytes': (_I64, [C.POINTER(OrthShape)]),
    'dl_orth_update': (C.c_int, [C.POINTER(OrthShape), _P, _P, _P, _P, _P, _P, _P]),
}

_lib = None
_ops = None


def _sources():
    return [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC)) if f.endswith(('.hip', '.hpp'))] + [os.path.join(lib.INCLUDE, 'drloco_learner.h')]


def _fresh(path, sources):
    return os.path.exists(path) and all(os.path.getmtime(s) <= os.path.getmtime(path) for s in sources)


def _run(cmd, verbose):
    if verbose:
        print(' '.join(cmd))
    subprocess.check_call(cmd)


def build(force=False, verbose=False):
    """hipcc --offload-arch=gfx950 of the learner's kernels and g++ of their torch binding, into in-tree shared libraries."""
    root = os.path.dirname(lib.INCLUDE)
    if force or not _fresh(LIB_PATH, _sources()):
        hipcc = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')
        _run([hipcc, '--offload-arch=gfx950', '-O3', '-std=c++17', '-fPIC', '-shared', '-Wno-unused-command-line-argument', '-ffile-prefix-map=' + root + '=.', '-I' + lib.INCLUDE, '-I' + CSRC] +
             EXTRA_FLAGS + [os.path.join(CSRC, 'dl_learner.hip'), '-o', LIB_PATH], verbose)
    source = os.path.join(CSRC, 'dl_torch.cpp')
    if force or not _fresh(TORCH_PATH, [source, os.path.join(lib.INCLUDE, 'drloco_learner.h')]):
        from torch.utils import cpp_extension
        rocm = os.environ.get('ROCM_PATH', '/opt/rocm')
        _run(['g++', '-O2', '-std=c++17', '-fPIC', '-shared', '-w', '-D__HIP_PLATFORM_AMD__=1', '-DUSE_ROCM=1', f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}',
              '-ffile-prefix-map=' + root + '=.', '-I' + lib.INCLUDE] + ['-I' + p for p in cpp_extension.include_paths()] + ['-I' + os.path.join(rocm, 'include'), '-I' + sysconfig.get_paths()['include'],
              source, '-o', TORCH_PATH] + ['-L' + p for p in cpp_extension.library_paths()] + ['-lc10', '-lc10_hip', '-ltorch_cpu', '-ltorch', '-ltorch_python', '-L' + lib.CSRC, '-ldrloco_learner', '-Wl,-rpath,$ORIGIN'], verbose)
    return LIB_PATH


def load():
    """Load the library; raises DrlocoError if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise lib.DrlocoError(f'{LIB_PATH} is missing: run `python -c "import __graft_entry__ as g; g.build()"` '
                                  '(hipcc --offload-arch=gfx950); there is no CPU fallback')
        so = C.CDLL(LIB_PATH)
        for name, (res, args) in _SIGNATURES.items():
            fn = getattr(so, name)
            fn.restype, fn.argtypes = res, args
        if so.dl_learner_abi_version() != ABI_VERSION:
            raise lib.DrlocoError(f'ABI version mismatch between drloco_amd/learner_lib.py and {os.path.basename(LIB_PATH)}')
        _lib = so
    return _lib


def check(rc):
    """rc of a call, or the DrlocoError of a negative one."""
    if rc < 0:
        raise lib.DrlocoError(f'drloco_learner error {rc}: {load().dl_learner_last_error().decode()}')
    return rc


def ops():
    """The torch binding (dl_torch.cpp); raises DrlocoError if it has not been built."""
    global _ops
    if _ops is None:
        load()
        if not os.path.exists(TORCH_PATH):
            raise lib.DrlocoError(f'{TORCH_PATH} is missing: run `python -c "import __graft_entry__ as g; g.build()"`')
        import importlib.machinery
        import importlib.util
        loader = importlib.machinery.ExtensionFileLoader('dl_learner_torch', TORCH_PATH)
        _ops = importlib.util.module_from_spec(importlib.util.spec_from_loader('dl_learner_torch', loader))
        loader.exec_module(_ops)
    return _ops


def require_device(name, *tensors):
    """All of `tensors` (None: skipped) on one HIP device, or ValueError / DrlocoError."""
    device = None
    for t in tensors:
        if t is None:
            continue
        if not torch.is_tensor(t):
            raise TypeError(f'{name}: expected tensors, got {type(t).__name__}')
        if t.device.type != 'cuda':
            raise lib.DrlocoError(f'{name}: needs tensors on a HIP device, got one on {t.device} (there is no CPU fallback)')
        if device is None:
            device = t.device
        elif t.device != device:
            raise ValueError(f'{name}: tensors on {device} and on {t.device}')
    return device
