"""The training operators on CPU tensors over their HOST-EXECUTED kernels -- TEST INFRASTRUCTURE.

``with train_on_host.patched():`` lets ``ops.linear_cross_entropy``, ``ops.orthogonalize`` and ``optim.muon_step_`` take CPU tensors: the
kernel sources of csrc/train compiled for the build host (lanes as fibers, tests/host_check) behind the library's own C ABI.  What it shows is
indexing, masks, layouts and arithmetic; never speed or waits."""
import contextlib
import ctypes
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(ROOT, 'unopticalflow_amd', 'csrc')
CHECK = os.path.join(HERE, 'host_check')
OUT = os.environ.get('UNFLOW_TRAIN_ON_HOST_DIR') or os.path.join(CHECK, '_build')
LIB = os.path.join(OUT, 'libunflow_train_on_host.so')
CLANG = '/opt/rocm/lib/llvm/bin/clang++'
FLAGS = os.environ.get('UNFLOW_TRAIN_ON_HOST_FLAGS', '-O2').split() + [
    '-std=c++20', '-fPIC', '-mf16c', '-ffp-contract=off', '-DUNFLOW_HOST_CHECK', '-Wno-unknown-attributes', '-Wno-unknown-pragmas', '-Wno-pass-failed',
    '-I', CHECK, '-I', CSRC, '-include', os.path.join(CHECK, 'hip_on_host_train.h')]
SOURCES = [os.path.join(CSRC, f) for f in ('train/linear_ce.hip', 'train/muon.hip', 'photo.hip', 'ssim.hip')]     # (photo.hip: the timing slots every launch asks about, and what it needs)
_cache = {}


def _deps():
    train = os.path.join(CSRC, 'train')
    return SOURCES + [os.path.join(train, f) for f in os.listdir(train)] + [os.path.join(CHECK, f) for f in os.listdir(CHECK) if f.endswith('.h')] + [
        os.path.abspath(__file__), os.path.join(CSRC, 'common.h'), os.path.join(ROOT, 'include', 'unflow_hip.h')]


def build():
    """-> path of the library, or None without the ROCm clang++."""
    if not os.path.exists(CLANG):
        return None
    os.makedirs(OUT, exist_ok=True)
    if os.path.exists(LIB) and all(os.path.getmtime(LIB) >= os.path.getmtime(p) for p in _deps()):
        return LIB
    jobs = []
    for src in SOURCES:
        obj = os.path.join(OUT, 'train_' + os.path.splitext(os.path.basename(src))[0] + '.o')
        jobs.append((src, obj, subprocess.Popen([CLANG, *FLAGS, '-x', 'c++', '-c', src, '-o', obj], stderr=subprocess.PIPE, text=True)))
    for src, _, p in jobs:
        err = p.communicate()[1]
        if p.returncode != 0:
            raise RuntimeError('%s:\n%s' % (src, err[-3000:]))
    subprocess.run([CLANG, '-shared', '-o', LIB] + [f for f in FLAGS if f.startswith('-fsan')] + [o for _, o, _ in jobs], check=True)
    return LIB


def library():
    if 'lib' not in _cache:
        path, lib = build(), None
        if path is not None:
            from unopticalflow_amd import _lib
            lib = ctypes.CDLL(path)
            for name, argtypes in _lib.SIGNATURES.items():
                if hasattr(lib, name):
                    fn = getattr(lib, name)
                    fn.argtypes = argtypes
                    fn.restype = ctypes.c_int
        _cache['lib'] = lib
    return _cache['lib']


@contextlib.contextmanager
def patched():
    from unopticalflow_amd import _lib, ops
    lib = library()
    if lib is None:
        import pytest
        pytest.skip('needs the ROCm clang++')
    old = (_lib._lib, ops._stream_of, ops._on, ops.on_device)
    _lib._lib, ops._stream_of, ops._on, ops.on_device = lib, (lambda d: None), (lambda d: contextlib.nullcontext()), (lambda t: True)
    try:
        yield lib
    finally:
        _lib._lib, ops._stream_of, ops._on, ops.on_device = old
