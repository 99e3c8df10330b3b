"""Ahead-of-time build of the CUDA library for sm_100a (in-tree shared object, no JIT cache)."""
import os
import subprocess

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, 'csrc')
LIB_NAME = 'libmegamoe_b200.so'
LIB_PATH = os.path.join(PKG_DIR, LIB_NAME)
# test build: the same library plus the CUDA-core cross-check engine (`engine='check'`), loaded by the tests only
CHECK_LIB_PATH = os.path.join(PKG_DIR, 'libmegamoe_b200_check.so')
# each source with the headers it is made from
_ABI = os.path.join('..', '..', 'include', 'megamoe_b200.h')
SOURCES = {
    'mm_abi.cu': ['mm_kernel.cuh', 'mm_frontend.cuh', 'mm_frontend_route.h', 'mm_device_attribute.h', 'mm_ptx.cuh', 'mm_prep.cuh', 'mm_batch.cuh',
                  'mm_decode.cuh', 'mm_error.h', _ABI],
    'mm_block.cu': ['mm_block_norm.h', 'mm_router.h', 'mm_error.h', _ABI],
    **{f'mm_block_norm_{t}.cu': ['mm_block_norm.cuh', 'mm_block_norm.h', 'mm_error.h', _ABI] for t in ('bf16', 'fp16', 'fp32')},
    **{f'mm_router_{t}.cu': ['mm_router.cuh', 'mm_router.h', 'mm_error.h', _ABI] for t in ('bf16', 'fp16', 'fp32')},
}
CHECK_SOURCES = ('mm_abi.cu',)           # those that the test build compiles anew; it shares the others' objects
OBJ_DIR = os.path.join(PKG_DIR, 'build')


def _stale(path: str, files) -> bool:
    if not os.path.exists(path):
        return True
    t = os.path.getmtime(path)
    return any(os.path.getmtime(f) > t for f in files)


def _run(cmds):
    """Run the commands side by side; returns what they printed, raises if one failed."""
    running = [subprocess.Popen(c, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True) for c in cmds]
    out = [p.communicate()[0] for p in running]
    for p, text in zip(running, out):
        if p.returncode != 0:
            raise RuntimeError(f'nvcc failed:\n{text}')
    return ''.join(out)


def build(force: bool = False, verbose: bool = False, check: bool = False) -> str:
    """Compile `csrc/*.cu` into `libmegamoe_b200.so` next to this file (`check`: the test build with the cross-check
    engine, `libmegamoe_b200_check.so`); returns its path. Sources whose object file is up to date are not compiled again."""
    path = CHECK_LIB_PATH if check else LIB_PATH
    inputs = [os.path.join(CSRC, f) for s in SOURCES for f in [s] + SOURCES[s]]
    if not force and not _stale(path, inputs):
        return path
    nvcc = os.environ.get('NVCC', '/usr/local/cuda/bin/nvcc')
    os.makedirs(OBJ_DIR, exist_ok=True)
    objects, cmds = [], []
    for source, headers in SOURCES.items():
        own = check and source in CHECK_SOURCES
        obj = os.path.join(OBJ_DIR, source[:-3] + ('_check.o' if own else '.o'))
        objects.append(obj)
        if force or _stale(obj, [os.path.join(CSRC, f) for f in [source] + headers]):
            cmds.append([nvcc] + (['-Xptxas', '-v'] if verbose else []) +
                        ['-gencode', 'arch=compute_100a,code=sm_100a', '-lineinfo', '-O3', '-std=c++17', '-Xcompiler', '-fPIC', '-c', '-o', obj] +
                        (['-DMM_WITH_CHECK_ENGINE'] if own else []) + [os.path.join(CSRC, source)])
    text = _run(cmds)
    _run([[nvcc, '-gencode', 'arch=compute_100a,code=sm_100a', '-shared', '-Xcompiler', '-fPIC', '-o', path] + objects])
    if verbose:
        print(text)
    return path


if __name__ == '__main__':
    print(build(force=True, verbose=True))
