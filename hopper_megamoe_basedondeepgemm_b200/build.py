"""Ahead-of-time build of the CUDA library for sm_100a (in-tree shared object, no JIT cache)."""
import importlib.util
import os
import runpy
import shutil
import subprocess
import sysconfig
import time
import warnings

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, 'csrc')
LIB_NAME = 'libmegamoe_b200.so'
LIB_PATH = os.path.join(PKG_DIR, LIB_NAME)
# test build: the same library plus the CUDA-core cross-check engine (`engine='check'`), loaded by the tests only
CHECK_LIB_PATH = os.path.join(PKG_DIR, 'libmegamoe_b200_check.so')
# Python binding of the operators around the layer: plain C++ on the C ABI and torch's tensors
BINDING_PATH = os.path.join(PKG_DIR, 'mm_block_binding.so')
BINDING_SOURCE = 'mm_block_binding.cpp'
# each source with the headers it is made from
_ABI = os.path.join('..', '..', 'include', 'megamoe_b200.h')
SOURCES = {
    'mm_abi.cu': ['mm_kernel.cuh', 'mm_frontend.cuh', 'mm_frontend_route.h', 'mm_device_attribute.h', 'mm_ptx.cuh', 'mm_prep.cuh', 'mm_batch.cuh',
                  'mm_decode.cuh', 'mm_error.h', 'mm_launch.h', _ABI],
    'mm_block.cu': ['mm_block_norm.h', 'mm_router.h', 'mm_error.h', _ABI],
    **{f'mm_block_norm_{w}{t}.cu': ['mm_block_norm.cuh', 'mm_block_norm.h', 'mm_launch.h', 'mm_ptx.cuh', 'mm_error.h', _ABI] for w in ('', 'wide_') for t in ('bf16', 'fp16', 'fp32')},
    **{f'mm_router_{t}.cu': ['mm_router.cuh', 'mm_router.h', 'mm_launch.h', 'mm_ptx.cuh', 'mm_error.h', _ABI] for t in ('bf16', 'fp16', 'fp32')},
}
CHECK_SOURCES = ('mm_abi.cu',)           # those that the test build compiles anew; it shares the others' objects
OBJ_DIR = os.path.join(PKG_DIR, 'obj')


def _stale(path: str, files) -> bool:
    if not os.path.exists(path):
        return True
    t = os.path.getmtime(path)
    return any(os.path.getmtime(f) > t for f in files)


def _record(path: str) -> str:
    """Where it says by which commands a file was made."""
    return os.path.join(OBJ_DIR, os.path.basename(path) + '.cmd')


def _named(*commands) -> str:
    """Commands as they count: wherever the package lies, and whatever they print."""
    return '\n'.join(' '.join(c.replace(PKG_DIR, '.') for c in command if c not in ('-Xptxas', '-v')) for command in commands)


def _recorded(path: str):
    if not os.path.exists(_record(path)):
        return None
    with open(_record(path)) as f:
        return f.read()


def _run(cmds, start, names=None):
    """Run the commands side by side, each with the file that it makes behind `-o`; returns what they printed, raises if one failed. A file is made under another name and takes its own
    when it is complete: what a compiler leaves that was stopped is not taken for it. Its time is `start`, so a source that changes meanwhile is newer."""
    running = []
    for c in cmds:
        at = c.index('-o') + 1
        part = f'{c[at]}.{os.getpid()}.part'
        running.append((c, c[at], part, subprocess.Popen(c[:at] + [part] + c[at + 1:], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    out, failed = [], ''
    for c, path, part, p in running:
        out.append(p.communicate()[0])
        if p.returncode == 0:
            os.utime(part, (start, start))
            os.replace(part, path)
            with open(_record(path), 'w') as f:
                f.write(names or _named(c))
        else:
            failed = failed or f'{c[0]} failed:\n{out[-1]}'
            if os.path.exists(part):
                os.remove(part)
    if failed:
        raise RuntimeError(failed)
    return ''.join(out)


def build(force: bool = False, verbose: bool = False, check: bool = False) -> str:
    """Compile `csrc/*.cu` into `libmegamoe_b200.so` next to this file (`check`: the test build with the cross-check
    engine, `libmegamoe_b200_check.so`); returns its path. Sources whose object file is up to date, and was made by the same command, are not compiled again."""
    start = time.time()
    path = CHECK_LIB_PATH if check else LIB_PATH
    nvcc = os.environ.get('NVCC', '/usr/local/cuda/bin/nvcc')
    cmds, inputs = {}, {}                    # by object file
    for source, headers in SOURCES.items():
        own = check and source in CHECK_SOURCES
        obj = os.path.join(OBJ_DIR, source[:-3] + ('_check.o' if own else '.o'))
        inputs[obj] = [os.path.join(CSRC, f) for f in [source] + headers]
        cmds[obj] = [nvcc] + (['-Xptxas', '-v'] if verbose else []) + \
            ['-gencode', 'arch=compute_100a,code=sm_100a', '-lineinfo', '-O3', '-std=c++17', '-Xcompiler', '-fPIC', '-c', '-o', obj] + \
            (['-DMM_WITH_CHECK_ENGINE'] if own else []) + [os.path.join(CSRC, source)]
    link = [nvcc, '-gencode', 'arch=compute_100a,code=sm_100a', '-shared', '-Xcompiler', '-fPIC', '-o', path] + list(cmds)
    names = _named(*cmds.values(), link)
    # (a library that came without its record is taken as it is)
    if not force and not _stale(path, [f for files in inputs.values() for f in files]) and _recorded(path) in (None, names):
        if not check:
            _build_binding(False, start)
        return path
    os.makedirs(OBJ_DIR, exist_ok=True)
    text = _run([c for obj, c in cmds.items() if force or _stale(obj, inputs[obj]) or _recorded(obj) != _named(c)], start)
    text += _run([link], start, names)
    if not check:
        text += _build_binding(force, start)
    if verbose:
        print(text)
    return path


def _compiler() -> str:
    """The system's compiler, whatever CXX names: a binding with a C++ library of its own in it would not share torch's."""
    return '/usr/bin/g++' if os.path.exists('/usr/bin/g++') else 'g++'


def built_for(torch_dir: str) -> str:
    """What a binding is good for besides its sources, as it carries it in itself: the torch and the Python whose headers it was compiled with."""
    torch = runpy.run_path(os.path.join(torch_dir, 'version.py'))
    return f'for torch {torch["__version__"]} {torch.get("git_version")}, {sysconfig.get_config_var("SOABI")}.'


def binding_fits(torch_dir: str) -> bool:
    with open(BINDING_PATH, 'rb') as f:
        return built_for(torch_dir).encode() in f.read()


def _build_binding(force: bool, start: float) -> str:
    """Compile the Python binding against the installed torch and the library next to it; returns what the compiler printed. A host that has no torch or no Python.h
    gets the library without it."""
    inputs = [os.path.join(CSRC, BINDING_SOURCE), os.path.join(CSRC, _ABI)]
    torch_spec = importlib.util.find_spec('torch')
    torch_dir = os.path.dirname(torch_spec.origin) if torch_spec is not None else ''
    if not force and not _stale(BINDING_PATH, inputs) and torch_spec is not None and binding_fits(torch_dir):
        return ''
    cxx = _compiler()
    include = [os.path.join(torch_dir, 'include'), os.path.join(torch_dir, 'include', 'torch', 'csrc', 'api', 'include'), '/usr/local/cuda/include',
               sysconfig.get_paths()['include']]
    needs = [('torch', os.path.join(include[0], 'ATen')), ("Python's header", os.path.join(include[3], 'Python.h')), ('a C++ compiler', shutil.which(cxx) or '')]
    missing = [what for what, path in needs if not os.path.exists(path)]
    if missing:
        # the library is complete without it; a binding of older sources, or for another torch, must not stay
        if os.path.exists(BINDING_PATH):
            os.remove(BINDING_PATH)
        text = f'{os.path.basename(BINDING_PATH)} is not built, for want of {" and ".join(missing)}: the operators around the layer are to be had through the C ABI only'
        warnings.warn(text)
        return text + '\n'
    os.makedirs(OBJ_DIR, exist_ok=True)
    return _run([[cxx, '-O2', '-std=c++17', '-shared', '-fPIC', '-fvisibility=hidden', f'-DMM_BUILT_FOR="{built_for(torch_dir)}"', '-o', BINDING_PATH] + [f'-I{i}' for i in include] +
                 [inputs[0], f'-L{PKG_DIR}', f'-l:{LIB_NAME}', f'-L{os.path.join(torch_dir, "lib")}', '-lc10', '-lc10_cuda', '-ltorch_cpu', '-ltorch_cuda',
                  '-ltorch_python', '-Wl,-rpath,$ORIGIN']], start)


if __name__ == '__main__':
    print(build(force=True, verbose=True))
