"""The build of the library and of its Python binding, with compilers that only write down that they were called."""
import os
import sys
import sysconfig
import warnings

import pytest

from hopper_megamoe_basedondeepgemm_b200 import build as b

FAKE = """#!{python}
import os, sys
out = sys.argv[sys.argv.index('-o') + 1]
log = os.path.join({folder!r}, 'log')
with open(log, 'a') as f:
    f.write({name!r} + ' ' + os.path.basename(out).split('.')[0] + '\\n')
with open(out, 'w') as f:
    f.write('made by {name}')
if os.path.exists(os.path.join({folder!r}, 'break')):
    sys.exit(1)
"""


class Tree:
    """A package of two CUDA sources and a binding in a folder of its own."""

    def __init__(self, folder, monkeypatch):
        self.folder, self.patch = folder, monkeypatch
        csrc = folder / 'csrc'
        csrc.mkdir()
        for f in ('a.cu', 'b.cu', 'a.h', 'bind.cpp', 'abi.h'):
            (csrc / f).write_text('')
            self.age(csrc / f)
        for name in ('nvcc', 'g++'):
            (folder / name).write_text(FAKE.format(python=sys.executable, folder=str(folder), name=name))
            (folder / name).chmod(0o755)
        for k, v in dict(PKG_DIR=str(folder), CSRC=str(csrc), LIB_PATH=str(folder / 'lib.so'), CHECK_LIB_PATH=str(folder / 'lib_check.so'), BINDING_PATH=str(folder / 'bind.so'),
                         BINDING_SOURCE='bind.cpp', _ABI='abi.h', SOURCES={'a.cu': ['a.h'], 'b.cu': []}, CHECK_SOURCES=('a.cu',), OBJ_DIR=str(folder / 'obj')).items():
            monkeypatch.setattr(b, k, v)
        monkeypatch.setenv('NVCC', str(folder / 'nvcc'))
        monkeypatch.setattr(b, '_compiler', lambda: str(folder / 'g++'), raising=False)

    def age(self, path):
        os.utime(path, (1e9, 1e9))

    def built(self, **kw):
        """What a call of build compiles and links, in order of name."""
        log = self.folder / 'log'
        if log.exists():
            log.unlink()
        b.build(**kw)
        return sorted(log.read_text().split('\n')[:-1]) if log.exists() else []


@pytest.fixture
def tree(tmp_path, monkeypatch):
    return Tree(tmp_path, monkeypatch)


def test_library_without_python_headers(tree, tmp_path):
    """A host that has no Python.h gets the library, and is told that the binding is missing; one of older sources does not stay."""
    tree.patch.setattr(b, '_compiler', lambda: 'g++', raising=False)
    (tmp_path / 'csrc' / 'bind.cpp').write_text('#include <Python.h>\n')
    (tmp_path / 'bind.so').write_text('older')
    tree.age(tmp_path / 'bind.so')
    paths = dict(sysconfig.get_paths(), include=str(tmp_path / 'nowhere'))
    tree.patch.setattr(sysconfig, 'get_paths', lambda *a, **k: paths)
    with warnings.catch_warnings(record=True) as seen:
        warnings.simplefilter('always')
        assert b.build() == str(tmp_path / 'lib.so')
    assert os.path.exists(tmp_path / 'lib.so') and not os.path.exists(tmp_path / 'bind.so')
    assert any('Python' in str(w.message) for w in seen)
