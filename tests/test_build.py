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


FAKE_BINDING = """#!{python}
import os, sys
with open({log!r}, 'a') as f:
    f.write('binding\\n')
with open(sys.argv[sys.argv.index('-o') + 1], 'w') as f:
    f.write(' '.join(sys.argv))
"""


@pytest.fixture
def versions(tree, tmp_path):
    """A torch of a version that can be set, and a compiler that leaves its command in what it makes."""
    (tmp_path / 'g++').write_text(FAKE_BINDING.format(python=sys.executable, log=str(tmp_path / 'log')))
    torch_dir = tmp_path / 'torch'
    (torch_dir / 'include' / 'ATen').mkdir(parents=True)
    (torch_dir / '__init__.py').write_text('')
    import importlib.util
    find = importlib.util.find_spec
    spec = importlib.util.spec_from_file_location('torch', str(torch_dir / '__init__.py'))
    tree.patch.setattr(importlib.util, 'find_spec', lambda name, *a: spec if name == 'torch' else find(name, *a))

    def set_version(v):
        (torch_dir / 'version.py').write_text(f'__version__ = {v!r}\ngit_version = "abc"\n')
        tree.age(torch_dir / 'version.py')
    set_version('2.0')
    return set_version


def test_binding_goes_with_torch_and_python(tree, versions, tmp_path):
    """Built again for another torch or Python although its sources are older; not without a reason."""
    assert 'binding' in tree.built()
    assert tree.built() == []
    versions('2.1')
    assert tree.built() == ['binding'] and tree.built() == []
    assert b.binding_fits(str(tmp_path / 'torch'))
    get = sysconfig.get_config_var
    tree.patch.setattr(sysconfig, 'get_config_var', lambda name: 'cpython-399' if name == 'SOABI' else get(name))
    assert not b.binding_fits(str(tmp_path / 'torch'))
    assert tree.built() == ['binding'] and tree.built() == []


def test_a_binding_that_fits_stays_without_headers(tree, versions, tmp_path):
    assert 'binding' in tree.built()
    paths = dict(sysconfig.get_paths(), include=str(tmp_path / 'nowhere'))
    tree.patch.setattr(sysconfig, 'get_paths', lambda *a, **k: paths)
    with warnings.catch_warnings():
        warnings.simplefilter('error')
        assert tree.built() == []
    assert os.path.exists(tmp_path / 'bind.so')
    versions('2.1')                            # and goes where it does not fit and cannot be built
    with pytest.warns(UserWarning):
        assert tree.built() == []
    assert not os.path.exists(tmp_path / 'bind.so')


def test_the_package_does_not_load_a_binding_for_another_torch(monkeypatch, tmp_path):
    from hopper_megamoe_basedondeepgemm_b200 import _binding
    other = tmp_path / 'mm_block_binding.so'
    other.write_bytes(b'for torch 1.0 abc, cpython-27.')
    monkeypatch.setattr(b, 'BINDING_PATH', str(other))
    monkeypatch.setattr(_binding, 'BINDING_PATH', str(other))
    with pytest.raises(RuntimeError, match='another torch'):
        _binding._Binding().block_norm


LIBRARY = ['nvcc a', 'nvcc b', 'nvcc lib']


def test_only_what_changed_is_compiled(tree, tmp_path, versions):
    assert tree.built() == ['binding'] + LIBRARY and tree.built() == []
    (tmp_path / 'csrc' / 'a.h').write_text('x')
    os.utime(tmp_path / 'csrc' / 'a.h', (2e9, 2e9))
    assert tree.built() == ['nvcc a', 'nvcc lib']
    tree.age(tmp_path / 'csrc' / 'a.h')
    assert tree.built() == []
    assert tree.built(force=True, verbose=True) == ['binding'] + LIBRARY and tree.built() == []
    assert tree.built(check=True) == ['nvcc a_check', 'nvcc lib_check'] and tree.built(check=True) == []


def test_what_a_stopped_compiler_leaves_is_not_taken(tree, tmp_path, versions):
    """Its file is newer than the source, and not complete."""
    (tmp_path / 'break').write_text('')
    with pytest.raises(RuntimeError):
        tree.built()
    assert not os.path.exists(tmp_path / 'obj' / 'a.o') and not os.path.exists(tmp_path / 'lib.so')
    (tmp_path / 'break').unlink()
    assert tree.built() == ['binding'] + LIBRARY
    assert not [f for _, _, files in os.walk(tmp_path) for f in files if f.endswith('.part')]


def test_other_commands_make_other_files(tree, tmp_path, versions, monkeypatch):
    """Another compiler: all again. The same tree in another place: nothing. A library that came without objects and records is taken as it is."""
    tree.built()
    (tmp_path / 'nvcc2').write_text((tmp_path / 'nvcc').read_text())
    (tmp_path / 'nvcc2').chmod(0o755)
    monkeypatch.setenv('NVCC', str(tmp_path / 'nvcc2'))
    assert tree.built() == LIBRARY and tree.built() == []
    for f in os.listdir(tmp_path / 'obj'):
        os.unlink(tmp_path / 'obj' / f)
    assert tree.built() == []
    os.unlink(tmp_path / 'lib.so')
    assert tree.built() == LIBRARY


def test_a_source_that_changes_while_it_is_compiled(tree, tmp_path, versions):
    """What is made of it is older than it."""
    fake = (tmp_path / 'nvcc').read_text()
    (tmp_path / 'nvcc').write_text(fake + f"if out.split('/')[-1].startswith('a.o'):\n    os.utime({str(tmp_path / 'csrc' / 'a.cu')!r})\n")
    assert 'nvcc a' in tree.built()
    (tmp_path / 'nvcc').write_text(fake)
    assert tree.built() == ['nvcc a', 'nvcc lib'] and tree.built() == []
