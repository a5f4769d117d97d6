"""When the extension module of the paged cache is built: for another torch anew, without torch not at all (the compiler is a fake)."""
import importlib.util
import os
import sys
from types import SimpleNamespace

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'hyperattention_b200', 'csrc')


@pytest.fixture
def build(monkeypatch, tmp_path):
    spec = importlib.util.spec_from_file_location('build_of_a_copy', os.path.join(CSRC, 'build.py'))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    (tmp_path / 'csrc').mkdir()
    (tmp_path / 'csrc' / 'paged_ext.cpp').write_text('')
    (tmp_path / 'include').mkdir()
    (tmp_path / 'include' / 'hyperattn_b200.h').write_text('')
    monkeypatch.setattr(mod, 'HERE', str(tmp_path / 'csrc'))
    monkeypatch.setattr(mod, 'ROOT', str(tmp_path))
    monkeypatch.setattr(mod, 'EXT', str(tmp_path / '_paged_ext.so'))
    mod.calls = []

    def run(cmd, **kw):
        mod.calls.append(cmd)
        open(mod.EXT, 'w').close()
        return SimpleNamespace(returncode=0, stdout='', stderr='')

    monkeypatch.setattr(mod, 'subprocess', SimpleNamespace(run=run))
    return mod


def test_another_torch(build, monkeypatch):
    for _ in range(2):
        assert build.build_ext() == build.EXT
    assert len(build.calls) == 1
    monkeypatch.setattr('importlib.metadata.version', lambda name: '0.0.1')
    for _ in range(2):
        build.build_ext()
    assert len(build.calls) == 2


def test_a_module_of_unknown_torch(build):
    open(build.EXT, 'w').close()
    build.build_ext()
    assert len(build.calls) == 1


def test_no_torch(build, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, 'torch', None)
    assert build.build_ext() is None and not build.calls
    assert 'not installed' in capsys.readouterr().err
