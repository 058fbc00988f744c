"""__graft_entry__.build(): compiles whether or not a built library is there."""
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_build_compiles_every_time(monkeypatch):
    sys.path.insert(0, ROOT)
    import __graft_entry__
    import oracle
    from oracle import build_ref
    from gendr_amd import _native, build
    forced = []
    monkeypatch.setattr(build, 'build_all', lambda force=False, **kw: forced.append(('library', force)))
    monkeypatch.setattr(build, 'build_torch_ext', lambda force=False, **kw: forced.append(('autograd node', force)))
    monkeypatch.setattr(oracle, 'build', lambda *a, **kw: None)
    monkeypatch.setattr(build_ref, 'build', lambda *a, **kw: None)
    monkeypatch.setattr(_native, 'lib', lambda *a, **kw: None)
    __graft_entry__.build()
    assert forced == [('library', True), ('autograd node', True)]
