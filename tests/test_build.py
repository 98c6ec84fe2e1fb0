"""CPU: what is compiled when."""
import os

import pytest


@pytest.fixture
def commands(monkeypatch):
  """build.build()'s compile commands, none of which is run"""
  from sg2im_amd import build
  cmds = []

  class NoProcess(object):
    def __init__(self, cmd):
      cmds.append(cmd)

    def wait(self):
      return 0
  monkeypatch.setattr(build.subprocess, 'Popen', NoProcess)
  monkeypatch.setattr(build.subprocess, 'check_call', lambda cmd: cmds.append(cmd))
  return cmds


def sources(cmds):
  return {os.path.basename(a) for c in cmds for a in c if a.endswith(('.hip', '.cpp'))}


def test_a_change_of_the_flags_compiles_everything_again(commands, monkeypatch):
  from sg2im_amd import build
  os.makedirs(build.LIBDIR, exist_ok=True)
  newest = max([os.path.getmtime(os.path.join(build.LIBDIR, f)) for f in os.listdir(build.LIBDIR)] or [0.0])
  real = os.path.getmtime
  monkeypatch.setattr(build.os.path, 'getmtime', lambda f: newest + 1 if os.path.abspath(f) == os.path.abspath(build.__file__) else real(f))
  build.build(verbose=False)
  assert sources(commands) == set(build.SOURCES) | {'native.cpp'}


def test_the_entry_point_always_compiles(commands, monkeypatch):
  import __graft_entry__
  from sg2im_amd import build
  if not (os.path.exists(build.LIB) and os.path.exists(build.NATIVE)):
    pytest.skip('nothing is built that the entry point could load')
  monkeypatch.setattr(build.os.path, 'getmtime', lambda f: 0.0)            # (nothing is older than anything)
  __graft_entry__.build()
  assert sources(commands) == set(build.SOURCES) | {'native.cpp'}
  assert all('-packed-fp32-ops' in c for c in commands if any(a.endswith('.hip') for a in c))
