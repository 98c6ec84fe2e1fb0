"""Build libsg2im_hip.so (gfx950) in-tree with hipcc.  No torch involved: the library is a
plain C-ABI shared object (include/sg2im_hip.h) loaded through ctypes.  Next to it lib/sg2im_native.so, a host-only
module against torch: checks, buffers and autograd nodes around some of its entry points (csrc/native.cpp)."""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, 'csrc')
LIBDIR = os.path.join(HERE, 'lib')
LIB = os.path.join(LIBDIR, 'libsg2im_hip.so')
SOURCES = ['conv.hip', 'graph.hip', 'gconv.hip', 'gcn_persist.hip', 'heads.hip', 'norm.hip', 'layout.hip', 'loss.hip',
           'groupnorm.hip', 'linear.hip', 'linear_dw.hip']
NATIVE = os.path.join(LIBDIR, 'sg2im_native.so')
INCLUDES = {}      # (.hip files another translation unit includes: none)
# (packed fp32 arithmetic off: hipcc -O3 forms v_pk_{add,mul,fma}_f32 from ordinary float code, and some of their forms have
# given wrong results now and then; the host pass does not know the feature and says so, which is harmless)
FLAGS = ['--offload-arch=gfx950', '-O3', '-std=c++17', '-fPIC', '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops',
         '-I' + os.path.join(ROOT, 'include'), '-I' + CSRC]


def _stale(target, deps):
  if not os.path.exists(target):
    return True
  t = os.path.getmtime(target)
  return any(os.path.getmtime(d) > t for d in deps)


def build_native(force=False, verbose=True):
  """lib/sg2im_native.so with the host compiler (csrc/native.cpp holds no device code)"""
  import sysconfig
  src = os.path.join(CSRC, 'native.cpp')
  if not (force or _stale(NATIVE, [src, os.path.join(ROOT, 'include', 'sg2im_hip.h'), os.path.abspath(__file__)])):
    return None
  import torch
  inc = os.path.join(os.path.dirname(torch.__file__), 'include')
  lib = os.path.join(os.path.dirname(torch.__file__), 'lib')
  cmd = ['g++', '-O2', '-std=c++17', '-fPIC', '-shared', '-w', '-D__HIP_PLATFORM_AMD__', '-DUSE_ROCM', '-DTORCH_EXTENSION_NAME=sg2im_native',
         '-D_GLIBCXX_USE_CXX11_ABI=%d' % int(torch._C._GLIBCXX_USE_CXX11_ABI), '-I' + os.path.join(ROOT, 'include'), '-I' + inc,
         '-I' + os.path.join(inc, 'torch', 'csrc', 'api', 'include'), '-I' + sysconfig.get_paths()['include'],
         '-I/opt/rocm/include', src, '-o', NATIVE, '-L' + lib, '-ltorch', '-ltorch_cpu', '-ltorch_python', '-lc10', '-lc10_hip']
  if verbose:
    print(' '.join(cmd), flush=True)
  return subprocess.Popen(cmd)


def build(force=False, verbose=True, cflags=(), tag=''):
  """tag/cflags: experimental variants, e.g. build(cflags=['-DSG2IM_LDS_STAGES=1'], tag='_lds1')
  -> lib/libsg2im_hip_lds1.so, selected at run time with SG2IM_LIB=<path>."""
  hipcc = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')
  os.makedirs(LIBDIR, exist_ok=True)
  lib_path = LIB.replace('.so', tag + '.so')
  headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith('.h')]
  headers += [os.path.join(ROOT, 'include', 'sg2im_hip.h'), os.path.abspath(__file__)]      # (the flags are here)
  objs, procs = [], []
  for src in SOURCES:
    sp = os.path.join(CSRC, src)
    op = os.path.join(LIBDIR, src.replace('.hip', tag + '.o'))
    objs.append(op)
    if force or _stale(op, [sp] + headers + [os.path.join(CSRC, f) for f in INCLUDES.get(src, ())]):
      cmd = [hipcc] + FLAGS + list(cflags) + ['-c', sp, '-o', op]
      if verbose:
        print(' '.join(cmd), flush=True)
      procs.append((src, subprocess.Popen(cmd)))
  native = build_native(force, verbose) if not tag else None
  for src, pr in procs:
    if pr.wait() != 0:
      raise RuntimeError('hipcc failed on %s' % src)
  if native is not None and native.wait() != 0:
    raise RuntimeError('g++ failed on native.cpp')
  if force or procs or _stale(lib_path, objs):
    cmd = [hipcc, '--offload-arch=gfx950', '-shared', '-fPIC', '-o', lib_path] + objs
    if verbose:
      print(' '.join(cmd), flush=True)
    subprocess.check_call(cmd)
  return lib_path


if __name__ == '__main__':
  tag = [a[6:] for a in sys.argv if a.startswith('--tag=')]
  print(build(force='--force' in sys.argv, cflags=[a for a in sys.argv[1:] if a.startswith('-D')],
              tag=tag[0] if tag else ''))
