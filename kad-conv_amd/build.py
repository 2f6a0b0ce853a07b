"""Builds libkadconv_hip.so (gfx950) and the torch binding _native.so in-tree from csrc/.

    python kad-conv_amd/build.py            # incremental
    python kad-conv_amd/build.py --force    # rebuild everything

Objects go to kad-conv_amd/_build/, the shared libraries to
kad-conv_amd/kadconv/, where kadconv._ext loads them.
"""
import argparse
import concurrent.futures as cf
import glob
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, 'csrc')
OBJ = os.path.join(HERE, '_build')
LIB = os.path.join(HERE, 'kadconv', 'libkadconv_hip.so')
NATIVE_SRC = os.path.join(CSRC, 'torch', 'kad_torch.cpp')
NATIVE_SRCS = sorted(glob.glob(os.path.join(CSRC, 'torch', '*.cpp')))
NATIVE = os.path.join(HERE, 'kadconv', '_native.so')
INCLUDE = os.path.join(os.path.dirname(HERE), 'include')
HIPCC = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')
ARCH = 'gfx950'
# Packed FP32 VALU ops are disabled for all device code (see the kernels' notes).
FLAGS = ['-O3', '-std=c++17', '-fPIC', f'--offload-arch={ARCH}', '-I', CSRC, '-I', INCLUDE,
         '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops', '-Wno-unused-result']


def _deps():
    return glob.glob(os.path.join(CSRC, '*.h')) + [os.path.join(INCLUDE, 'kadconv_hip.h')]


def _compile(src, force):
    obj = os.path.join(OBJ, os.path.basename(src) + '.o')
    newest = max([os.path.getmtime(src)] + [os.path.getmtime(d) for d in _deps()])
    if not force and os.path.exists(obj) and os.path.getmtime(obj) >= newest:
        return obj, None
    cmd = [HIPCC] + FLAGS + ['-c', src, '-o', obj]
    if src.endswith('.cpp'):
        cmd[1:1] = ['-x', 'hip']
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        return obj, f'{" ".join(cmd)}\n{r.stdout}\n{r.stderr}'
    return obj, None


def _compile_native(force, src=NATIVE_SRC):
    """An object of the binding: host code only, against torch's headers.  What it was built for is recorded beside it:
    these headers' classes change from one version of torch to the next."""
    import torch
    from torch.utils import cpp_extension
    obj = os.path.join(OBJ, os.path.basename(src) + '.o')
    dirs = cpp_extension.include_paths() + ['/opt/rocm/include', sysconfig.get_paths()['include']]
    # the platform's name is what HIP's own headers ask for outside hipcc
    cmd = ['g++', '-O2', '-std=c++17', '-fPIC', '-D__HIP_PLATFORM_AMD__', '-DUSE_ROCM', '-I', INCLUDE]
    cmd += [w for d in dirs for w in ('-isystem', d)] + ['-c', src, '-o', obj]
    built_for = '\n'.join([f'torch {torch.__version__}', f'hip {torch.version.hip}', str(sysconfig.get_config_var('SOABI')),
                           ' '.join(cmd)])
    record = obj + '.for'
    newest = max(os.path.getmtime(f) for f in [src, *glob.glob(os.path.join(CSRC, 'torch', '*.h')), *_deps()])
    if not force and os.path.exists(obj) and os.path.getmtime(obj) >= newest and os.path.exists(record):
        with open(record) as f:
            if f.read() == built_for:
                return obj, None
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode:
        return obj, f'{" ".join(cmd)}\n{r.stdout}\n{r.stderr}'
    with open(record, 'w') as f:
        f.write(built_for)
    return obj, None


def _link_native(objs):
    import torch
    libs = os.path.join(os.path.dirname(torch.__file__), 'lib')
    tmp = NATIVE + '.tmp'
    cmd = ['g++', '-shared', '-o', tmp, *objs, '-L', os.path.dirname(LIB), '-l:' + os.path.basename(LIB), '-L', libs,
           '-lc10', '-lc10_hip', '-ltorch_cpu', '-ltorch_hip', '-ltorch', '-ltorch_python', '-Wl,-rpath,$ORIGIN']
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f'link failed:\n{" ".join(cmd)}\n{r.stdout}\n{r.stderr}')
    os.replace(tmp, NATIVE)


def build(force=False, jobs=8, verbose=False):
    os.makedirs(OBJ, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, '*.hip')) + glob.glob(os.path.join(CSRC, '*.cpp')))
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        native = [ex.submit(_compile_native, force, s) for s in NATIVE_SRCS]
        results = list(ex.map(lambda s: _compile(s, force), srcs))
    native = [n.result() for n in native]
    errs = [e for _, e in results + native if e]
    if errs:
        raise RuntimeError('HIP build failed:\n' + '\n'.join(errs))
    objs = [o for o, _ in results]
    if force or not os.path.exists(LIB) or os.path.getmtime(LIB) < max(os.path.getmtime(o) for o in objs):
        tmp = LIB + '.tmp'
        cmd = [HIPCC, f'--offload-arch={ARCH}', '-shared', '-fPIC', '-o', tmp] + objs
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f'link failed:\n{" ".join(cmd)}\n{r.stdout}\n{r.stderr}')
        os.replace(tmp, LIB)
    native = [o for o, _ in native]
    if force or not os.path.exists(NATIVE) or os.path.getmtime(NATIVE) < max(os.path.getmtime(o) for o in native):
        _link_native(native)
    if verbose:
        print('built', LIB, 'and', NATIVE)
    return LIB


if __name__ == '__main__':
    ap = argparse.ArgumentParser()
    ap.add_argument('--force', action='store_true')
    ap.add_argument('-j', type=int, default=8)
    args = ap.parse_args()
    build(force=args.force, jobs=args.j, verbose=True)
    sys.exit(0)
