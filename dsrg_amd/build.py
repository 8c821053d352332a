"""Build libdsrg_hip.so for gfx950 with hipcc (cross-compiles without a GPU) and the host module _dsrg_bind.so.

    python -m dsrg_amd.build [--force]
"""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, 'csrc')
LIB = os.path.join(CSRC, 'libdsrg_hip.so')
BIND = os.path.join(CSRC, '_dsrg_bind.so')          # CPython module (bind.cpp): native host side of the serving operators
SOURCES = ['gemm.hip', 'rowops.hip', 'attention.hip', 'train.hip', 'train_rows.hip', 'graphmap.hip', 'optim.hip', 'kvcache.hip', 'sample.hip']
HEADERS = ['common.h', os.path.join('..', '..', 'include', 'dsrg_hip.h')]

# gfx950's packed fp32 instructions (v_pk_fma_f32 and its like) are left out of the compiler's choice: some of their forms have given
# wrong results on this hardware now and then
NO_PACKED_FP32 = ['-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']


def _stale():
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    if not os.path.exists(BIND) or os.path.getmtime(os.path.join(CSRC, 'bind.cpp')) > os.path.getmtime(BIND):
        return True
    return any(os.path.getmtime(os.path.join(CSRC, f)) > t for f in SOURCES + HEADERS)


def _bind_command():
    """host code only, against this interpreter's and this torch's headers (HIP's headers want to be told the platform by a compiler that
    is not hipcc)"""
    import sysconfig
    import torch
    t = os.path.dirname(torch.__file__)
    inc = [os.path.join(t, 'include'), os.path.join(t, 'include', 'torch', 'csrc', 'api', 'include'), '/opt/rocm/include', sysconfig.get_paths()['include']]
    return [os.environ.get('CXX', 'g++'), '-O2', '-std=c++17', '-fPIC', '-shared', '-D__HIP_PLATFORM_AMD__=1', '-DUSE_ROCM=1', *['-isystem' + i for i in inc],
            os.path.join(CSRC, 'bind.cpp'), '-o', BIND, '-L' + os.path.join(t, 'lib'), '-ltorch_python', '-ltorch_cpu', '-lc10', '-lc10_hip']


def build(force=False, verbose=True):
    if not force and not _stale():
        return LIB
    hipcc = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')
    objs = []
    procs = []
    for src in SOURCES:
        obj = os.path.join(CSRC, src.replace('.hip', '.o'))
        cmd = [hipcc, '-O3', '-std=c++17', '--offload-arch=gfx950', '-fPIC', *NO_PACKED_FP32, '-c', os.path.join(CSRC, src), '-o', obj]
        if verbose:
            print(' '.join(cmd), flush=True)
        procs.append((src, subprocess.Popen(cmd)))
        objs.append(obj)
    cmd = _bind_command()
    if verbose:
        print(' '.join(cmd), flush=True)
    procs.append(('bind.cpp', subprocess.Popen(cmd)))
    for src, p in procs:
        if p.wait() != 0:
            raise RuntimeError('the compiler failed on %s' % src)
    cmd = [hipcc, '--offload-arch=gfx950', '-shared', '-fPIC', '-o', LIB] + objs
    if verbose:
        print(' '.join(cmd), flush=True)
    subprocess.check_call(cmd)
    return LIB


if __name__ == '__main__':
    print(build(force='--force' in sys.argv))
