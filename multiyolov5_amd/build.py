"""Build libmyolo.so (the gfx950 HIP kernels + C ABI) in-tree with hipcc.  No JIT cache: the .so travels with the repo
snapshot to the GPU box; it is git-ignored."""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, 'csrc')
LIB = os.path.join(HERE, 'lib', 'libmyolo.so')
EXT = os.path.join(HERE, 'lib', '_token_autograd.so')           # autograd nodes of utils/tokens.py (host C++ over the C ABI)
EXT_SRC = os.path.join(CSRC, 'token_autograd.cpp')
ARCH = 'gfx950'


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith('.hip'))


def stale_ext():
    hdr = os.path.join(os.path.dirname(HERE), 'include', 'myolo.h')
    return not os.path.exists(EXT) or os.path.getmtime(EXT) < max(os.path.getmtime(EXT_SRC), os.path.getmtime(hdr))


def build_ext(verbose=True):
    import sysconfig
    import torch
    from torch.utils.cpp_extension import include_paths, library_paths
    inc = include_paths() + ['/opt/rocm/include', sysconfig.get_paths()['include']]
    cmd = ['g++', '-O2', '-std=c++17', '-fPIC', '-shared', '-D__HIP_PLATFORM_AMD__=1', '-DTORCH_EXTENSION_NAME=_token_autograd',
           f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}'] + [f'-I{p}' for p in inc] + [EXT_SRC] + \
        [f'-L{p}' for p in library_paths()] + ['-ltorch_python', '-ltorch', '-ltorch_cpu', '-lc10', '-lc10_hip', '-o', EXT]
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    if r.returncode != 0:
        raise RuntimeError('%s\n%s' % (' '.join(cmd), r.stdout.decode()))
    if verbose:
        print('built', EXT)


def stale():
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = sources() + [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith('.h')] + \
        [os.path.join(os.path.dirname(HERE), 'include', 'myolo.h')]
    return any(os.path.getmtime(d) > t for d in deps)


# no v_pk_{add,mul,fma}_f32 anywhere: scalar fp32 instructions give the same IEEE results
NO_PACKED_F32 = ['-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']
# augment.hip restates C code compiled for baseline x86-64 (Pillow / OpenCV float arithmetic): a fused multiply-add changes the
# truncated uint8 results.  hipcc's default -ffp-contract=fast ignores source pragmas, so the whole file is built without contraction.
PER_FILE_FLAGS = {'augment.hip': ['-ffp-contract=off']}


def build(force=False, verbose=True):
    if force or stale_ext():
        os.makedirs(os.path.dirname(EXT), exist_ok=True)
        build_ext(verbose)
    if not force and not stale():
        return LIB
    hipcc = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')
    os.makedirs(os.path.dirname(LIB), exist_ok=True)
    objs = []
    procs = []
    hdrs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith('.h')] + \
        [os.path.join(os.path.dirname(HERE), 'include', 'myolo.h')]
    hdr_t = max(os.path.getmtime(h) for h in hdrs)
    for src in sources():
        obj = os.path.join(HERE, 'lib', os.path.basename(src)[:-4] + '.o')
        objs.append(obj)
        if not force and os.path.exists(obj) and os.path.getmtime(obj) > max(os.path.getmtime(src), hdr_t):
            continue                                     # object is newer than its source and every header
        cmd = [hipcc, f'--offload-arch={ARCH}', '-O3', '-std=c++17', '-fPIC'] + NO_PACKED_F32 + PER_FILE_FLAGS.get(os.path.basename(src), []) + ['-c', src, '-o', obj]
        procs.append((cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
    for cmd, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            raise RuntimeError('hipcc failed: %s\n%s' % (' '.join(cmd), out.decode()))
        text = '\n'.join(ln for ln in out.decode().splitlines() if 'packed-fp32-ops' not in ln)   # (the host pass does not know the feature)
        if verbose and text.strip():
            print(text)
    cmd = [hipcc, f'--offload-arch={ARCH}', '-shared', '-fPIC', '-o', LIB] + objs
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    if r.returncode != 0:
        raise RuntimeError('link failed:\n' + r.stdout.decode())
    if verbose:
        print('built', LIB)
    return LIB


if __name__ == '__main__':
    build(force='--force' in sys.argv)
