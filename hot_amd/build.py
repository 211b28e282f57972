"""Build libhotk.so in-tree with hipcc for gfx950, and hot_amd/_ffn beside it (`python -m hot_amd.build`).

One object per csrc/*.hip (compiled in parallel, only when the source or a header is newer), linked into
hot_amd/libhotk.so.  Objects live under hot_amd/csrc/_obj/ (git-ignored)."""
import glob
import hashlib
import os
import re
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
OUT = os.path.join(HERE, 'libhotk.so')
OBJ = os.path.join(HERE, 'csrc', '_obj')
FLAGS = ['--offload-arch=gfx950', '-O3', '-std=c++17', '-fPIC', '-Wno-unused-value',
         '-mllvm', '-amdgpu-mfma-vgpr-form',   # MFMA results in VGPRs: no v_accvgpr_read/write around the tile code
         # no packed fp32 arithmetic: -O3 forms v_pk_{add,mul,fma}_f32 from ordinary float code by itself, and some of their
         # operand forms have given wrong results now and then (the host pass warns that it does not know the feature)
         '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']


def sources():
    return sorted(glob.glob(os.path.join(HERE, 'csrc', '*.hip')))


def _headers():
    return glob.glob(os.path.join(HERE, 'csrc', '*.h')) + [os.path.join(HERE, '..', 'include', 'hotk.h')]


def _src_time(src):
    """mtime of a source and of the csrc files it includes by name (gemm6_n128.hip is a second build of gemm6.hip)"""
    t = os.path.getmtime(src)
    for m in re.finditer(r'^#include "([^"]+\.hip)"', open(src).read(), re.M):
        inc = os.path.join(os.path.dirname(src), m.group(1))
        if os.path.exists(inc):
            t = max(t, os.path.getmtime(inc))
    return t


def build(force=False, verbose=True, extra_flags=(), out=OUT):
    """extra_flags / out: A/B builds of the same ABI (load with HOTK_LIB=<out>)"""
    srcs = sources()
    hdr_time = max(os.path.getmtime(h) for h in _headers())
    hipcc = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')
    tag = '' if out == OUT else '.' + os.path.basename(out)
    os.makedirs(OBJ, exist_ok=True)
    # objects are reused only when they were compiled by the same compiler with the same flags: the stamp holds a hash
    # of (hipcc, FLAGS + extra_flags), so an A/B build with other flags under the same name never measures stale code
    cfg = hashlib.sha256('\0'.join([hipcc] + FLAGS + list(extra_flags)).encode()).hexdigest()
    stamp = os.path.join(OBJ, 'flags' + tag + '.stamp')
    if not os.path.exists(stamp) or open(stamp).read() != cfg:
        force = True
    jobs = []
    for s in srcs:
        o = os.path.join(OBJ, os.path.basename(s)[:-4] + tag + '.o')
        if force or not os.path.exists(o) or os.path.getmtime(o) < max(_src_time(s), hdr_time):
            jobs.append([hipcc] + FLAGS + list(extra_flags) + ['-c', s, '-o', o])
    objs = [os.path.join(OBJ, os.path.basename(s)[:-4] + tag + '.o') for s in srcs]
    if not jobs and os.path.exists(out) and all(os.path.getmtime(out) >= os.path.getmtime(o) for o in objs):
        return out

    def run(cmd):
        if verbose:
            print(' '.join(cmd), flush=True)
        subprocess.check_call(cmd)

    with ThreadPoolExecutor(max_workers=min(8, max(len(jobs), 1))) as ex:
        list(ex.map(run, jobs))
    link_extra = [f for f in extra_flags if f.startswith(('-L', '-l', '-Wl,', '-fsanitize', '-g'))]
    run([hipcc, '--offload-arch=gfx950', '-shared', '-fPIC', '-o', out] + link_extra + objs)
    with open(stamp, 'w') as f:
        f.write(cfg)
    return out


EXT_SRC = os.path.join(HERE, 'csrc', 'ffn_torch.cpp')
EXT_OUT = os.path.join(HERE, '_ffn' + sysconfig.get_config_var('EXT_SUFFIX'))


def build_ext(force=False, verbose=True):
    """hot_amd/_ffn: the compiled host side of the feed-forward operators (torch's C++ interface; host code only).  It takes
    libhotk's entries from the running process, so it is linked against torch alone."""
    import torch
    from torch.utils import cpp_extension
    newest = max(os.path.getmtime(f) for f in (EXT_SRC, os.path.join(HERE, '..', 'include', 'hotk.h')))
    if not force and os.path.exists(EXT_OUT) and os.path.getmtime(EXT_OUT) >= newest:
        return EXT_OUT
    lib = os.path.join(os.path.dirname(torch.__file__), 'lib')
    cmd = ['g++', '-O2', '-std=c++17', '-fPIC', '-shared', '-fvisibility=hidden', '-w', '-D__HIP_PLATFORM_AMD__=1', '-DUSE_ROCM=1',
           f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}']
    for d in cpp_extension.include_paths(device_type='cuda') + [sysconfig.get_paths()['include']]:
        cmd += ['-isystem', d]
    cmd += [EXT_SRC, '-o', EXT_OUT, '-L' + lib, '-Wl,-rpath,' + lib, '-lc10', '-lc10_hip', '-ltorch', '-ltorch_cpu', '-ltorch_hip',
            '-ltorch_python']
    if verbose:
        print(' '.join(cmd), flush=True)
    subprocess.check_call(cmd)
    return EXT_OUT


def assembly(src, out, extra_flags=()):
    """device assembly of one source, compiled with the library's own flags (for tests/asm_hazards.py)"""
    hipcc = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')
    subprocess.check_call([hipcc] + FLAGS + list(extra_flags) + ['-S', '--cuda-device-only', '-o', out, src],
                          stderr=subprocess.DEVNULL)
    return out


if __name__ == '__main__':
    build(force='--force' in sys.argv)
    build_ext(force='--force' in sys.argv)
