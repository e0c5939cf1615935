"""Build ``tempo_amd/lib/libtempo_unproject.so`` in-tree with hipcc for gfx950.

    python -m tempo_amd.build [--force]

hipcc cross-compiles without a GPU.  ``-ffp-contract=off`` is part of the
numerical contract of the unprojection (see ``csrc/unproject_math.h``): every fused
multiply-add in its coordinate chain is written out as an explicit ``fmaf``.

Every source is compiled without packed fp32 instructions: ``v_pk_*_f32`` has been seen to
return wrong values now and then, with no error.  (The host pass of hipcc warns that it does
not know the feature; that is harmless.)
"""
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, 'csrc')
HEADER = os.path.join(HERE, '..', 'include', 'tempo_unproject.h')
OUT = os.path.join(HERE, 'lib', 'libtempo_unproject.so')
FLAGS = ['--offload-arch=gfx950', '-O3', '-fPIC', '-std=c++17', '-Wall',
         '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']
# source -> (what it includes, flags of its own)
SOURCES = {
    'tempo_unproject.hip': (['unproject_math.h'], ['-ffp-contract=off']),
    'recurrence.hip': ([], []),
    'linear.hip': (['linear_plan.h'], []),
}


def hipcc_path():
    for cand in (shutil.which('hipcc'), '/opt/rocm/bin/hipcc'):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError('hipcc not found (need ROCm with gfx950 support)')


def _object(source):
    return os.path.join(HERE, 'lib', os.path.splitext(source)[0] + '.o')


def _older(path, deps):
    if not os.path.exists(path):
        return True
    t = os.path.getmtime(path)
    return any(os.path.getmtime(d) > t for d in deps)


def _deps(source):
    return [os.path.join(CSRC, n) for n in [source] + SOURCES[source][0]] + [HEADER]


def stale():
    return any(_older(OUT, _deps(s)) for s in SOURCES)


def build(force=False, verbose=True):
    if not force and not stale():
        return OUT
    os.makedirs(os.path.dirname(OUT), exist_ok=True)
    running = []
    for source, (_, flags) in SOURCES.items():  # all at once: one compiler process each
        if not force and not _older(_object(source), _deps(source)):
            continue
        cmd = ([hipcc_path()] + FLAGS + flags +
               ['-c', os.path.join(CSRC, source), '-o', _object(source)])
        if verbose:
            print(' '.join(cmd), flush=True)
        running.append((cmd, subprocess.Popen(cmd)))
    for code, cmd in [(p.wait(), cmd) for cmd, p in running]:
        if code:
            raise subprocess.CalledProcessError(code, cmd)
    cmd = ([hipcc_path(), '--offload-arch=gfx950', '-shared', '-fPIC'] +
           [_object(s) for s in SOURCES] + ['-o', OUT])
    if verbose:
        print(' '.join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    return OUT


if __name__ == '__main__':
    build(force='--force' in sys.argv)
    print(OUT)
