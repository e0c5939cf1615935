import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line('markers', 'gpu: needs a real MI355X (run with -m gpu)')


@pytest.fixture(scope='session')
def emul():
    """gcc build of the kernels' per-voxel arithmetic (tests/emul), CPU only."""
    import ctypes
    d = os.path.join(ROOT, 'tests', 'emul')
    so = os.path.join(d, '_emul.so')
    deps = [os.path.join(d, 'emul.c'),
            os.path.join(ROOT, 'tempo_amd', 'csrc', 'unproject_math.h')]
    if not os.path.exists(so) or any(os.path.getmtime(p) > os.path.getmtime(so) for p in deps):
        subprocess.run(['gcc', '-O2', '-ffp-contract=off', '-mfma', '-shared', '-fPIC',
                        deps[0], '-o', so, '-lm'], check=True)
    return ctypes.CDLL(so)


@pytest.fixture(scope='session')
def linear_plan():
    """g++ build of the fused linear layer's choice of kernels (tests/emul), CPU only."""
    import ctypes
    d = os.path.join(ROOT, 'tests', 'emul')
    so = os.path.join(d, '_plan.so')
    deps = [os.path.join(d, 'plan.cpp'),
            os.path.join(ROOT, 'tempo_amd', 'csrc', 'linear_plan.h'),
            os.path.join(ROOT, 'include', 'tempo_unproject.h')]
    if not os.path.exists(so) or any(os.path.getmtime(p) > os.path.getmtime(so) for p in deps):
        subprocess.run(['g++', '-O2', '-Wall', '-Werror', '-std=c++17', '-shared', '-fPIC',
                        deps[0], '-o', so], check=True)
    lib = ctypes.CDLL(so)
    ll, i = ctypes.c_longlong, ctypes.c_int
    lib.emul_plan_product.argtypes = [ll] * 3 + [i] * 4 + [ctypes.POINTER(ll)]
    lib.emul_streamable.argtypes = [ll, ll, i, ll, ll, i]
    lib.emul_product_bytes.argtypes = [ll] * 3 + [i] * 3
    lib.emul_product_bytes.restype = ll
    return lib


@pytest.fixture(scope='session')
def gpu_device():
    import torch
    if not torch.cuda.is_available():
        pytest.fail('a gpu-marked test was selected but no HIP device is visible')
    return torch.device('cuda:0')
