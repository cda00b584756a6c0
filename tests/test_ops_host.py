"""The operators of include/gsage_ops.h without a GPU: what is declared is bound, exported and driven by the validation
program, which runs under AddressSanitizer + UndefinedBehaviorSanitizer; and the Python side refuses host tensors."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from graphsage_amd import _lib, kernels

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _declared():
    header = open(os.path.join(ROOT, 'include', 'gsage_ops.h')).read()
    header = re.sub(r'/\*.*?\*/', '', header, flags=re.S)
    return set(re.findall(r'\b(gs_[a-z0-9_]+)\s*\(', header))


def test_declared_bound_and_exported():
    assert _declared() == set(_lib.SIGNATURES_OPS)
    lib = ctypes.CDLL(_lib.LIB_PATH)
    for name in _declared():
        assert hasattr(lib, name), name


def test_argument_checks_are_clean_under_asan_and_ubsan():
    subprocess.check_call(['make', '-C', os.path.join(ROOT, 'graphsage_amd', 'csrc'), 'asan', '-j8'],
                          stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
    env = dict(os.environ, ASAN_OPTIONS='detect_leaks=0:abort_on_error=0', UBSAN_OPTIONS='print_stacktrace=1')
    env.pop('LD_PRELOAD', None)                       # the sanitizer runtime must come first in the process
    res = subprocess.run([os.path.join(ROOT, 'tests', 'abi', 'ops_validate')], capture_output=True, text=True, env=env, timeout=300)
    assert res.returncode == 0, (res.stdout[-3000:], res.stderr[-3000:])
    assert 'ops_validate ok' in res.stdout
    assert 'runtime error' not in res.stderr and 'AddressSanitizer' not in res.stderr


def test_every_declared_entry_point_is_validated():
    used = set(re.findall(r'\b(gs_[a-z0-9_]+)\s*\(', open(os.path.join(ROOT, 'tests', 'abi', 'ops_validate.cpp')).read()))
    assert _declared() - used == set()


def test_host_tensors_are_refused():
    x = torch.zeros(4, 2, 8)
    for call in (lambda: kernels.dropout(x, 0.5, 1),
                 lambda: kernels.neighbor_attention(x, x, None, None, 1),
                 lambda: kernels.neighbor_inverse(torch.zeros(4, dtype=torch.int32), 4),
                 lambda: kernels.catalog_log_probs(x[0], x[1])):
        with pytest.raises(_lib.GsageError):
            call()
    with pytest.raises(TypeError):
        kernels.catalog_log_probs([1.0], [2.0])
