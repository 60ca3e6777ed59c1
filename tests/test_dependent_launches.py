"""Kernels that may start before the one in front of them has ended do not declare what it writes read-only: `__ldg` and
`const __restrict__` let a load go past the cache coherence that the wait for that kernel relies on."""
import os
import re

import pytest

import _native as N

CSRC = N._CSRC


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r'//[^\n]*|/\*.*?\*/', '', f.read(), flags=re.S)


def kernels(text):
    """(name, parameters, body) of every __global__ function."""
    for m in re.finditer(r'__global__[^;{]*?(\w+)\(', re.sub(r'__launch_bounds__\((?:[^()]|\([^()]*\))*\)|__cluster_dims__\([^()]*\)', lambda k: ' ' * len(k.group()), text)):
        depth, i = 1, m.end()
        while depth:
            depth += {'(': 1, ')': -1}.get(text[i], 0)
            i += 1
        start = j = text.index('{', i)
        depth = 0
        while True:
            depth += {'{': 1, '}': -1}.get(text[j], 0)
            j += 1
            if not depth:
                break
        yield m.group(1), text[m.end():i - 1], text[start:j]


FILES = [f for f in sorted(os.listdir(CSRC)) if f.endswith(('.cu', '.cuh'))]
WAITING = [(f, *k) for f in FILES for k in kernels(source(f)) if 'grid_dependency_wait' in k[2]]


def test_the_waiting_kernels_are_found():
    assert {k[1] for k in WAITING} >= {'dropout_kernel', 'gate_dropout_fwd_kernel', 'gate_dropout_bwd_kernel', 'add_dropout_norm_fwd_kernel',
                                       'add_dropout_norm_bwd_kernel', 'streamed_ce_kernel', 'streamed_ce_join_kernel', 'streamed_ce_finish_kernel', 'col_sum_kernel'}


@pytest.mark.parametrize('file,name,params,body', WAITING, ids=[k[1] for k in WAITING])
def test_a_waiting_kernel_reads_coherently(file, name, params, body):
    assert '__ldg' not in body and '__restrict__' not in params + body
    for header in re.findall(r'#include "(\w+\.cuh)"', source(file)):
        assert '__ldg' not in source(header) and 'ld.global.nc' not in source(header)
