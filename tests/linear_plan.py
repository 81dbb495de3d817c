"""
Which tiles a call of grouped_linear takes: the rules of csrc/psh_linear_plan.h, compiled for the CPU.
"""
import collections
import ctypes as C
import functools
import os
import subprocess
import tempfile

from simurlacra_amd import _abi as abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROWS16, T64, T128, T128D, T256D = range(5)
KINDS = ('16 rows', '64', '128', '128 direct', '256 direct')
Plan = collections.namedtuple('Plan', 'forward dx dw joint piece space')
NATIVE = ['-D__host__=', '-D__device__=', '-D__forceinline__=inline', '-I', os.path.join(ROOT, 'simurlacra_amd', 'csrc')]


@functools.lru_cache(None)
def _function():
    with tempfile.TemporaryDirectory() as d:
        so = os.path.join(d, 'plan.so')
        subprocess.check_call(['g++', '-std=c++17', '-O1', '-shared', '-fPIC', *NATIVE, os.path.join(ROOT, 'tests', 'native', 'linear_plan.cpp'), '-o', so])
        f = C.CDLL(so).plan
    f.argtypes, f.restype = [C.POINTER(abi.PshLinearDesc), C.POINTER(C.c_int64)], None
    return f


def plan(desc) -> Plan:
    out = (C.c_int64*6)()
    _function()(C.byref(desc), out)
    return Plan(*out[:3], bool(out[3]), out[4], out[5])


def kernels(p: Plan, want=(True, True, True)):
    """ The kernels of a forward and a backward call: {(kernel, kind of tile)}. """
    got = {('forward', p.forward)}
    if p.joint:
        return got | {('both', p.dw)}
    return got | ({('dx', p.dx)} if want[0] else set()) | ({('dw', p.dw)} if want[1] or want[2] else set())
