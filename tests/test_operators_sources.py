"""
CPU tests of the policy operators' kernel sources: what the compiler has to be told about assembly that is written by hand.
"""
import ctypes
import glob
import os
import re
import subprocess

import pytest

from simurlacra_amd import _abi as abi
from simurlacra_amd.engine import load_library
from tests import layer_cases, linear_plan

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCES = sorted(glob.glob(os.path.join(ROOT, 'simurlacra_amd', 'csrc', 'ops_*.hip')) + [os.path.join(ROOT, 'simurlacra_amd', 'csrc', 'psh_ops.h')])


def _assembly(path):
    """ The arguments of every asm statement of a file. """
    text = open(path).read()
    for at in re.finditer(r'\basm\b(?:\s+volatile)?\s*\(', text):
        depth, k, quoted = 1, at.end(), False
        while depth:
            c = text[k]
            if c == '"' and text[k - 1] != '\\':
                quoted = not quoted
            elif not quoted:
                depth += (c == '(') - (c == ')')
            k += 1
        yield text[at.end():k - 1]


def test_fixed_registers_that_assembly_writes_are_named_to_the_compiler():
    seen = 0
    for path in SOURCES:
        for body in _assembly(path):
            instructions = ''.join(re.findall(r'"((?:[^"\\]|\\.)*)"', body.split(' : ')[0]))
            for register in ('m0', 'vcc', 'exec', 'scc'):
                if re.search(rf'(?:^|\\n|\\t)\s*[a-z_0-9]+\s+{register}\b', instructions):
                    seen += 1
                    assert f'"{register}"' in body, (os.path.basename(path), body)
    assert seen >= 1


def test_rows_slots_and_segments_for_offsets_of_any_kind(tmp_path):
    """ The arithmetic of csrc/psh_parts.h, which every kernel of the operators takes its rows from, compiled for the CPU (overflows trap). """
    exe = str(tmp_path/'parts_check')
    subprocess.check_call(['g++', '-std=c++17', '-O1', '-ftrapv', '-include', 'algorithm', *linear_plan.NATIVE, os.path.join(ROOT, 'tests', 'native', 'parts_check.cpp'), '-o', exe])
    run = subprocess.run([exe, '6000'], capture_output=True, text=True)
    assert run.returncode == 0 and run.stdout.strip() == 'ok', run.stdout + run.stderr


def _descriptor(lengths, K, N, shift, nonlin):
    """ of a call as tests/test_gpu_operators_tiles.py makes it """
    d = abi.PshLinearDesc()
    ld = (K + 7)//8*8 + 8
    d.dtype, d.nonlin, d.n_groups, d.rows, d.in_dim, d.out_dim = abi.DTYPE_BF16, abi.NL_IDS[nonlin], len(lengths), sum(lengths) + 3, K, N
    d.ld_x = d.ld_w = ld
    d.stride_w, d.ld_dy = N*ld, (N + 7)//8*8
    d.x = d.weight = 4096 + 2*shift
    d.offsets = d.y = d.dy = d.dx = d.dweight = d.dbias = d.workspace = 4096
    return d


def test_the_layer_cases_reach_every_kind_of_tile():
    reached = set()
    for name, (lengths, K, N, shift, nonlin, forward, dx, dw, joint) in layer_cases.CASES.items():
        p = linear_plan.plan(_descriptor(lengths, K, N, shift, nonlin))
        assert (p.forward, p.dx, p.dw, p.joint) == (forward, dx, dw, joint), (name, [linear_plan.KINDS[k] for k in p[:3]], p.joint)
        reached |= linear_plan.kernels(p)
    kinds = range(len(linear_plan.KINDS))
    every = {(k, t) for k in ('forward', 'dx') for t in kinds} | {(k, t) for k in ('dw', 'both') for t in kinds if t != linear_plan.ROWS16}
    assert reached >= every, every - reached


def test_the_rules_are_those_of_the_library():
    """ (as far as the library tells: the size of the scratch memory, which follows from the tiles and pieces) """
    lib = load_library()
    for lengths, K, N, shift, nonlin, *_ in layer_cases.CASES.values():
        d = _descriptor(lengths, K, N, shift, nonlin)
        assert lib.psh_grouped_linear_grad_workspace(ctypes.byref(d)) == linear_plan.plan(d).space


@pytest.mark.parametrize('groups,rows,K,N', [(64, 640, 1024, 1024), (256, 2560, 2048, 2048), (1000, 130, 40, 72), (5000, 20000, 256, 256)])
def test_groups_that_are_not_cut_take_no_scratch_memory(groups, rows, K, N):
    """ Only a group of more rows than a piece has partial sums, of its pieces: there are no more than twice as many of those as
    pieces fit into the rows, and one, however many groups there are. """
    for dtype, wide in ((abi.DTYPE_BF16, 4), (abi.DTYPE_F32, 4), (abi.DTYPE_F64, 8)):
        d = _descriptor([rows//groups]*(groups - 1) + [rows - 3 - rows//groups*(groups - 1)], K, N, 0, None)
        d.dtype = dtype
        piece = linear_plan.plan(d).piece
        assert load_library().psh_grouped_linear_grad_workspace(ctypes.byref(d)) <= (2*rows//piece + 1)*(N*K + N)*wide + 2*256


def test_float64_gradients_of_the_recurrence_stay_on_eight_lanes():
    """ 16 lanes a channel make them slower (64 channels, 16 states, 480 sequences of 256 rows: 392 us on 8, 599 us on 16).  The lanes show
    in the channel blocks, each of which has room for its own sums over its channels. """
    lib = load_library()
    for seqs in (256, 300, 511, 512, 600):
        d = abi.PshScanDesc()
        d.n_policies, d.n_seqs, d.rows, d.channels, d.states, d.dtype = 1, seqs, 256*seqs, 64, 16, abi.DTYPE_F64
        sums = 2*d.rows*2*16*8          # two blocks of 32 channels
        d.dB = d.dC = 4096
        assert sums <= lib.psh_selective_scan_grad_workspace(ctypes.byref(d)) <= sums + 4*seqs + 512


@pytest.mark.parametrize('lengths,K,N', [(c[0], c[1], c[2]) for c in layer_cases.CASES.values()], ids=list(layer_cases.CASES))
@pytest.mark.parametrize('nonlin', [None, 'tanh'])
def test_the_size_of_the_scratch_memory_does_not_depend_on_addresses(lengths, K, N, nonlin):
    """ A caller may ask for it before the arrays are there: pointers are only compared with NULL.  It is enough for a call with any of them. """
    lib = load_library()
    sizes, needed = set(), []
    for shift in range(3):
        for dy in (4096, 4098):
            d = _descriptor(lengths, K, N, shift, nonlin)
            d.dy = dy
            sizes.add(lib.psh_grouped_linear_grad_workspace(ctypes.byref(d)))
            needed.append(linear_plan.plan(d).space)
    assert len(sizes) == 1 and max(needed) <= sizes.pop()
