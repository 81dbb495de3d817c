"""
CPU tests of the policy operators' kernel sources: what the compiler has to be told about assembly that is written by hand.
"""
import glob
import os
import re
import subprocess

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
    subprocess.check_call(['g++', '-std=c++17', '-O1', '-ftrapv', '-D__host__=', '-D__device__=', '-D__forceinline__=inline', '-include', 'algorithm',
                           '-I', os.path.join(ROOT, 'simurlacra_amd', 'csrc'), os.path.join(ROOT, 'tests', 'native', 'parts_check.cpp'), '-o', exe])
    run = subprocess.run([exe, '6000'], capture_output=True, text=True)
    assert run.returncode == 0 and run.stdout.strip() == 'ok', run.stdout + run.stderr
