"""The attention kernels' own assembly, as hipcc writes it for gfx950: what is left of a page's values behind the last token (`cut` in paged_attn.hip) is read before its
registers are written again.  hipcc 7.2 has broken that where a loop's next loads stood under a condition: registers of the values became scratch space of the
softmax.  The loops' last tile is a body of its own since; this looks whether that still helps."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, 'trtllm-llama_amd', 'csrc')
MASK = re.compile(r'v_lshrrev_b32_e64 v\d+, v\d+, -1')  # 0xffffffff >> n: the bytes of a word that stay
KEPT = re.compile(r'v_cndmask_b32_e(?:32|64) v(\d+), v\d+, v(\d+)')


def registers(operand):
    many, one = re.match(r'v\[(\d+):(\d+)\]$', operand), re.match(r'v(\d+)$', operand)
    return set(range(int(many[1]), int(many[2]) + 1)) if many else {int(one[1])} if one else set()


def cuts(lines):
    """-> [(registers that a masked block leaves, those of them that are written before they are read)]; a block ends at a label, and so does the search behind it"""
    found, i = [], 0
    while i < len(lines):
        if MASK.match(lines[i]):
            held = set()
            while i < len(lines) and not lines[i].startswith('.LBB'):
                m = KEPT.match(lines[i])
                held |= {int(m[1])} if m and m[1] == m[2] else set()
                i += 1
            left, lost, j = set(held), set(), i + 1
            while left and j < len(lines) and not lines[j].startswith('.LBB'):
                m = re.match(r'(v_\w+|ds_\w+|global_\w+|buffer_\w+|scratch_\w+|flat_\w+)\s+(.*)', lines[j])
                if m:
                    operands = [o.strip().split(' ')[0] for o in m[2].split(',')]
                    stores = re.match(r'ds_write|(global|buffer|scratch|flat)_store', m[1])
                    for o in operands if stores else operands[1:]:
                        left -= registers(o)
                    written = set() if stores else registers(operands[0])
                    lost |= written & left
                    left -= written
                j += 1
            if held:
                found.append((held, lost))
        i += 1
    return found


def kernels(text):
    for body in re.split(r'\n(?=_ZN4tllm7kernels\S+:)', text)[1:]:
        body = body.split('.section')[0]
        yield body.split(':')[0], [line.split(';')[0].strip() for line in body.split('\n')]


def test_the_search_finds_what_it_looks_for():
    block = ['v_lshrrev_b32_e64 v9, v9, -1', 'v_and_b32_e32 v8, v1, v9', 'v_cndmask_b32_e64 v1, v8, v1, s[2:3]', 'v_cndmask_b32_e32 v2, v8, v2, vcc', '.LBB0_1:']
    assert cuts(block + ['v_add_f32_e32 v3, v1, v2', 'v_mov_b32_e32 v1, v3']) == [({1, 2}, set())]
    assert cuts(block + ['v_sub_f32_e32 v1, v5, v6', 'v_perm_b32 v3, v1, v2, s0']) == [({1, 2}, {1})]
    assert cuts(block + ['v_mfma_f32_16x16x32_f16 a[0:3], v[4:7], v[0:3], a[0:3]', 'v_mov_b32_e32 v2, 0']) == [({1, 2}, set())]
    assert cuts(block + ['ds_write_b64 v7, v[1:2]', 'global_load_dwordx4 v[0:3], v[4:5], off']) == [({1, 2}, set())]
    assert cuts(block + ['global_load_dwordx4 v[0:3], v[4:5], off']) == [({1, 2}, {1, 2})]


def test_values_are_read_before_their_registers_are_written(tmp_path):
    make = open(os.path.join(CSRC, 'Makefile')).read()
    flags = re.search(r'^HIPFLAGS = (.*)$', make, re.M)[1].replace('$(ARCH)', 'gfx950').replace('$(CXXFLAGS)', re.search(r'^CXXFLAGS = (.*)$', make, re.M)[1]).split()
    hipcc = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')
    out = str(tmp_path / 'paged_attn.s')
    subprocess.run([hipcc] + flags + ['-x', 'hip', '--cuda-device-only', '-S', os.path.join(CSRC, 'kernels', 'paged_attn.hip'), '-o', out], check=True, stderr=subprocess.DEVNULL)
    seen = {}
    for name, lines in kernels(open(out).read()):
        for held, lost in cuts(lines):
            seen[name] = seen.get(name, 0) + 1
            assert not lost, f'{name}: v{sorted(lost)} of v{sorted(held)} written before they are read'
    # rows_kernel: 3 head sizes x 2 types x 2 caches with four waves, 2 of the sizes with eight; tile_kernel 12: the loop's body and the last tile of each
    assert sum('rows_kernel' in n for n in seen) == 20 and sum('tile_kernel' in n for n in seen) == 12 and min(seen.values()) >= 2, seen
