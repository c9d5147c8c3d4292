"""The waits behind matrix instructions in the library's own device code.

A vector or memory instruction that reads or overwrites the result of a
matrix instruction has to come a number of wait states behind it; the hardware
does not look.  The compiler puts them in, but where several exits of a loop
meet it has taken the longer way for the shorter and left some out.  So every
way through the built kernels is followed here.
"""

import collections
import heapq
import os
import re
import struct
import subprocess

import pytest

import chainermn_amd

LIBRARY = os.path.join(os.path.dirname(chainermn_amd.__file__), '_C.so')
OBJDUMP = '/opt/rocm/llvm/bin/llvm-objdump'
# four passes, the only matrix instruction in use; 8 is also the least that
# the compiler leaves within a block
STATES = {'v_mfma_f32_16x16x32_bf16': 8}


def code_objects(library):
    with open(library, 'rb') as f:
        data = f.read()
    magic = b'__CLANG_OFFLOAD_BUNDLE__'
    at = data.find(magic)
    while at >= 0:
        entries, = struct.unpack_from('<Q', data, at + len(magic))
        p = at + len(magic) + 8
        for _ in range(entries):
            offset, size, length = struct.unpack_from('<QQQ', data, p)
            name = data[p + 24:p + 24 + length]
            p += 24 + length
            if name.endswith(b'gfx950'):
                yield data[at + offset:at + offset + size]
        at = data.find(magic, at + 1)


def registers(operand):
    m = re.match(r'[-|]*([va])(?:(\d+)|\[(\d+):(\d+)\])\|?(?:\s|$)', operand)
    if not m:
        return frozenset()
    first = int(m[2] or m[3])
    return frozenset(m[1] + str(i)
                     for i in range(first, int(m[4] or first) + 1))


def kernels(listing):
    """name: (instructions, labels)."""
    found, code, labels = {}, [], {}
    for line in listing.splitlines():
        line = line.split('//')[0].strip()
        m = re.match(r'[0-9a-f]+ <(\w+)>:$', line)
        if m and re.match(r'L\d+$', m[1]):
            labels[m[1]] = len(code)
        elif m:
            code, labels = found[m[1]] = ([], {})
        elif re.match(r'[a-z]\w+', line):
            name, _, rest = line.partition(' ')
            operands = [x.strip() for x in rest.split(',')]
            code.append((name, operands, [registers(x) for x in operands]))
    return found


def too_early(code, labels):
    """(matrix instruction, what comes too early behind it, wait states)."""
    def next_of(i):
        name, operands, _ = code[i]
        if name in ('s_endpgm', 's_setpc_b64'):
            return []
        if name == 's_branch':
            return [labels[operands[0]]]
        if name.startswith('s_cbranch'):
            return [i + 1, labels[operands[0]]]
        return [i + 1] if i + 1 < len(code) else []

    wrong = []
    for i, (name, _, regs) in enumerate(code):
        need = STATES.get(name)
        if need is None:
            assert not name.startswith(('v_mfma', 'v_smfmac')), name
            continue
        result, seen = regs[0], set()
        heap = [(0, j) for j in next_of(i)]
        while heap:
            states, j = heapq.heappop(heap)
            if states >= need or j in seen:
                continue
            seen.add(j)
            other, operands, used = code[j]
            takes = frozenset().union(*used)
            if other in STATES:  # a sum goes on without a wait
                takes = used[1] | used[2]
            if takes & result:
                wrong.append((i, j, states))
            wait = int(operands[0], 0) if other == 's_nop' else 0
            for k in next_of(j):
                heapq.heappush(heap, (states + 1 + wait, k))
    return wrong


def test_the_shortest_way_is_found():
    # the way over L0 is long, the branch before it is not
    listing = '''
0000000000001000 <kernel>:
	v_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], v[0:3] // 0: 0
	s_cbranch_vccnz L1
	s_nop 7
0000000000001020 <L0>:
	v_mov_b32_e32 v9, v3
	s_endpgm
0000000000001030 <L1>:
	v_mov_b64_e32 v[20:21], v[2:3]
	s_branch L0
'''
    code, labels = kernels(listing)['kernel']
    assert labels == {'L0': 3, 'L1': 5}
    assert sorted(too_early(code, labels)) == [(0, 3, 3), (0, 5, 1)]
    fine = listing.replace('v_mov_b64_e32 v[20:21], v[2:3]', 's_nop 5')
    assert not too_early(*kernels(fine)['kernel'])


@pytest.mark.skipif(not os.path.exists(LIBRARY) or not os.path.exists(OBJDUMP),
                    reason='needs the built library and llvm-objdump')
def test_results_of_matrix_instructions_are_waited_for(tmp_path):
    seen = collections.Counter()
    for i, image in enumerate(code_objects(LIBRARY)):
        path = tmp_path / '{}.elf'.format(i)
        path.write_bytes(image)
        listing = subprocess.run(
            [OBJDUMP, '-d', '--symbolize-operands', '--no-show-raw-insn',
             str(path)], check=True, stdout=subprocess.PIPE,
            universal_newlines=True).stdout
        for name, (code, labels) in kernels(listing).items():
            seen['matrix'] += sum(c[0] in STATES for c in code)
            seen['kernels'] += 1
            wrong = too_early(code, labels)
            assert not wrong, '{}: {}'.format(name, [
                (code[i][:2], code[j][:2], n) for i, j, n in wrong])
    assert seen['kernels'] > 100 and seen['matrix'] > 1000
