"""Wait states that the hardware asks the program for, in the machine code of the built library.  The compiler puts them between the instructions that it
writes; it does not look inside inline assembly, so vector memory instructions written by hand have to bring their own.  Read from the disassembled gfx950
code objects of libgdn_hip.so (CPU: nothing runs).

  a scalar write of M0, then a load into LDS (which takes its place in LDS from M0): one wait state
  a vector instruction that writes a scalar register, then a vector memory instruction that reads it: five, unless a scalar
  instruction (which waits by itself) has written the register in between
  a store of more than 8 bytes, then a vector instruction that writes the stored registers: two"""
import collections
import functools
import os
import re
import struct
import subprocess
import sys

import pytest

OBJDUMP = '/opt/rocm/llvm/bin/llvm-objdump'
BUNDLE = b'__CLANG_OFFLOAD_BUNDLE__'


def _code_objects(data):
    """The gfx950 code objects in the offload bundles of a shared library."""
    at = data.find(BUNDLE)
    while at >= 0:
        (entries,) = struct.unpack_from('<Q', data, at + len(BUNDLE))
        head = at + len(BUNDLE) + 8
        for _ in range(entries):
            offset, size, name = struct.unpack_from('<QQQ', data, head)
            target = data[head + 24:head + 24 + name]
            head += 24 + name
            if b'gfx950' in target and size:
                yield data[at + offset:at + offset + size]
        at = data.find(BUNDLE, at + 1)


def library_code_objects():
    from fla_hip import _lib
    if not os.path.exists(_lib.LIB_PATH) or not os.path.exists(OBJDUMP):
        pytest.skip('not built in this checkout')
    with open(_lib.LIB_PATH, 'rb') as f:
        return list(_code_objects(f.read()))


@functools.lru_cache(maxsize=1)
def _listing():
    """[(function, [instruction])] of the library."""
    functions = []
    for code in library_code_objects():
        text = subprocess.run([OBJDUMP, '-d', '--no-show-raw-insn', '-'], input=code, capture_output=True, check=True).stdout.decode()
        for line in text.splitlines():
            if line.endswith('>:'):
                functions.append((line.split('<')[1][:-2], []))
            elif line.startswith('\t'):
                functions[-1][1].append(sys.intern(line[1:].split(' //')[0].rstrip()))
    return functions


def _before(code, i, states):
    """The instructions that may run less than `states` + 1 wait states before instruction i (an instruction is one, `s_nop n` is n + 1)."""
    while i > 0 and states > 0:
        i -= 1
        if code[i].startswith(('s_branch', 's_endpgm')):
            return
        yield code[i]
        states -= int(code[i].split()[1]) + 1 if code[i].startswith('s_nop') else 1


def _short(test):
    """{function: how many instructions fail `test(code, i)`}, and how many were looked at (`test` says None where there is nothing to look at)."""
    failures, seen = collections.Counter(), 0
    for name, code in _listing():
        for i in range(len(code)):
            ok = test(code, i)
            seen += ok is not None
            if ok is False:
                failures[name] += 1
    return dict(failures), seen


def _into_lds(instruction):
    return '_load_lds' in instruction or instruction.endswith(' lds')


def test_loads_into_lds_wait_for_their_place():
    def test(code, i):
        if _into_lds(code[i]):
            return not any(re.match(r's_\w+ m0\b', before) for before in _before(code, i, 1))
    failures, seen = _short(test)
    assert seen > 1000 and not failures, (seen, failures)


def _registers(text, kind):
    found = set()
    for one, first, last in re.findall(rf'\b{kind}(?:(\d+)\b|\[(\d+):(\d+)\])', text):
        found |= {int(one)} if one else set(range(int(first), int(last) + 1))
    return found


def _scalars_written_by_a_vector_instruction(instruction):
    op, _, operands = instruction.partition(' ')
    operands = operands.split(',')
    if op.startswith(('v_readfirstlane', 'v_readlane', 'v_cmp')):
        return _registers(operands[0], 's')
    if op.startswith(('v_add_co', 'v_addc_co', 'v_sub', 'v_div_scale', 'v_mad_u64', 'v_mad_i64')) and len(operands) > 1:
        return _registers(operands[1], 's')                                    # (a carry)
    return set()


def test_vector_memory_waits_for_the_scalars_it_reads():
    def test(code, i):
        if code[i].startswith(('global_', 'buffer_', 'flat_', 'scratch_')):
            reads = _registers(code[i], 's')
            if not reads:
                return None
            for before in _before(code, i, 5):
                if before.startswith('v_') and _scalars_written_by_a_vector_instruction(before) & reads:
                    return False
                if before.startswith('s_') and ' ' in before:
                    reads = reads - _registers(before.split(' ', 1)[1].split(',')[0], 's')
            return True
    failures, seen = _short(test)
    assert seen > 1000 and not failures, (seen, failures)


def _after(code, i, states):
    """The instructions that may run less than `states` + 1 wait states after instruction i."""
    while i + 1 < len(code) and states > 0:
        i += 1
        if code[i].startswith(('s_branch', 's_endpgm')):
            return
        yield code[i]
        states -= int(code[i].split()[1]) + 1 if code[i].startswith('s_nop') else 1


def test_stored_registers_are_not_written_too_soon():
    def test(code, i):
        store = re.match(r'(global|flat|scratch|buffer)_store_dwordx[34] (.*)', code[i])
        if store:
            data = _registers(store.group(2).split(',')[0 if store.group(1) == 'buffer' else 1], 'v')
            return not any(after.startswith('v_') and ' ' in after and _registers(after.split(' ', 1)[1].split(',')[0], 'v') & data for after in _after(code, i, 2))
    failures, seen = _short(test)
    assert seen > 1000 and not failures, (seen, failures)
