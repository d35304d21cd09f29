"""Matrix products written as assembly (sa2_paged.hpp, mfma_in_place) leave their wait states to the source: the compiler neither adds them nor is kept from
moving an accumulator between two such products.  The assembly that it makes is read for it: no other instruction touches such a product's result before it is there."""
import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'simplicial_attention_amd', 'csrc')
WAIT = 18      # wait states behind a product of 16 passes
PASSES = 8     # the least that a product takes before the next instruction's wait states count


def registers(text):
    out = set()
    for first, last, one in re.findall(r'\bv\[(\d+):(\d+)\]|\bv(\d+)\b', text):
        out |= {int(one)} if one else set(range(int(first), int(last) + 1))
    return out


def violations(lines):
    """(products written as assembly, instructions that come too early) of a kernel's lines."""
    written, pending, products, early = False, {}, 0, []

    def pass_states(n):
        for r in list(pending):
            pending[r] -= n
            if pending[r] <= 0:
                del pending[r]

    for line in lines:
        written = ('#ASMSTART' in line or written) and '#ASMEND' not in line
        code = line.split(';')[0].strip()
        if not code or code.startswith('.') or code.endswith(':'):
            continue
        name, _, operands = code.partition(' ')
        if name == 's_nop':
            pass_states(int(operands) + 1)
        elif name.startswith('v_mfma'):
            result, a, b = re.split(r',\s*(?![^\[]*\])', operands)[:3]
            if (registers(a) | registers(b)) & pending.keys():
                early.append(code)
            pass_states(PASSES)
            if written:
                products += 1
                pending.update(dict.fromkeys(registers(result), WAIT))
        else:
            if not name.startswith('s_') and registers(operands) & pending.keys():
                early.append(code)
            pass_states(1)
    return products, early


PRODUCT = '\t;#ASMSTART\n\ts_nop 1\n\tv_mfma_f32_32x32x16_bf16 v[0:15], v[16:19], v[20:23], v[0:15]\n\t;#ASMEND\n'


@pytest.mark.parametrize('behind,early', [
    ('\tv_mov_b32_e32 v40, v3', 1),
    ('\ts_nop 7\n\ts_nop 7\n\tv_mov_b32_e32 v40, v3', 1),
    ('\ts_nop 7\n\ts_nop 7\n\ts_nop 1\n\tv_mov_b32_e32 v40, v3', 0),
    ('\tv_mov_b32_e32 v3, v40', 1),
    ('\tv_mov_b32_e32 v41, v40', 0),
    ('\tv_mfma_f32_32x32x16_bf16 v[50:65], v[12:15], v[20:23], v[50:65]', 1),
    ('\tscratch_store_dword off, v7, off', 1),
])
def test_the_reader_sees_what_it_looks_for(behind, early):
    products, found = violations((PRODUCT + behind).splitlines())
    assert products == 1 and len(found) == early


def test_no_result_is_touched_before_it_is_there(tmp_path):
    flags = subprocess.run(['make', '-n', '-B', 'build/sa2_paged.o'], cwd=CSRC, check=True, capture_output=True, text=True).stdout
    command = next(line for line in flags.splitlines() if 'sa2_paged.hip' in line and '-c' in line.split()).split()
    out = str(tmp_path / 'sa2_paged.s')
    at = command.index('-o')
    command[at:at + 2] = []
    command[command.index('-c')] = '-S'
    subprocess.run(command + ['--cuda-device-only', '-o', out], cwd=CSRC, check=True, capture_output=True)
    with open(out) as f:
        text = f.read()
    kernels = re.findall(r'^(_Z\S*paged_many_kernel\S*):(.*?)\.Lfunc_end', text, re.M | re.S)
    assert len(kernels) == 24                   # two types, four widths, dense, 2-simplicial and packed
    with_products = 0
    for name, body in kernels:
        products, early = violations(body.splitlines())
        with_products += products > 0
        assert not early, (name, early[:3])
        assert not products or 'v_accvgpr' not in body, name
    assert with_products == 12                  # 64 and 128 channels
