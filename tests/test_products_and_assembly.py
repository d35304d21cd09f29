"""The compiler puts the wait states between a matrix product and an instruction that reads its result, but does not look into assembly statements.  The assembly
that it makes of the paged attention is read for it, along every path: no statement touches the result of a product that the compiler issued before it is there."""
import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'simplicial_attention_amd', 'csrc')
WAIT = 18      # (a product of 32 x 32 x 16 takes 8 passes: the compiler itself leaves 12 wait states behind it)
PASSES = 8


def registers(text):
    out = set()
    for bank, first, last, bank1, one in re.findall(r'\b([va])\[(\d+):(\d+)\]|\b([va])(\d+)\b', text):
        out |= {(bank1, int(one))} if one else {(bank, r) for r in range(int(first), int(last) + 1)}
    return out


def blocks_of(lines):
    """Basic blocks: label -> (instructions (name, operands, in a statement), labels that follow)."""
    blocks, label, code, written, order = {}, '', [], False, ['']
    after = {}

    def close(next_label, falls):
        blocks[label] = code
        after.setdefault(label, set()).update({next_label} if falls else ())

    for line in lines:
        written = ('#ASMSTART' in line or written) and '#ASMEND' not in line
        text = line.split(';')[0].strip()
        found = re.match(r'(\.?\w+):$', text)
        if found:
            close(found.group(1), True)
            label, code = found.group(1), []
            continue
        if not text or text.startswith('.'):
            continue
        name, _, operands = text.partition(' ')
        code.append((name, operands, written))
        if name.startswith('s_cbranch') or name == 's_branch' or name == 's_endpgm':
            following = f'{label}+{len(order)}'
            order.append(following)
            close(following, name.startswith('s_cbranch'))
            if name != 's_endpgm':
                after[label].add(operands.strip())
            label, code = following, []
    close(None, False)
    return blocks, after


def walk(code, pending, early):
    pending = dict(pending)
    for name, operands, written in code:
        states = int(operands) + 1 if name == 's_nop' else PASSES if name.startswith('v_mfma') else 1
        touched = set() if name.startswith('s_') else registers(operands)
        if written and touched & pending.keys():
            early.add(f'{name} {operands}')
        if not written:
            for r in touched:          # (the compiler has waited for it)
                pending.pop(r, None)
        pending = {r: left - states for r, left in pending.items() if left > states}
        if name.startswith('v_mfma') and not written:
            pending.update(dict.fromkeys(registers(operands.split(',')[0]), WAIT))
    return pending


def violations(lines):
    """Instructions of assembly statements that come too early behind a product of the compiler's."""
    blocks, after = blocks_of(lines)
    entry, early, todo = {label: {} for label in blocks}, set(), list(blocks)
    while todo:
        label = todo.pop()
        out = walk(blocks[label], entry[label], early)
        for follower in after.get(label, ()):
            if follower not in entry:
                continue
            merged = {r: max(out.get(r, 0), entry[follower].get(r, 0)) for r in out.keys() | entry[follower].keys()}
            if merged != entry[follower]:
                entry[follower] = merged
                todo.append(follower)
    return early


PRODUCT = '\tv_mfma_f32_32x32x16_bf16 v[0:15], v[16:19], v[20:23], 0\n'
SELECT = '\t;#ASMSTART\n\tv_cndmask_b32 v3, v40, v3, s[4:5]\n\t;#ASMEND\n'


@pytest.mark.parametrize('text,early', [
    (PRODUCT + SELECT, 1),
    (PRODUCT + '\ts_add_i32 s0, s0, 1\n' * 12 + SELECT, 1),
    (PRODUCT + '\ts_nop 15\n\ts_nop 1\n' + SELECT, 0),
    (PRODUCT + '\ts_nop 11\n\tv_max_f32_e32 v3, v3, v3\n' + SELECT, 0),           # (the compiler has read it)
    (PRODUCT + '\ts_nop 11\n\tv_max_f32_e32 v4, v4, v4\n' + SELECT, 1),           # (another register of it)
    (PRODUCT + '\ts_cbranch_vccz .LBB0_2\n\ts_nop 15\n\ts_nop 1\n.LBB0_2:\n' + SELECT, 1),
    ('.LBB0_1:\n' + SELECT + '\ts_nop 15\n' + PRODUCT + '\ts_cbranch_scc1 .LBB0_1\n\ts_endpgm\n', 1),
    (PRODUCT + '\ts_branch .LBB0_3\n' + SELECT + '.LBB0_3:\n\ts_endpgm\n', 0),
    (SELECT + PRODUCT, 0),
])
def test_the_reader_sees_what_it_looks_for(text, early):
    assert len(violations(text.splitlines())) == early


def test_no_statement_reads_a_product_before_it_is_there(tmp_path):
    flags = subprocess.run(['make', '-n', '-B', 'build/sa2_paged.o'], cwd=CSRC, check=True, capture_output=True, text=True).stdout
    command = next(line for line in flags.splitlines() if 'sa2_paged.hip' in line and '-c' in line.split()).split()
    out = str(tmp_path / 'sa2_paged.s')
    at = command.index('-o')
    command[at:at + 2] = []
    command[command.index('-c')] = '-S'
    subprocess.run(command + ['--cuda-device-only', '-o', out], cwd=CSRC, check=True, capture_output=True)
    with open(out) as f:
        text = f.read()
    kernels = re.findall(r'^(_Z\S*paged_(?:many|few)_kernel\S*):(.*?)\.Lfunc_end', text, re.M | re.S)
    assert len(kernels) == 48                   # two types and four widths: dense, 2-simplicial and packed; dense of one and of more tokens, 2-simplicial
    for name, body in kernels:
        assert 'v_mfma' in body, name
        early = violations(body.splitlines())
        assert not early, (name, sorted(early)[:3])
