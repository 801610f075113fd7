#!/usr/bin/env python3
"""Static check of the wait states before inline-asm matrix instructions.

A matrix instruction that reads a register needs two wait states behind the
VALU instruction that wrote it.  hipcc keeps them for its builtins and puts
none before inline asm, so the scheduler may leave a VALU write right before
an asm matrix instruction.  This script compiles every unit that issues its
matrix instructions as inline asm to gfx950 assembly and follows all paths
that lead to one of them back over two wait states.

    python tools/check_asm_waits.py
"""
import concurrent.futures
import os
import re
import subprocess
import sys
import tempfile

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')
KERNELS = os.path.join(ROOT, 'csrc', 'kernels')
NEEDED = 2
REGISTER = re.compile(r'\b([av])(?:(\d+)\b|\[(\d+):(\d+)\])')
# both operands are written
BOTH = ('v_swap_', 'v_permlane16_swap', 'v_permlane32_swap')


def units():
    """Sources with inline-asm matrix instructions."""
    found = []
    for name in sorted(os.listdir(KERNELS)):
        path = os.path.join(KERNELS, name)
        if name.endswith('.hip') and re.search(
                r'asm volatile\("v_mfma', open(path).read()):
            found.append(path)
    return found


def registers(operand):
    out = set()
    for kind, one, lo, hi in REGISTER.findall(operand):
        lo, hi = (one, one) if one else (lo, hi)
        out.update((kind, i) for i in range(int(lo), int(hi) + 1))
    return out


def operands(inst):
    parts = inst.split(None, 1)
    return [] if len(parts) < 2 else parts[1].split(',')


def writes(inst):
    """Registers a VALU instruction writes (a matrix instruction's results
    have rules of their own)."""
    if not inst.startswith('v_') or inst.startswith('v_mfma'):
        return set()
    ops = operands(inst)
    out = registers(ops[0]) if ops else set()
    if inst.startswith(BOTH):
        out |= registers(ops[1])
    return out


def states(inst):
    if inst.startswith('s_nop'):
        return int(inst.split()[1], 0) + 1
    return 1


def parse(lines):
    """``(instructions, asm flags, labels before each, branch targets)``."""
    insts, asm, labels, inside, pending = [], [], {}, False, []
    for line in lines:
        text = line.strip()
        if text.startswith(';;#ASMSTART') or text.startswith(';#ASMSTART'):
            inside = True
            continue
        if text.startswith(';;#ASMEND') or text.startswith(';#ASMEND'):
            inside = False
            continue
        text = text.split(';')[0].strip()
        if not text:
            continue
        label = re.match(r'^([\w.$]+):', text)
        if label:
            pending.append(label.group(1))
            continue
        if text.startswith('.'):
            continue
        for name in pending:
            labels[name] = len(insts)
        pending = []
        insts.append(text)
        asm.append(inside)
    return insts, asm, labels


def check_function(name, lines):
    """``(asm matrix instructions, problems)``."""
    insts, asm, labels = parse(lines)
    into = {}
    for i, inst in enumerate(insts):
        if inst.startswith(('s_branch', 's_cbranch')):
            target = labels.get(inst.split()[-1])
            if target is not None:
                into.setdefault(target, []).append(i)

    def before(i):
        out = list(into.get(i, ()))
        if i > 0 and not insts[i - 1].startswith(('s_branch', 's_endpgm',
                                                  's_setpc')):
            out.append(i - 1)
        return out

    count, problems = 0, []
    for i, inst in enumerate(insts):
        if not (asm[i] and inst.startswith('v_mfma')):
            continue
        count += 1
        need = set().union(*(registers(o) for o in operands(inst)[1:]))
        todo = [(p, 0) for p in before(i)]
        while todo:
            at, seen = todo.pop()
            hit = writes(insts[at]) & need
            if hit:
                problems.append('%s: %d wait states between "%s" and "%s"' % (
                    name, seen, insts[at], inst))
                break
            seen += states(insts[at])
            if seen < NEEDED:
                todo += [(p, seen) for p in before(at)]
    return count, problems


def check(asm_text):
    """``(kernels with asm matrix instructions, problems)``."""
    kernels, problems = [], []
    for match in re.finditer(r'^(_Z\S+):[^\n]*\n(.*?)^\.Lfunc_end', asm_text,
                             re.M | re.S):
        count, found = check_function(match.group(1),
                                      match.group(2).split('\n'))
        if count:
            kernels.append(match.group(1))
        problems += found
    return kernels, problems


def assembly(source):
    sys.path.insert(0, os.path.join(ROOT, 'tools'))
    import build_native
    with tempfile.TemporaryDirectory() as tmp:
        out = os.path.join(tmp, 'unit.s')
        subprocess.check_call(
            [HIPCC] + build_native.device_flags() +
            ['--cuda-device-only', '-S', source, '-o', out],
            stderr=subprocess.DEVNULL)
        return open(out).read()


def main():
    sources = units()
    with concurrent.futures.ThreadPoolExecutor(max_workers=4) as pool:
        texts = list(pool.map(assembly, sources))
    bad = 0
    for source, text in zip(sources, texts):
        kernels, problems = check(text)
        for p in problems:
            print('FAIL', p)
        if not kernels:
            problems = ['no asm matrix instruction found']
        print('%s: %d kernels: %s' % (
            os.path.basename(source), len(kernels),
            'ok' if not problems else '%d problem(s)' % len(problems)))
        bad += len(problems)
    return 1 if bad else 0


if __name__ == '__main__':
    sys.exit(main())
