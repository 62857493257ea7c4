"""CPU: what the compiler does not check for inline asm, on the assembly of exactly the commands that build the shipped library (csrc/Makefile):

* no instruction touches a register that an asm read may still be filling (scripts/check_inflight_regs.py: gemm_packed, gse_embed);
* a buffer load issued by asm may read a scalar register that a vector instruction (v_readfirstlane, v_readlane, a compare) wrote only after
  five wait states, along every path of the control flow, branches and loop back edges included."""
import os
import re
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, 'geotransformer_amd', 'csrc')
HIPCC = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')
ATTENTION = ('diff_attention_f32', 'diff_attention_bf16', 'diff_attention_f16')
NEEDED = 5  # wait states between a vector instruction's write of a scalar register and a buffer load that reads it


def shipped_command(name):
    """The words of the line with which make compiles name.hip, without -fPIC and the output."""
    plan = subprocess.run(['make', '-C', CSRC, '-n', '-W', name + '.hip', name + '.o'], capture_output=True, text=True).stdout
    words = next(ln for ln in plan.splitlines() if f' -c {name}.hip ' in ln).split()
    return [w for w in words[:words.index('-c')] if w != '-fPIC']


@pytest.fixture(scope='module')
def assembly(tmp_path_factory):
    """name -> the text of the assembly of name.hip as it is shipped."""
    if not os.path.exists(HIPCC):
        pytest.skip('hipcc not available')
    folder = tmp_path_factory.mktemp('shipped')

    def one(name):
        out = str(folder / (name + '.s'))
        res = subprocess.run(shipped_command(name) + ['-S', '--cuda-device-only', name + '.hip', '-o', out], capture_output=True, text=True, cwd=CSRC)
        assert res.returncode == 0, res.stderr[-2000:]
        return name, out

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
        return dict(pool.map(one, ATTENTION + ('transformer', 'gemm')))


def kernels_of(path):
    """(name, lines, the numbers that follow the code) of every kernel of an assembly file."""
    text = open(path).read()
    found = []
    for m in re.finditer(r'^(_Z\w+):.*?^\.Lfunc_end\d+:.*?; ScratchSize: (\d+)', text, re.S | re.M):
        found.append((m[1], m[0][:m[0].index('.Lfunc_end')].splitlines(), int(m[2])))
    return found


def test_the_checked_commands_are_the_shipped_ones():
    for name in ATTENTION + ('transformer', 'gemm'):
        words = shipped_command(name)
        assert '-packed-fp32-ops' in words and '-fno-slp-vectorize' in words and '--offload-arch=gfx950' in words, words


@pytest.mark.parametrize('source,prefix,min_kernels', [('transformer', '_ZN5geotr23gse_embed_bf16x3_kernel', 32),
                                                       ('gemm', '_ZN5geotr18gemm_packed_kernel', 12)])
def test_no_instruction_of_the_shipped_build_touches_a_register_in_flight(assembly, source, prefix, min_kernels):
    chk = subprocess.run([sys.executable, os.path.join(ROOT, 'scripts', 'check_inflight_regs.py'), assembly[source], prefix],
                         capture_output=True, text=True)
    lines = [ln for ln in chk.stdout.splitlines() if ln.startswith(prefix)]
    assert chk.returncode == 0, chk.stdout[-3000:]
    assert len(lines) >= min_kernels and all(int(ln.split(': ')[1].split()[0]) > 0 for ln in lines), chk.stdout[-2000:]


def _parse(lines):
    """([(opcode, operands, text)], label -> index) of the lines of a kernel."""
    code, labels = [], {}
    for line in lines:
        text = line.split(';')[0].strip()
        if text.endswith(':'):
            labels[text[:-1]] = len(code)
        elif text and text[0] not in '.#':
            op = text.split()[0]
            code.append((op, [x.strip().split()[0] for x in text[len(op):].split(',') if x.strip()], text))
    return code, labels


# ---- wait states ------------------------------------------------------------------------------------------------------------------------
def _scalars(token):
    m = re.match(r's\[(\d+):(\d+)\]$', token)
    if m:
        return range(int(m[1]), int(m[2]) + 1)
    m = re.match(r's(\d+)$', token)
    if m:
        return [int(m[1])]
    return [106, 107] if token == 'vcc' else []


def too_early(lines):
    """The loads of a kernel that some path reaches too soon after a vector instruction wrote a scalar register that they read.  State at a
    point: scalar register -> wait states since (the fewest over the paths); blocks are walked until nothing changes."""
    code, labels = _parse(lines)
    found, seen, todo = set(), {}, [(0, ())]
    while todo:
        at, state = todo.pop()
        state = dict(state)
        while at < len(code):
            if at in seen:  # join: the fewest wait states; on where that says something new
                old = seen[at]
                if all(r in old and old[r] <= age for r, age in state.items()):
                    break
                state = {r: min(old.get(r, NEEDED), state.get(r, NEEDED)) for r in {**old, **state}}
            seen[at] = dict(state)
            op, args, text = code[at]
            if op.startswith(('buffer_', 'global_', 'scratch_', 'flat_')):
                if any(r in state for x in args for r in _scalars(x)):
                    found.add(text)
            states = int(args[0], 0) + 1 if op == 's_nop' else 1
            state = {r: age + states for r, age in state.items() if age + states < NEEDED}
            if op.startswith(('v_readlane', 'v_readfirstlane', 'v_cmp')) and args:
                state.update((r, 0) for r in _scalars(args[0]))
            elif op.startswith('s_') and args and not op.startswith(('s_cbranch', 's_branch', 's_nop', 's_waitcnt', 's_cmp')):
                for r in _scalars(args[0]):  # a scalar instruction's result has no such wait
                    state.pop(r, None)
            if op in ('s_endpgm', 's_setpc_b64'):
                break
            if op == 's_branch':
                at = labels[args[0]]
                continue
            if op.startswith('s_cbranch'):
                todo.append((labels[args[0]], tuple(state.items())))
            at += 1
    return sorted(found)


def test_the_check_follows_branches_and_back_edges():
    load, write = 'buffer_load_dwordx4 v2, s[8:11], 0 offen lds', 'v_readfirstlane_b32 s8, v1'
    assert too_early([write, 's_mov_b32 m0, s3', 's_nop 0', load]) and not too_early([write, 's_mov_b32 m0, s3', 's_nop 3', load])
    loop = ['.L1:', load, 's_nop 7', write, 's_cbranch_scc1 .L1', 's_endpgm']  # early over the back edge alone
    assert too_early(loop) and not too_early(loop[:4] + ['s_nop 4'] + loop[4:])
    jump = [write, 's_cbranch_scc1 .L2', 's_nop 7', '.L2:', load]              # early over the jump alone
    assert too_early(jump) and not too_early([write, 's_nop 3', 's_cbranch_scc1 .L2', 's_nop 7', '.L2:', load])
    assert not too_early([write, 's_mov_b32 s8, s20', load])                   # the register was written anew
    assert too_early(['v_readlane_b32 s10, v9, 3', 's_nop 0', load])           # a spilled scalar that comes back


@pytest.mark.parametrize('name', ATTENTION)
def test_tile_loads_wait_for_their_descriptors_on_every_path(assembly, name):
    kernels = kernels_of(assembly[name])
    assert len(kernels) >= 20 and sum('offen lds' in ln for _, lines, _ in kernels for ln in lines) > 100
    found = {kernel: early[:3] for kernel, early in ((k, too_early(lines)) for k, lines, _ in kernels) if early}
    assert not found, found
