"""CPU: what the compiler does not check for inline asm, on the assembly of exactly the commands that build the shipped library (csrc/Makefile):

* no instruction touches a register that an asm read may still be filling (scripts/check_inflight_regs.py: gemm_packed, gse_embed);
* a buffer load issued by asm may read a scalar register that a vector instruction (v_readfirstlane, v_readlane, a compare) wrote only after
  five wait states, along every path of the control flow, branches and loop back edges included;
* no kernel that pins accumulators (its assembly carries the marker of `held`) spills vector registers, and no kernel multiplies by an
  accumulator that stands in the place of a lost copy;
* the asm that writes m0 says so."""
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


# ---- accumulators -----------------------------------------------------------------------------------------------------------------------
def _vectors(token):
    m = re.match(r'([av])\[(\d+):(\d+)\]$', token)
    if m:
        return [m[1] + str(i) for i in range(int(m[2]), int(m[3]) + 1)]
    return [token] if re.match(r'[av]\d+$', token) else []


COPIES = ('v_accvgpr_read', 'v_accvgpr_write', 'v_accvgpr_mov', 'v_mov_b32', 'v_mov_b64', 'scratch_store', 'scratch_load')


def sums_as_factors(lines):
    """The matrix products of a kernel one of whose factors (not the sum that it adds to) may be another product's sum as it stands.  No kernel
    here multiplies a sum before vector instructions worked on it, so such a factor is a register that a copy was lost for: fp32 dQ of heads
    of 128 with pinned accumulators and spills multiplied K by an accumulator in place of one element of Q.  State at a point: the registers and
    spill slots that may hold a sum; copies pass it on."""
    code, labels = _parse(lines)
    code = [(op, [_vectors(x) for x in args], args, int((re.search(r'offset:(\d+)', text) or [0, 0])[1]), text) for op, args, text in code]
    ends = ('s_endpgm', 's_setpc_b64', 's_branch')
    leaders = {0, *labels.values(), *(i + 1 for i, c in enumerate(code) if c[0].startswith('s_cbranch') or c[0] in ends)}
    found, before, todo = set(), {0: frozenset()}, [0]
    while todo:
        at = todo.pop()
        sums, following = set(before[at]), []
        while at < len(code):
            op, vec, args, slot, text = code[at]
            if op.startswith('v_mfma'):
                if any(r in sums for r in vec[1] + vec[2]):
                    found.add((at, text))
                sums.update(vec[0])
            elif op.startswith(COPIES):  # pairs (to, from); a spill slot is its byte offset
                if op.startswith('scratch_store'):
                    pairs = [(slot + 4 * i, r) for i, r in enumerate(vec[1])]
                elif op.startswith('scratch_load'):
                    pairs = [(r, slot + 4 * i) for i, r in enumerate(vec[0])]
                else:
                    pairs = list(zip(vec[0], vec[1] or [None] * len(vec[0])))
                for to, held in [(to, source in sums) for to, source in pairs]:
                    (sums.add if held else sums.discard)(to)
            elif vec and ' lds' not in text and not op.startswith(('s_', 'ds_write', 'buffer_store', 'global_store', 'v_cmp', 'v_read')):
                sums.difference_update(vec[0], *(vec[1:2] if op.startswith(('v_permlane', 'v_swap')) else []))
            if op.startswith('s_cbranch') or op == 's_branch':
                following.append(labels[args[0]])
            if op in ends:
                break
            at += 1
            if at in leaders:
                following.append(at)
                break
        for nxt in following:
            if nxt < len(code) and (nxt not in before or not sums <= before[nxt]):
                before[nxt] = before.get(nxt, frozenset()) | sums
                todo.append(nxt)
    return [text for _, text in sorted(found)]


def test_the_check_finds_a_sum_in_the_place_of_a_factor():
    product, zero = 'v_mfma_f32_32x32x2_f32 a[0:15], v1, {}, a[0:15]', 'v_accvgpr_write_b32 a1, v0'
    assert not sums_as_factors([product.format('v2'), product.format('v2')])
    assert sums_as_factors([product.format('v2'), product.format('a1')])
    assert sums_as_factors([zero, '.L1:', 'v_mfma_f32_32x32x2_f32 a[16:31], v1, a1, 0', product.format('v2'), 's_cbranch_scc1 .L1', 's_endpgm'])
    copied = [product.format('v2'), 'v_accvgpr_read_b32 v9, a3', 'scratch_store_dword off, v9, off offset:8', 'v_mov_b32_e32 v9, 0',
              'scratch_load_dword v8, off, off offset:8']
    assert sums_as_factors(copied + [product.format('v8')]) and not sums_as_factors(copied + ['v_exp_f32_e32 v8, v8', product.format('v8')])


@pytest.mark.parametrize('name', ATTENTION)
def test_no_product_takes_an_accumulator_for_a_factor(assembly, name):
    found = {kernel: bad[:3] for kernel, bad in ((k, sums_as_factors(lines)) for k, lines, _ in kernels_of(assembly[name])) if bad}
    assert not found, found


@pytest.mark.parametrize('name', ATTENTION)
def test_no_kernel_with_pinned_accumulators_spills(assembly, name):
    kernels = kernels_of(assembly[name])
    pinned = {k: scratch for k, lines, scratch in kernels if any('; held' in ln for ln in lines)}
    assert len(pinned) >= 4 and not any(pinned.values()), pinned


def test_asm_that_writes_m0_says_so():
    """A compiler that used m0 itself (indexed registers, messages) would otherwise find it changed."""
    found = 0
    for name in sorted(f for f in os.listdir(CSRC) if f.endswith(('.h', '.hip'))):
        for m in re.finditer(r'asm\s*(?:volatile)?\s*\((.*?)\);', open(os.path.join(CSRC, name)).read(), re.S):
            if re.search(r'\bm0\s*,', m[1]):
                found += 1
                assert '"m0"' in m[1].rsplit(':', 1)[1], (name, m[0])
    assert found >= 2
