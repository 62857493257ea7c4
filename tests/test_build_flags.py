"""CPU: the shipped build holds no packed fp32 instruction (csrc/Makefile, NO_PK): every source, compiled as the Makefile compiles it."""
import os
import re
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, 'geotransformer_amd', 'csrc')
HIPCC = shutil.which('hipcc') or '/opt/rocm/bin/hipcc'


def test_no_shipped_kernel_holds_a_packed_fp32_instruction(tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip('hipcc not available')
    sources = sorted(f for f in os.listdir(CSRC) if f.endswith('.hip'))

    def packed(src):
        plan = subprocess.run(['make', '-C', CSRC, '-n', '-W', src, src[:-4] + '.o'], capture_output=True, text=True).stdout
        line = next(ln for ln in plan.splitlines() if f' -c {src} ' in ln).split()
        asm = str(tmp_path / (src[:-4] + '.s'))
        cmd = [HIPCC] + [w for w in line[1:line.index('-c')] if w != '-fPIC'] + ['-S', '--cuda-device-only', src, '-o', asm]
        res = subprocess.run(cmd, capture_output=True, text=True, cwd=CSRC)
        assert res.returncode == 0, res.stderr[-2000:]
        return src, [ln.strip() for ln in open(asm) if re.match(r'\s*v_pk_(add|mul|fma|mov)_(f32|b32)', ln)]

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
        found = {src: ops[:3] for src, ops in pool.map(packed, sources) if ops}
    assert len(sources) >= 11 and not found, found
