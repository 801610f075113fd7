"""Static checks of the gfx950 GEMM assembly (CPU: hipcc cross-compiles).

The 4-wave GEMM issues its MFMAs as inline asm (accumulators pinned to
AGPRs), for which hipcc inserts no wait states: the kernels must not spill
and must not touch an accumulator before the drain that ends the k-loop.
"""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(not shutil.which(os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')),
                    reason='hipcc not available')
def test_four_wave_gemm_asm_contract():
    proc = subprocess.run([sys.executable,
                           os.path.join(ROOT, 'tools', 'check_asm_mfma.py')],
                          stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                          text=True, timeout=600)
    assert proc.returncode == 0, proc.stdout[-3000:]
    # 9 gemm256_kernel<., 256, 4, .> instantiations (the spilling persistent
    # bias+GELU one is gone, round 6) + 4 gemm256p_kernel
    assert 'checked 13 4-wave kernels: ok' in proc.stdout


def test_checker_flags_violations():
    sys.path.insert(0, os.path.join(ROOT, 'tools'))
    import check_asm_mfma
    name = '_ZN5kiosk12_GLOBAL__N_114gemm256_kernelILi0ELi256ELi4EEEvPKt'
    good = '\n'.join([name + ':', '\tv_mfma_f32_16x16x32_bf16 a[0:3], v[0:3], '
                      'v[4:7], a[0:3]', '\ts_waitcnt vmcnt(0)', '\ts_nop 7',
                      '\tv_accvgpr_read_b32 v8, a0', '.Lfunc_end0:'])
    assert check_asm_mfma.check(good)[1] == []
    bad = good.replace('\ts_waitcnt vmcnt(0)',
                       '\tv_accvgpr_read_b32 v9, a1')
    assert check_asm_mfma.check(bad)[1]
    spill = good.replace('\ts_waitcnt vmcnt(0)',
                         '\tscratch_store_dword off, v1, off')
    assert check_asm_mfma.check(spill)[1]


@pytest.mark.skipif(not shutil.which(os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')),
                    reason='hipcc not available')
def test_asm_matrix_instructions_have_their_wait_states():
    """Every kernel with inline-asm matrix instructions: two wait states
    between the VALU instruction that writes a register and the matrix
    instruction that reads it, on every path."""
    proc = subprocess.run([sys.executable,
                           os.path.join(ROOT, 'tools', 'check_asm_waits.py')],
                          stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                          text=True, timeout=600)
    assert proc.returncode == 0, proc.stdout[-3000:]
    for unit in ('gemm256', 'product256_bf16', 'product256_mx', 'warmstart'):
        assert unit + '.hip: ' in proc.stdout, proc.stdout[-3000:]


MFMA = 'v_mfma_scale_f32_32x32x64_f8f6f4 a[0:15], v[0:3], v[4:7], 0, v8, v9'


@pytest.mark.parametrize('before,wrong', [
    (['v_mov_b32_e32 v8, v20'], True),
    (['v_mov_b32_e32 v20, v8'], False),
    (['v_mov_b32_e32 v8, v20', 'ds_read_b128 v[30:33], v40'], True),
    (['v_mov_b32_e32 v8, v20', 's_nop 0'], True),
    (['v_mov_b32_e32 v8, v20', 's_nop 1'], False),
    (['v_mov_b32_e32 v8, v20', 's_waitcnt lgkmcnt(0)', 's_barrier'], False),
    (['v_pk_mov_b32 v[2:3], v[20:21], v[22:23]'], True),
    (['v_permlane32_swap_b32_e32 v20, v9'], True),
    (['v_accvgpr_write_b32 a3, v20'], False),
    # around a loop: the write stands behind the matrix instruction
    (['.LBB0_1:'], True),
])
def test_wait_state_checker(before, wrong):
    sys.path.insert(0, os.path.join(ROOT, 'tools'))
    import check_asm_waits
    after = ['v_mov_b32_e32 v9, v20', 's_cbranch_scc1 .LBB0_1'] \
        if before == ['.LBB0_1:'] else []
    text = '\n'.join(['_Z1kv:'] + before + [';;#ASMSTART', MFMA, ';;#ASMEND']
                     + after + ['s_endpgm', '.Lfunc_end0:', ''])
    kernels, problems = check_asm_waits.check(text)
    assert kernels == ['_Z1kv']
    assert bool(problems) is wrong, problems
