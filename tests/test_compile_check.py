"""The driver-free gfx950 compile check (CPU only: hipcc cross-compiles).

Counterpart of the reference's AOT compile check (scripts/aot_compile_check.py:81-156).
"""

from __future__ import annotations

import pytest

from triton_flash_attention import _lib, compile_check

REMARKS = """\
fa_fwd.hip:61:1: remark: Function Name: _ZN2fa15fwd_pipe_kernelILi64ELb1ELi4ELi1ENS_3F16EEEvNS_7FwdArgsE [-Rpass-analysis=kernel-resource-usage]
fa_fwd.hip:61:1: remark:     TotalSGPRs: 64 [-Rpass-analysis=kernel-resource-usage]
fa_fwd.hip:61:1: remark:     VGPRs: 168 [-Rpass-analysis=kernel-resource-usage]
fa_fwd.hip:61:1: remark:     AGPRs: 0 [-Rpass-analysis=kernel-resource-usage]
fa_fwd.hip:61:1: remark:     ScratchSize [bytes/lane]: 0 [-Rpass-analysis=kernel-resource-usage]
fa_fwd.hip:61:1: remark:     Occupancy [waves/SIMD]: 3 [-Rpass-analysis=kernel-resource-usage]
fa_fwd.hip:61:1: remark:     LDS Size [bytes/block]: 49152 [-Rpass-analysis=kernel-resource-usage]
fa_bwd.hip:37:1: remark: Function Name: _ZN2fa17preprocess_kernelILi32ENS_3F16EEEvPKDF16_S3_Pfl [-Rpass-analysis=kernel-resource-usage]
fa_bwd.hip:37:1: remark:     VGPRs: 16 [-Rpass-analysis=kernel-resource-usage]
fa_bwd.hip:37:1: remark:     AGPRs: 0 [-Rpass-analysis=kernel-resource-usage]
fa_bwd.hip:37:1: remark:     ScratchSize [bytes/lane]: 12 [-Rpass-analysis=kernel-resource-usage]
fa_bwd.hip:37:1: remark:     Occupancy [waves/SIMD]: 8 [-Rpass-analysis=kernel-resource-usage]
fa_bwd.hip:37:1: remark:     LDS Size [bytes/block]: 0 [-Rpass-analysis=kernel-resource-usage]
"""


def test_resource_report_parsing():
    ks = compile_check.parse_resource_usage(REMARKS)
    # c++filt demangles the first; the second (fp16 pointer arguments) may stay
    # mangled there and is named by the fallback decoder instead.
    assert [k.name.split("(")[0] for k in ks] == ["fa::fwd_pipe_kernel<64, true, 4, 1, fa::F16>",
                                                  "fa::preprocess_kernel<32, fa::F16>"]
    fwd, pre = ks
    assert (fwd.vgprs, fwd.agprs, fwd.scratch, fwd.occupancy, fwd.lds) == (168, 0, 0, 3, 49152)
    assert (pre.vgprs, pre.scratch, pre.occupancy) == (16, 12, 8)
    spills, missing = compile_check.spilling_defaults(ks)
    assert [k.name.split("(")[0] for k in spills] == ["fa::preprocess_kernel<32, fa::F16>"]
    assert "fa::dkdv_pipe_kernel<64, true, 4, fa::BF16>" in missing


def test_resource_report_with_the_place_behind_the_word():
    """As the compiler words it where it keeps the assembly."""
    lines = [f"remark: {place}: {rest}" for place, rest in
             (line.split(": remark: ") for line in REMARKS.splitlines())]
    assert compile_check.parse_resource_usage("\n".join(lines)) == \
        compile_check.parse_resource_usage(REMARKS)


def test_spill_allowance_is_per_kernel_and_capped():
    """A default kernel listed in ALLOWED_SPILLS may spill up to its measured
    bytes per lane and no more; every other default kernel may not spill."""
    name, cap = next(iter(compile_check.ALLOWED_SPILLS.items()))
    assert name in compile_check.DEFAULT_KERNELS
    other = "fa::dq_kernel<128, false, 4, 32, fa::F16>"
    assert other in compile_check.DEFAULT_KERNELS and other not in compile_check.ALLOWED_SPILLS

    def spills(scratch_of):
        ks = [compile_check.KernelUsage(name=f"{n}(fa::BwdArgs)", scratch=scratch_of.get(n, 0))
              for n in compile_check.DEFAULT_KERNELS]
        return [k.name.split("(")[0] for k in compile_check.spilling_defaults(ks)[0]]

    assert spills({name: cap}) == []
    assert spills({name: cap + 4}) == [name]
    assert spills({other: 4}) == [other]


def test_fallback_names_for_undemangled_kernels():
    assert compile_check._short_name("_ZN2fa17preprocess_kernelILi128ENS_4BF16EEEvPKDF16_S3_Pfl") == \
        "fa::preprocess_kernel<128, fa::BF16>(...)"
    assert compile_check._short_name("_ZN2fa14dq_pipe_kernelILi32ELb0ELi4EEEvNS_7BwdArgsE") == \
        "fa::dq_pipe_kernel<32, false, 4>(...)"
    assert compile_check._short_name("_ZN2fa19split_reduce_kernelEPKfPDF16_S2_li") == \
        "fa::split_reduce_kernel(...)"


def test_default_kernel_list_follows_the_tiling_table():
    ok, why = _lib.available()
    assert ok, why
    for (kind, D, causal), variant in compile_check.DEFAULT_VARIANTS.items():
        assert _lib.get_tiling(kind, D, causal)["variant"] == variant, (kind, D, causal)
    assert len(compile_check.DEFAULT_VARIANTS) == 3 * 3 * 2


def test_unsupported_arch_is_rejected():
    with pytest.raises(ValueError, match="unsupported arch"):
        compile_check.compile_library("gfx942")


def test_library_compiles_for_gfx950_without_spills_in_the_defaults(capsys):
    assert compile_check.main(["--strict"]) == 0
    assert "compile check passed for gfx950" in capsys.readouterr().out


ASSEMBLY = """\
	.globl	_ZN2fa5tile_kernelE
_ZN2fa5tile_kernelE:                    ; @_ZN2fa5tile_kernelE
; %bb.0:
	v_readlane_b32 s6, v3, 2
	s_mov_b32 s7, 0x20000
	{first}
	s_cbranch_scc1 .LBB0_2
; %bb.1:
	s_add_u32 s4, s4, 64
.LBB0_2:                                ; =>This Inner Loop Header: Depth=1
	;;#ASMSTART
	s_mov_b32 s9, m0
	s_mov_b32 m0, s8
	{second}
	buffer_load_dwordx4 v1, s[4:7], 0 offen lds
	s_mov_b32 m0, s9
	;;#ASMEND
	s_cbranch_vccnz .LBB0_2
	s_endpgm
.Lfunc_end0:
"""


@pytest.mark.parametrize(("first", "second", "found"), [
    ("", "s_nop 0", []),                       # five states behind the readlane, one behind M0
    ("s_nop 0", "", ["m0"]),
    ("s_nop 7", "", ["m0"]),
    ("", "", ["m0", "readlane"]),
    ("s_cmp_eq_u32 s2, 0", "s_nop 0", []),
    ("s_mov_b32 s6, 0", "", ["m0"]),           # the descriptor's word is a scalar instruction's by then
    ("v_readlane_b32 s4, v3, 1", "s_nop 0", ["readlane"]),  # on the path past the addition
    ("v_add_co_u32 v2, s[4:5], v2, v4", "s_nop 0", ["v_add_co"]),
    ("v_add_co_u32 v2, s[4:5], v2, v4", "s_nop 1", []),
    ("v_add_f32 v2, s4, v4", "s_nop 0", []),
])
def test_missing_wait_states_are_found(first, second, found):
    faults = compile_check.wait_state_faults(ASSEMBLY.format(first=first, second=second))
    assert len(faults) == len(found)
    for word in found:
        assert any(word in f.split("behind")[1] for f in faults), faults


def test_memory_instructions_without_operands_are_read():
    """Cache maintenance between a write of M0 and the load is one wait state; it reads nothing."""
    text = ASSEMBLY.format(first="buffer_inv", second="buffer_wbl2")
    assert compile_check.wait_state_faults(text) == []
