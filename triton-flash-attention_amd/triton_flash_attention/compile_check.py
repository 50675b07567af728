"""Driver-free compile check of the gfx950 kernel library.

The MI355X counterpart of the reference's ``scripts/aot_compile_check.py``
(which AOT-compiles its forward, preprocess and backward kernels for an NVIDIA
target without a GPU, lines 81-156): this compiles every HIP source of the
library for ``--offload-arch=gfx950`` with the production flags into a
temporary file, no GPU or driver needed, and reads the compiler's per-kernel
resource report (VGPRs, AGPRs, scratch, occupancy, LDS). With ``--strict`` it
also fails when a kernel the default tiling table selects spills registers to
scratch memory: a spill reload inside a pipelined loop is a vector-memory load,
and waiting for it drains the kernel's DMA ring. It also reads the assembly of
every kernel for wait states that the hardware wants and inline assembly leaves
out (wait_state_faults), and fails where one is missing.

    python -m triton_flash_attention.compile_check [--arch gfx950] [--report] [--strict]
"""

from __future__ import annotations

import argparse
import re
import shutil
import subprocess
import sys
import tempfile
from dataclasses import dataclass
from pathlib import Path

from . import _build

SUPPORTED_ARCHS = ("gfx950",)

# Kernel instances the default tiling table (kDefault in csrc/fa_capi.hip) and
# its shape rules select, and the kernels of the operators around the attention
# call, as demangled name prefixes, for D = 32, 64, 128, both
# mask modes and both element types (at D = 128 the forward takes the 4-wave
# pipelined kernel, the 8-wave one where its rounds are whole, the two-key-group
# one for launches of about one work-group per CU, and the classic one for short
# queries; at D = 32 causal launches over few heads take the two-key-group
# forward, and the other causal launches from 512 queries its 16x16x32 form; at
# D <= 64 small launches without the mask the two-key-group forward; the smallest
# launches, and decoding at every head size, the 16x16x32 form with 64-query
# work-groups;
# at D <= 64 a backward
# whose dK/dV launch splits next to a short dQ launch runs the combined dK/dV + dQ
# kernel; dQ takes the pipelined kernel at D = 128 for short causal launches, and
# dQ and dK/dV their 16x16x32 forms at D = 64 and, without the mask, D = 32;
# short-query launches at D = 128 without the mask run the classic 4 x 32 dQ
# and dK/dV).
def _defaults() -> tuple[str, ...]:
    names = []
    for e in ("fa::F16", "fa::BF16"):
        for c in ("false", "true"):
            names += [f"fa::fwd_pipe_kernel<32, {c}, 4, 1, {e}, 1>",
                      f"fa::fwd_pipe_kernel<64, {c}, 4, 1, {e}, 1>",
                      f"fa::fwd_pipe_kernel<128, {c}, 8, 1, {e}, 1>", f"fa::fwd_kernel<128, {c}, 4, 32, {e}>",
                      f"fa::fwd_pipe_kernel<128, {c}, 4, 1, {e}, 1>",
                      f"fa::fwd_pipe_kernel<128, {c}, 8, 1, {e}, 2>",
                      f"fa::fwd_pipe_used96_kernel<{c}, 4, {e}, 1>",
                      f"fa::fwd_pipe_used96_kernel<{c}, 8, {e}, 1>",
                      f"fa::fwd_pipe_used96_kernel<{c}, 8, {e}, 2>",
                      f"fa::dkdv_pipe_used96_kernel<{c}, 4, {e}>",
                      f"fa::dq_pipe_used96_kernel<{c}, 4, {e}, true>",
                      f"fa::dq_pipe_used96_kernel<{c}, 4, {e}, false>",
                      f"fa::dkdv_pipe_kernel<32, {c}, 4, {e}>", f"fa::dkdv_pipe_kernel<64, {c}, 4, {e}>",
                      f"fa::dkdv_pipe_kernel<128, {c}, 4, {e}>", f"fa::dkdv_pipe16_kernel<64, {c}, 4, {e}>",
                      f"fa::dkdv_pipe16_kernel<32, false, 4, {e}>",
                      f"fa::dq_kernel<128, true, 4, 32, {e}>" if c == "true"
                      else f"fa::dq_pipe_kernel<128, false, 4, {e}, false>"]
            # dQ with and without the key-tail test (dq_tail_free)
            for t in ("false", "true"):
                names += [f"fa::dq_pipe_kernel<32, {c}, 4, {e}, {t}>",
                          f"fa::dq_pipe_kernel<64, {c}, 4, {e}, {t}>",
                          f"fa::bwd_pair_kernel<32, {c}, 4, {e}, {t}>",
                          f"fa::bwd_pair_kernel<64, {c}, 4, {e}, {t}>"]
            if c == "false":
                names.append(f"fa::dq_pipe_kernel<128, false, 4, {e}, true>")
                names += [f"fa::dq_pipe16_kernel<{d}, false, 4, {e}, {t}>"
                          for d in (32, 64) for t in ("false", "true")]
            else:
                names += [f"fa::dq_pipe_kernel<128, true, 4, {e}, {t}>" for t in ("false", "true")]
                names += [f"fa::dq_pipe16_kernel<64, true, 4, {e}, {t}>" for t in ("false", "true")]
        names.append(f"fa::fwd_pipe_kernel<32, true, 8, 1, {e}, 2>")
        names += [f"fa::fwd_pipe_kernel<{d}, false, 8, 1, {e}, 2>" for d in (32, 64)]
        names.append(f"fa::fwd_pipe16_kernel<32, true, {e}, 2>")
        names += [f"fa::fwd_pipe16_kernel<{d}, {c}, {e}, 1>"
                  for d in (32, 64, 128) for c in ("false", "true")]
        names += [f"fa::{k}_kernel<{d}, {e}>" for k in ("fwd_decode", "preprocess")
                  for d in (32, 64, 128)]
        names.append(f"fa::split_reduce_kernel<{e}>")
    # The operators around the attention call.
    flags = [f"{n}, {i}" for n in ("false", "true") for i in ("false", "true")]
    for e in ("fa::F16", "fa::BF16"):
        names += [f"fa::{k}_kernel<{lanes}, {e}, {f}>" for k in ("rope", "rope_bwd")
                  for lanes in (2, 4, 8) for f in flags]
        names += [f"fa::paged_fwd_kernel<{d}, {e}, {r}, {s}>" for d in (32, 64, 128)
                  for r in (1, 2) for s in ("false", "true")]
        names += [f"fa::paged_join_kernel<{d}, {e}>" for d in (32, 64, 128)]
        names.append(f"fa::rope_reduce_kernel<{e}>")
        names += [f"fa::prefix_fwd_kernel<{d}, {e}, {w}>" for d in (32, 64, 128)
                  for w in ("false", "true")]
        names += [f"fa::prefix_join_kernel<{d}, {e}, {w}>" for d in (32, 64, 128) for w in (4, 16)]
    names += [f"fa::{k}_kernel" for k in ("fork_small", "fork_children", "fork_finish", "page_copy",
                                          "compact_small", "compact_mark", "compact_count",
                                          "compact_scan", "compact_apply")]
    names += [f"fa::{k}_kernel<{c}>" for k in ("fork_count", "compact_rank") for c in ("false", "true")]
    names += ["fa::paged_plan_kernel<1>", "fa::paged_plan_kernel<2>"]
    names += [f"fa::paged_store_kernel<{w}>" for w in (32, 64, 128, 256)]
    names += [f"fa::{k}_kernel<128, false, 4, 32, {e}>" for k in ("dq", "dkdv")
              for e in ("fa::F16", "fa::BF16")]
    return tuple(names)


DEFAULT_KERNELS = _defaults()
# Default kernels allowed a measured spill (bytes per lane, at most): the
# short-query dK/dV at D = 128 asks for two waves per SIMD (256 registers) and
# reloads two 16-byte values per 32-query unit; with them it is 13-15 % faster
# than the pipelined kernel at one wave per SIMD for 4-64 queries (select_dkdv,
# csrc/fa_capi.hip). The attention over shared prefixes at D = 64 keeps up to
# three values of a work-group's place in scratch while it works on a piece of
# a prefix: they are stored and read outside the loops over keys, and three
# work-groups a CU are worth more. Any other spill, or a larger one, fails
# --strict.
ALLOWED_SPILLS = {f"fa::dkdv_kernel<128, false, 4, 32, {e}>": 52 for e in ("fa::F16", "fa::BF16")}
ALLOWED_SPILLS |= {f"fa::prefix_fwd_kernel<64, {e}, {w}>": 16 for e in ("fa::F16", "fa::BF16")
                   for w in ("false", "true")}
# The same table as (kernel kind, head_dim, causal) -> default variant index,
# for the test that keeps this list in step with kDefault (kinds: 0 fwd,
# 1 dK/dV, 2 dQ).
DEFAULT_VARIANTS = {
    (0, 32, False): 6, (0, 32, True): 6, (0, 64, False): 6, (0, 64, True): 6,
    (0, 128, False): 7, (0, 128, True): 7,
    (1, 32, False): 4, (1, 32, True): 4, (1, 64, False): 4, (1, 64, True): 4,
    (1, 128, False): 4, (1, 128, True): 4,
    (2, 32, False): 4, (2, 32, True): 4, (2, 64, False): 4, (2, 64, True): 4,
    (2, 128, False): 4, (2, 128, True): 1,
}


@dataclass
class KernelUsage:
    name: str
    vgprs: int = -1
    agprs: int = -1
    scratch: int = -1
    occupancy: int = -1
    lds: int = -1


# (with -save-temps the source's place stands behind the word)
_REMARK = r"remark:\s+(?:\S+:\d+:\d+:\s+)?"
_FIELDS = (
    ("vgprs", re.compile(_REMARK + r"VGPRs: (\d+)")),
    ("agprs", re.compile(_REMARK + r"AGPRs: (\d+)")),
    ("scratch", re.compile(_REMARK + r"ScratchSize \[bytes/lane\]: (\d+)")),
    ("occupancy", re.compile(_REMARK + r"Occupancy \[waves/SIMD\]: (\d+)")),
    ("lds", re.compile(_REMARK + r"LDS Size \[bytes/block\]: (\d+)")),
)
_NAME = re.compile(_REMARK + r"Function Name: (\S+)")


_MANGLED = re.compile(r"^_ZN2fa(\d+)")
_TARG = re.compile(r"L([ib])(\d+)E|NS_\d+(F16|BF16)E")


def _short_name(mangled: str) -> str:
    """``fa::name<args>`` of this library's kernels (integer / bool template
    arguments only), for names a demangler leaves as they are."""
    m = _MANGLED.match(mangled)
    if m is None:
        return mangled
    n = int(m.group(1))
    start = m.end()
    name = mangled[start:start + n]
    rest = mangled[start + n:]
    args = []
    if rest.startswith("I"):
        body = rest[1:rest.index("EE") + 1] if "EE" in rest else ""
        for kind, val, elem in _TARG.findall(body):
            if elem:
                args.append("fa::" + elem)
            else:
                args.append(("true" if val == "1" else "false") if kind == "b" else val)
    return f"fa::{name}<{', '.join(args)}>(...)" if args else f"fa::{name}(...)"


def _demangle(names: list[str]) -> list[str]:
    tool = shutil.which("c++filt") or shutil.which("llvm-cxxfilt")
    out_names = names
    if tool is not None and names:
        out = subprocess.run([tool], input="\n".join(names), capture_output=True, text=True)
        lines = out.stdout.splitlines()
        if out.returncode == 0 and len(lines) == len(names):
            out_names = lines
    return [_short_name(n) if n.startswith("_Z") else n for n in out_names]


def parse_resource_usage(text: str) -> list[KernelUsage]:
    """Kernel records from hipcc's ``-Rpass-analysis=kernel-resource-usage`` remarks."""
    kernels: list[KernelUsage] = []
    for line in text.splitlines():
        m = _NAME.search(line)
        if m:
            kernels.append(KernelUsage(m.group(1)))
            continue
        if not kernels:
            continue
        for field, pattern in _FIELDS:
            m = pattern.search(line)
            if m:
                setattr(kernels[-1], field, int(m.group(1)))
                break
    for k, name in zip(kernels, _demangle([k.name for k in kernels])):
        k.name = name.removeprefix("void ")
    return kernels


# ---- wait states ------------------------------------------------------------------------
#
# The compiler keeps instructions apart that the hardware does not, but looks into no block of
# inline assembly. Two such rules of gfx950 meet the blocks that move tiles to LDS:
M0_WAIT = 1    # from a scalar write of M0 to a load that goes to LDS through it
SGPR_WAIT = 5  # from a vector instruction that writes a scalar register to a memory access that reads it

_FUNCTION = re.compile(r"^(\w+):\s*; @")
_LABEL = re.compile(r"^([.\w$]+):")
_SCALARS = re.compile(r"(?<![\w\[:.])(?:s\[(\d+):(\d+)\]|s(\d+)\b|(vcc|m0)\b)")


def _scalars(operands: str) -> frozenset:
    found = set()
    for lo, hi, one, name in _SCALARS.findall(operands):
        found |= {name} if name else {int(one)} if one else set(range(int(lo), int(hi) + 1))
    return frozenset(found)


def _functions(assembly: str):
    """(name, instructions, labels) of each function: ("op", "operands") in order, and the place that
    a label stands for."""
    name = None
    for line in assembly.splitlines():
        line = line.strip()
        m = _FUNCTION.match(line)
        if m:
            name, code, labels = m.group(1), [], {}
            continue
        if name is None:
            continue
        if line.startswith(".Lfunc_end"):
            yield name, code, labels
            name = None
            continue
        line = line.split(";")[0].strip()
        if not line:
            continue
        m = _LABEL.match(line)
        if m:
            labels[m.group(1)] = len(code)
        elif not line.startswith("."):
            op, _, operands = line.partition(" ")
            code.append((op, operands.strip()))


def wait_state_faults(assembly: str) -> list[str]:
    """Instructions of gfx950 assembly that follow what they read too soon (M0_WAIT, SGPR_WAIT), along
    every path to them."""
    faults = []
    for name, code, labels in _functions(assembly):
        before = [[] for _ in range(len(code) + 1)]
        for i, (op, operands) in enumerate(code):
            if op == "s_branch" or op.startswith("s_cbranch"):
                before[labels[operands]].append(i)
            if op not in ("s_branch", "s_endpgm", "s_setpc_b64"):
                before[i + 1].append(i)
        for i, (op, operands) in enumerate(code):
            if not op.startswith(("buffer_", "global_", "scratch_", "flat_")):
                continue
            reads = _scalars(operands)
            if operands.endswith(" lds"):
                reads |= {"m0"}
            todo, seen = [(p, 0, reads) for p in before[i]], set()
            while todo:
                state = todo.pop()
                p, waited, left = state
                if waited >= SGPR_WAIT or not left or state in seen:
                    continue
                seen.add(state)
                by, args = code[p]
                to = args.split(",")
                if by.startswith("v_"):
                    two = "_co_" in by or by.startswith(("v_div_scale", "v_mad_u64", "v_mad_i64"))
                    if _scalars(",".join(to[:2 if two else 1])) & left:
                        faults.append(f"{name}: '{op} {operands}' {waited} wait states behind "
                                      f"'{by} {args}', not {SGPR_WAIT}")
                        continue
                elif by.startswith("s_") and not by.startswith(("s_cmp", "s_bitcmp", "s_wait", "s_nop")):
                    written = _scalars(to[0])
                    if "m0" in written & left and waited < M0_WAIT:
                        faults.append(f"{name}: '{op} {operands}' {waited} wait states behind "
                                      f"'{by} {args}', not {M0_WAIT}")
                    left -= written
                waited += int(args, 0) + 1 if by == "s_nop" else 1
                todo += [(q, waited, left) for q in before[p]]
    return faults


def compile_library(arch: str = "gfx950",
                    faults: list[str] | None = None) -> tuple[list[KernelUsage], str]:
    """Compile the library into a temporary file; returns (kernels, diagnostics). ``faults`` takes
    what wait_state_faults finds in the kernels' assembly."""
    if arch not in SUPPORTED_ARCHS:
        raise ValueError(f"unsupported arch {arch!r}: the kernels are written for {SUPPORTED_ARCHS}")
    with tempfile.TemporaryDirectory() as tmp:
        jobs = _build.object_commands(Path(tmp), extra=(
            "-Rpass-analysis=kernel-resource-usage",
            *(() if faults is None else ("-save-temps=obj",))))
        procs = [subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)
                 for _, cmd in jobs]
        results = [(p.returncode, err) for p in procs for _, err in [p.communicate()]]
        for path in () if faults is None else sorted(Path(tmp).glob(f"*-amdgcn-*{arch}.s")):
            faults += wait_state_faults(path.read_text())
    stderr = "\n".join(err or "" for _, err in results)
    diag = "\n".join(ln for ln in stderr.splitlines()
                     if "packed-fp32-ops" not in ln and "remark:" not in ln)
    if any(rc != 0 for rc, _ in results):
        raise RuntimeError("hipcc failed:\n" + diag[-6000:])
    return parse_resource_usage(stderr), diag


def spilling_defaults(kernels: list[KernelUsage]) -> tuple[list[KernelUsage], list[str]]:
    """(default kernels that use scratch beyond ALLOWED_SPILLS, default kernels
    missing from the report)."""
    spills, missing = [], []
    for prefix in DEFAULT_KERNELS:
        found = [k for k in kernels if k.name.startswith(prefix + "(")]
        if not found:
            missing.append(prefix)
        spills += [k for k in found if k.scratch > ALLOWED_SPILLS.get(prefix, 0)]
    return spills, missing


def main(argv: list[str] | None = None) -> int:
    parser = argparse.ArgumentParser(description="Driver-free gfx950 compile check")
    parser.add_argument("--arch", default="gfx950", help="offload target (only gfx950)")
    parser.add_argument("--report", action="store_true", help="print every kernel's resource usage")
    parser.add_argument("--strict", action="store_true",
                        help="fail if a default-tiling kernel spills to scratch, or a wait state "
                             "is missing")
    args = parser.parse_args(argv)
    faults: list[str] = []
    try:
        kernels, _ = compile_library(args.arch, faults if args.strict else None)
    except (ValueError, RuntimeError) as e:
        print(f"compile check FAILED: {e}", file=sys.stderr)
        return 1
    if args.report:
        print(f"{'kernel':58s} {'VGPR':>5s} {'AGPR':>5s} {'scratch':>7s} {'waves/SIMD':>10s} {'LDS':>7s}")
        for k in kernels:
            print(f"{k.name[:58]:58s} {k.vgprs:5d} {k.agprs:5d} {k.scratch:7d} {k.occupancy:10d} {k.lds:7d}")
    spills, missing = spilling_defaults(kernels)
    if args.strict and (spills or missing or faults):
        for line in faults:
            print(f"missing wait state: {line}", file=sys.stderr)
        for k in spills:
            print(f"default kernel spills {k.scratch} bytes/lane to scratch: {k.name}", file=sys.stderr)
        for name in missing:
            print(f"default kernel not in the compiler report: {name}", file=sys.stderr)
        return 1
    print(f"compile check passed for {args.arch}: {len(kernels)} kernels (forward, preprocess, "
          f"dK/dV, dQ, split reduce; causal/bidirectional; D 32/64/128; MHA/GQA)"
          + ("; no scratch in the default tilings beyond the measured allowance"
             if args.strict else ""))
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
