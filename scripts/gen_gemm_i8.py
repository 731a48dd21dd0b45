#!/usr/bin/env python3
"""Generator of the hand-placed K loops of the 8-bit integer products (ecad_amd/csrc/gemm_int8_asm.h): C[256 x BN] += A[256 x K] W[BN x K]^T per workgroup.

The loops of gen_gemm4.py with another matrix instruction: v_mfma_i32_16x16x64_i8 takes 16 bytes per lane and operand as v_mfma_f32_16x16x32_bf16 does, so a stage of 128
bytes of K per row, its two half-steps, the ring, the fragment sets and the schedule are the 16-bit ones, for twice the multiplications.  What these loops add:
  * rows that do not exist (edge tiles) read the last one: %[ra], %[rw] = index of the last row of A / W in the tile;
  * any number of stages from `period` up: %[trips] = stages / period - 1 trips, then one of `period` tails of period + %[rem] stages, rem = stages % period.
K behind the last whole stage is the caller's (gemm_int8.h adds it to the accumulators with matrix instructions of its own).

BN 256: waves as 2 x 2 of 128 x 128, ring of two; BN 144: waves as 4 x 1 of 64 x 144, ring of three; BN 288: 2 x 2 of 128 x 144, ring of two, the ninth column of
accumulators in 32 registers of the caller.  hipcc's own schedule of the same 256 x 256 loop (accumulators moved between register files around half of the matrix
instructions) reached 1940 TOP/s at 8192 x 8192 x 4096.
"""
from __future__ import annotations

import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent))
from gen_gemm4 import ABLATE, ROOT, Gen, clobbers, v  # noqa: E402


class GenI8(Gen):
    def __init__(self, bn):
        super().__init__("f16", bn)
        self.mfma = "v_mfma_i32_16x16x64_i8"

    def clamp_row(self, which, reg):
        self.I(f"v_min_u32_e32 {v(reg)}, %[r{which}], {v(reg)}")

    def last_trip(self, emit, vm):
        for rem in range(1, self.period):
            self.I(f"s_cmp_eq_u32 %[rem], {rem}")
            self.I(f"s_cbranch_scc1 {self.lbl(f'LAST{rem}')}")
        for rem in range(self.period):
            if rem:
                self.L(f"LAST{rem}")
            stages = self.period + rem
            for k in range(stages):
                left = stages - 1 - k
                fetch = left >= self.NS - 1
                emit(k, fetch, vm if fetch else 0, left == 0)
            if rem + 1 < self.period:
                self.I(f"s_branch {self.lbl('DONE')}")
        self.L("DONE")


OPERANDS = """\
      : {out}
      : [ap] "s"(ap), [wp] "s"(wp), [rsa] "s"(rsa), [rsw] "s"(rsw), [ra] "s"(ra), [rw] "s"(rw), [trips] "s"(trips), [rem] "s"(rem), [lds] "s"(lds), [wave] "s"(wave), [zero] "s"(zero)
"""
C8 = ", ".join(f'[c8_{i}] "+v"(c8[{i}])' for i in range(8))


def main():
    out = ROOT / "ecad_amd" / "csrc" / "gemm_int8_asm.h"
    parts = ["// gemm_int8_asm.h -- GENERATED by scripts/gen_gemm_i8.py (rationale there, register map and schedule in gen_gemm4.py); do not edit.\n#pragma once\n"]
    for bn in (256, 144, 288):
        g = GenI8(bn)
        lines = g.build()
        print(f"i8 BN {bn}: {len(lines)} lines, {sum('v_mfma' in x for x in lines)} MFMAs, {g.NV} VGPRs, stages per trip {g.period}, barrier at {g.barrier_at}, DMA stride {g.dma_stride}", file=sys.stderr)
        body = "\n".join('    "' + ln + '\\n"' for ln in lines)
        operands = OPERANDS.format(out=C8 if bn == 288 else "/* accumulators stay in AGPRs */")
        parts.append(f"#define GEMM_I8_PERIOD_{bn} {g.period}  // stages per trip, and the fewest the loop takes\n"
                     f"#define GEMM_I8_ASM_{bn}(ap, wp, rsa, rsw, ra, rw, trips, rem, lds, wave, zero{', c8' if bn == 288 else ''}) \\\n  asm volatile( \\\n" + "\n".join(x + " \\" for x in body.split("\n")) + "\n"
                     + "\n".join(x + " \\" for x in operands.rstrip("\n").split("\n")) + "\n      : " + clobbers(g.NV, 76 if g.narrow else 70) + ")\n")
    text = "\n".join(parts)
    if "--check" in sys.argv:  # the committed header is what this generator writes (tests/test_cpu_operators.py)
        if ABLATE or out.read_text() != text:
            print(f"{out} differs from the generator's output", file=sys.stderr)
            sys.exit(1)
        return
    out.write_text(text)


if __name__ == "__main__":
    main()
