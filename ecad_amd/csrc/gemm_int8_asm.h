// gemm_int8_asm.h -- GENERATED by scripts/gen_gemm_i8.py (rationale there, register map and schedule in gen_gemm4.py); do not edit.
#pragma once

#define GEMM_I8_PERIOD_256 2  // stages per trip, and the fewest the loop takes
#define GEMM_I8_ASM_256(ap, wp, rsa, rsw, ra, rw, trips, rem, lds, wave, zero) \
  asm volatile( \
    "	s_mov_b32 s66, m0\n" \
    "	v_mbcnt_lo_u32_b32 v152, -1, 0\n" \
    "	v_mbcnt_hi_u32_b32 v152, -1, v152\n" \
    "	v_and_b32_e32 v153, 15, v152\n" \
    "	v_lshrrev_b32_e32 v154, 4, v152\n" \
    "	v_bfe_u32 v155, v152, 1, 3\n" \
    "	s_and_b32 s67, %[wave], 1\n" \
    "	s_lshr_b32 s68, %[wave], 1\n" \
    "	s_lshl_b32 s67, s67, 14\n" \
    "	s_mul_i32 s68, s68, 16384\n" \
    "	v_lshlrev_b32_e32 v156, 7, v153\n" \
    "	v_add_u32_e32 v156, %[lds], v156\n" \
    "	v_add_u32_e32 v157, 0, v154\n" \
    "	v_xor_b32_e32 v157, v157, v155\n" \
    "	v_lshl_add_u32 v157, v157, 4, v156\n" \
    "	v_add_u32_e32 v128, s67, v157\n" \
    "	v_add_u32_e32 v132, s68, v157\n" \
    "	v_add_u32_e32 v132, 32768, v132\n" \
    "	v_add_u32_e32 v157, 4, v154\n" \
    "	v_xor_b32_e32 v157, v157, v155\n" \
    "	v_lshl_add_u32 v157, v157, 4, v156\n" \
    "	v_add_u32_e32 v129, s67, v157\n" \
    "	v_add_u32_e32 v133, s68, v157\n" \
    "	v_add_u32_e32 v133, 32768, v133\n" \
    "	v_add_u32_e32 v157, 0, v154\n" \
    "	v_xor_b32_e32 v157, v157, v155\n" \
    "	v_lshl_add_u32 v157, v157, 4, v156\n" \
    "	v_add_u32_e32 v130, s67, v157\n" \
    "	v_add_u32_e32 v134, s68, v157\n" \
    "	v_add_u32_e32 v130, 65536, v130\n" \
    "	v_add_u32_e32 v134, 98304, v134\n" \
    "	v_add_u32_e32 v157, 4, v154\n" \
    "	v_xor_b32_e32 v157, v157, v155\n" \
    "	v_lshl_add_u32 v157, v157, 4, v156\n" \
    "	v_add_u32_e32 v131, s67, v157\n" \
    "	v_add_u32_e32 v135, s68, v157\n" \
    "	v_add_u32_e32 v131, 65536, v131\n" \
    "	v_add_u32_e32 v135, 98304, v135\n" \
    "	v_lshrrev_b32_e32 v156, 3, v152\n" \
    "	v_and_b32_e32 v157, 7, v152\n" \
    "	s_mul_i32 s67, %[wave], 64\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 0\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v158, s68, v154\n" \
    "	v_xor_b32_e32 v158, v158, v157\n" \
    "	v_lshlrev_b32_e32 v158, 4, v158\n" \
    "	v_add_u32_e32 v159, 0, v156\n" \
    "	v_add_u32_e32 v159, s67, v159\n" \
    "	v_min_u32_e32 v159, %[ra], v159\n" \
    "	v_mad_u32_u24 v136, v159, %[rsa], v158\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 4\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v158, s68, v154\n" \
    "	v_xor_b32_e32 v158, v158, v157\n" \
    "	v_lshlrev_b32_e32 v158, 4, v158\n" \
    "	v_add_u32_e32 v159, 8, v156\n" \
    "	v_add_u32_e32 v159, s67, v159\n" \
    "	v_min_u32_e32 v159, %[ra], v159\n" \
    "	v_mad_u32_u24 v137, v159, %[rsa], v158\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 8\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v158, s68, v154\n" \
    "	v_xor_b32_e32 v158, v158, v157\n" \
    "	v_lshlrev_b32_e32 v158, 4, v158\n" \
    "	v_add_u32_e32 v159, 16, v156\n" \
    "	v_add_u32_e32 v159, s67, v159\n" \
    "	v_min_u32_e32 v159, %[ra], v159\n" \
    "	v_mad_u32_u24 v138, v159, %[rsa], v158\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 12\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v158, s68, v154\n" \
    "	v_xor_b32_e32 v158, v158, v157\n" \
    "	v_lshlrev_b32_e32 v158, 4, v158\n" \
    "	v_add_u32_e32 v159, 24, v156\n" \
    "	v_add_u32_e32 v159, s67, v159\n" \
    "	v_min_u32_e32 v159, %[ra], v159\n" \
    "	v_mad_u32_u24 v139, v159, %[rsa], v158\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 16\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v158, s68, v154\n" \
    "	v_xor_b32_e32 v158, v158, v157\n" \
    "	v_lshlrev_b32_e32 v158, 4, v158\n" \
    "	v_add_u32_e32 v159, 32, v156\n" \
    "	v_add_u32_e32 v159, s67, v159\n" \
    "	v_min_u32_e32 v159, %[ra], v159\n" \
    "	v_mad_u32_u24 v140, v159, %[rsa], v158\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 20\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v158, s68, v154\n" \
    "	v_xor_b32_e32 v158, v158, v157\n" \
    "	v_lshlrev_b32_e32 v158, 4, v158\n" \
    "	v_add_u32_e32 v159, 40, v156\n" \
    "	v_add_u32_e32 v159, s67, v159\n" \
    "	v_min_u32_e32 v159, %[ra], v159\n" \
    "	v_mad_u32_u24 v141, v159, %[rsa], v158\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 24\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v158, s68, v154\n" \
    "	v_xor_b32_e32 v158, v158, v157\n" \
    "	v_lshlrev_b32_e32 v158, 4, v158\n" \
    "	v_add_u32_e32 v159, 48, v156\n" \
    "	v_add_u32_e32 v159, s67, v159\n" \
    "	v_min_u32_e32 v159, %[ra], v159\n" \
    "	v_mad_u32_u24 v142, v159, %[rsa], v158\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 28\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v158, s68, v154\n" \
    "	v_xor_b32_e32 v158, v158, v157\n" \
    "	v_lshlrev_b32_e32 v158, 4, v158\n" \
    "	v_add_u32_e32 v159, 56, v156\n" \
    "	v_add_u32_e32 v159, s67, v159\n" \
    "	v_min_u32_e32 v159, %[ra], v159\n" \
    "	v_mad_u32_u24 v143, v159, %[rsa], v158\n" \
    "	s_mul_i32 s67, %[wave], 64\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 0\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v158, s68, v154\n" \
    "	v_xor_b32_e32 v158, v158, v157\n" \
    "	v_lshlrev_b32_e32 v158, 4, v158\n" \
    "	v_add_u32_e32 v159, 0, v156\n" \
    "	v_add_u32_e32 v159, s67, v159\n" \
    "	v_min_u32_e32 v159, %[rw], v159\n" \
    "	v_mad_u32_u24 v144, v159, %[rsw], v158\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 4\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v158, s68, v154\n" \
    "	v_xor_b32_e32 v158, v158, v157\n" \
    "	v_lshlrev_b32_e32 v158, 4, v158\n" \
    "	v_add_u32_e32 v159, 8, v156\n" \
    "	v_add_u32_e32 v159, s67, v159\n" \
    "	v_min_u32_e32 v159, %[rw], v159\n" \
    "	v_mad_u32_u24 v145, v159, %[rsw], v158\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 8\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v158, s68, v154\n" \
    "	v_xor_b32_e32 v158, v158, v157\n" \
    "	v_lshlrev_b32_e32 v158, 4, v158\n" \
    "	v_add_u32_e32 v159, 16, v156\n" \
    "	v_add_u32_e32 v159, s67, v159\n" \
    "	v_min_u32_e32 v159, %[rw], v159\n" \
    "	v_mad_u32_u24 v146, v159, %[rsw], v158\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 12\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v158, s68, v154\n" \
    "	v_xor_b32_e32 v158, v158, v157\n" \
    "	v_lshlrev_b32_e32 v158, 4, v158\n" \
    "	v_add_u32_e32 v159, 24, v156\n" \
    "	v_add_u32_e32 v159, s67, v159\n" \
    "	v_min_u32_e32 v159, %[rw], v159\n" \
    "	v_mad_u32_u24 v147, v159, %[rsw], v158\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 16\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v158, s68, v154\n" \
    "	v_xor_b32_e32 v158, v158, v157\n" \
    "	v_lshlrev_b32_e32 v158, 4, v158\n" \
    "	v_add_u32_e32 v159, 32, v156\n" \
    "	v_add_u32_e32 v159, s67, v159\n" \
    "	v_min_u32_e32 v159, %[rw], v159\n" \
    "	v_mad_u32_u24 v148, v159, %[rsw], v158\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 20\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v158, s68, v154\n" \
    "	v_xor_b32_e32 v158, v158, v157\n" \
    "	v_lshlrev_b32_e32 v158, 4, v158\n" \
    "	v_add_u32_e32 v159, 40, v156\n" \
    "	v_add_u32_e32 v159, s67, v159\n" \
    "	v_min_u32_e32 v159, %[rw], v159\n" \
    "	v_mad_u32_u24 v149, v159, %[rsw], v158\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 24\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v158, s68, v154\n" \
    "	v_xor_b32_e32 v158, v158, v157\n" \
    "	v_lshlrev_b32_e32 v158, 4, v158\n" \
    "	v_add_u32_e32 v159, 48, v156\n" \
    "	v_add_u32_e32 v159, s67, v159\n" \
    "	v_min_u32_e32 v159, %[rw], v159\n" \
    "	v_mad_u32_u24 v150, v159, %[rsw], v158\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 28\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v158, s68, v154\n" \
    "	v_xor_b32_e32 v158, v158, v157\n" \
    "	v_lshlrev_b32_e32 v158, 4, v158\n" \
    "	v_add_u32_e32 v159, 56, v156\n" \
    "	v_add_u32_e32 v159, s67, v159\n" \
    "	v_min_u32_e32 v159, %[rw], v159\n" \
    "	v_mad_u32_u24 v151, v159, %[rsw], v158\n" \
    "	s_lshl_b32 s67, %[wave], 13\n" \
    "	s_add_u32 s61, %[lds], s67\n" \
    "	s_mul_i32 s67, %[wave], 8192\n" \
    "	s_add_u32 s69, %[lds], s67\n" \
    "	s_mov_b64 s[62:63], %[ap]\n" \
    "	s_mov_b64 s[64:65], %[wp]\n" \
    "	s_cmp_eq_u32 %[zero], 0\n" \
    "	s_cbranch_scc1 KEEP_%=\n" \
    "	v_accvgpr_write_b32 a0, 0\n" \
    "	v_accvgpr_write_b32 a1, 0\n" \
    "	v_accvgpr_write_b32 a2, 0\n" \
    "	v_accvgpr_write_b32 a3, 0\n" \
    "	v_accvgpr_write_b32 a4, 0\n" \
    "	v_accvgpr_write_b32 a5, 0\n" \
    "	v_accvgpr_write_b32 a6, 0\n" \
    "	v_accvgpr_write_b32 a7, 0\n" \
    "	v_accvgpr_write_b32 a8, 0\n" \
    "	v_accvgpr_write_b32 a9, 0\n" \
    "	v_accvgpr_write_b32 a10, 0\n" \
    "	v_accvgpr_write_b32 a11, 0\n" \
    "	v_accvgpr_write_b32 a12, 0\n" \
    "	v_accvgpr_write_b32 a13, 0\n" \
    "	v_accvgpr_write_b32 a14, 0\n" \
    "	v_accvgpr_write_b32 a15, 0\n" \
    "	v_accvgpr_write_b32 a16, 0\n" \
    "	v_accvgpr_write_b32 a17, 0\n" \
    "	v_accvgpr_write_b32 a18, 0\n" \
    "	v_accvgpr_write_b32 a19, 0\n" \
    "	v_accvgpr_write_b32 a20, 0\n" \
    "	v_accvgpr_write_b32 a21, 0\n" \
    "	v_accvgpr_write_b32 a22, 0\n" \
    "	v_accvgpr_write_b32 a23, 0\n" \
    "	v_accvgpr_write_b32 a24, 0\n" \
    "	v_accvgpr_write_b32 a25, 0\n" \
    "	v_accvgpr_write_b32 a26, 0\n" \
    "	v_accvgpr_write_b32 a27, 0\n" \
    "	v_accvgpr_write_b32 a28, 0\n" \
    "	v_accvgpr_write_b32 a29, 0\n" \
    "	v_accvgpr_write_b32 a30, 0\n" \
    "	v_accvgpr_write_b32 a31, 0\n" \
    "	v_accvgpr_write_b32 a32, 0\n" \
    "	v_accvgpr_write_b32 a33, 0\n" \
    "	v_accvgpr_write_b32 a34, 0\n" \
    "	v_accvgpr_write_b32 a35, 0\n" \
    "	v_accvgpr_write_b32 a36, 0\n" \
    "	v_accvgpr_write_b32 a37, 0\n" \
    "	v_accvgpr_write_b32 a38, 0\n" \
    "	v_accvgpr_write_b32 a39, 0\n" \
    "	v_accvgpr_write_b32 a40, 0\n" \
    "	v_accvgpr_write_b32 a41, 0\n" \
    "	v_accvgpr_write_b32 a42, 0\n" \
    "	v_accvgpr_write_b32 a43, 0\n" \
    "	v_accvgpr_write_b32 a44, 0\n" \
    "	v_accvgpr_write_b32 a45, 0\n" \
    "	v_accvgpr_write_b32 a46, 0\n" \
    "	v_accvgpr_write_b32 a47, 0\n" \
    "	v_accvgpr_write_b32 a48, 0\n" \
    "	v_accvgpr_write_b32 a49, 0\n" \
    "	v_accvgpr_write_b32 a50, 0\n" \
    "	v_accvgpr_write_b32 a51, 0\n" \
    "	v_accvgpr_write_b32 a52, 0\n" \
    "	v_accvgpr_write_b32 a53, 0\n" \
    "	v_accvgpr_write_b32 a54, 0\n" \
    "	v_accvgpr_write_b32 a55, 0\n" \
    "	v_accvgpr_write_b32 a56, 0\n" \
    "	v_accvgpr_write_b32 a57, 0\n" \
    "	v_accvgpr_write_b32 a58, 0\n" \
    "	v_accvgpr_write_b32 a59, 0\n" \
    "	v_accvgpr_write_b32 a60, 0\n" \
    "	v_accvgpr_write_b32 a61, 0\n" \
    "	v_accvgpr_write_b32 a62, 0\n" \
    "	v_accvgpr_write_b32 a63, 0\n" \
    "	v_accvgpr_write_b32 a64, 0\n" \
    "	v_accvgpr_write_b32 a65, 0\n" \
    "	v_accvgpr_write_b32 a66, 0\n" \
    "	v_accvgpr_write_b32 a67, 0\n" \
    "	v_accvgpr_write_b32 a68, 0\n" \
    "	v_accvgpr_write_b32 a69, 0\n" \
    "	v_accvgpr_write_b32 a70, 0\n" \
    "	v_accvgpr_write_b32 a71, 0\n" \
    "	v_accvgpr_write_b32 a72, 0\n" \
    "	v_accvgpr_write_b32 a73, 0\n" \
    "	v_accvgpr_write_b32 a74, 0\n" \
    "	v_accvgpr_write_b32 a75, 0\n" \
    "	v_accvgpr_write_b32 a76, 0\n" \
    "	v_accvgpr_write_b32 a77, 0\n" \
    "	v_accvgpr_write_b32 a78, 0\n" \
    "	v_accvgpr_write_b32 a79, 0\n" \
    "	v_accvgpr_write_b32 a80, 0\n" \
    "	v_accvgpr_write_b32 a81, 0\n" \
    "	v_accvgpr_write_b32 a82, 0\n" \
    "	v_accvgpr_write_b32 a83, 0\n" \
    "	v_accvgpr_write_b32 a84, 0\n" \
    "	v_accvgpr_write_b32 a85, 0\n" \
    "	v_accvgpr_write_b32 a86, 0\n" \
    "	v_accvgpr_write_b32 a87, 0\n" \
    "	v_accvgpr_write_b32 a88, 0\n" \
    "	v_accvgpr_write_b32 a89, 0\n" \
    "	v_accvgpr_write_b32 a90, 0\n" \
    "	v_accvgpr_write_b32 a91, 0\n" \
    "	v_accvgpr_write_b32 a92, 0\n" \
    "	v_accvgpr_write_b32 a93, 0\n" \
    "	v_accvgpr_write_b32 a94, 0\n" \
    "	v_accvgpr_write_b32 a95, 0\n" \
    "	v_accvgpr_write_b32 a96, 0\n" \
    "	v_accvgpr_write_b32 a97, 0\n" \
    "	v_accvgpr_write_b32 a98, 0\n" \
    "	v_accvgpr_write_b32 a99, 0\n" \
    "	v_accvgpr_write_b32 a100, 0\n" \
    "	v_accvgpr_write_b32 a101, 0\n" \
    "	v_accvgpr_write_b32 a102, 0\n" \
    "	v_accvgpr_write_b32 a103, 0\n" \
    "	v_accvgpr_write_b32 a104, 0\n" \
    "	v_accvgpr_write_b32 a105, 0\n" \
    "	v_accvgpr_write_b32 a106, 0\n" \
    "	v_accvgpr_write_b32 a107, 0\n" \
    "	v_accvgpr_write_b32 a108, 0\n" \
    "	v_accvgpr_write_b32 a109, 0\n" \
    "	v_accvgpr_write_b32 a110, 0\n" \
    "	v_accvgpr_write_b32 a111, 0\n" \
    "	v_accvgpr_write_b32 a112, 0\n" \
    "	v_accvgpr_write_b32 a113, 0\n" \
    "	v_accvgpr_write_b32 a114, 0\n" \
    "	v_accvgpr_write_b32 a115, 0\n" \
    "	v_accvgpr_write_b32 a116, 0\n" \
    "	v_accvgpr_write_b32 a117, 0\n" \
    "	v_accvgpr_write_b32 a118, 0\n" \
    "	v_accvgpr_write_b32 a119, 0\n" \
    "	v_accvgpr_write_b32 a120, 0\n" \
    "	v_accvgpr_write_b32 a121, 0\n" \
    "	v_accvgpr_write_b32 a122, 0\n" \
    "	v_accvgpr_write_b32 a123, 0\n" \
    "	v_accvgpr_write_b32 a124, 0\n" \
    "	v_accvgpr_write_b32 a125, 0\n" \
    "	v_accvgpr_write_b32 a126, 0\n" \
    "	v_accvgpr_write_b32 a127, 0\n" \
    "	v_accvgpr_write_b32 a128, 0\n" \
    "	v_accvgpr_write_b32 a129, 0\n" \
    "	v_accvgpr_write_b32 a130, 0\n" \
    "	v_accvgpr_write_b32 a131, 0\n" \
    "	v_accvgpr_write_b32 a132, 0\n" \
    "	v_accvgpr_write_b32 a133, 0\n" \
    "	v_accvgpr_write_b32 a134, 0\n" \
    "	v_accvgpr_write_b32 a135, 0\n" \
    "	v_accvgpr_write_b32 a136, 0\n" \
    "	v_accvgpr_write_b32 a137, 0\n" \
    "	v_accvgpr_write_b32 a138, 0\n" \
    "	v_accvgpr_write_b32 a139, 0\n" \
    "	v_accvgpr_write_b32 a140, 0\n" \
    "	v_accvgpr_write_b32 a141, 0\n" \
    "	v_accvgpr_write_b32 a142, 0\n" \
    "	v_accvgpr_write_b32 a143, 0\n" \
    "	v_accvgpr_write_b32 a144, 0\n" \
    "	v_accvgpr_write_b32 a145, 0\n" \
    "	v_accvgpr_write_b32 a146, 0\n" \
    "	v_accvgpr_write_b32 a147, 0\n" \
    "	v_accvgpr_write_b32 a148, 0\n" \
    "	v_accvgpr_write_b32 a149, 0\n" \
    "	v_accvgpr_write_b32 a150, 0\n" \
    "	v_accvgpr_write_b32 a151, 0\n" \
    "	v_accvgpr_write_b32 a152, 0\n" \
    "	v_accvgpr_write_b32 a153, 0\n" \
    "	v_accvgpr_write_b32 a154, 0\n" \
    "	v_accvgpr_write_b32 a155, 0\n" \
    "	v_accvgpr_write_b32 a156, 0\n" \
    "	v_accvgpr_write_b32 a157, 0\n" \
    "	v_accvgpr_write_b32 a158, 0\n" \
    "	v_accvgpr_write_b32 a159, 0\n" \
    "	v_accvgpr_write_b32 a160, 0\n" \
    "	v_accvgpr_write_b32 a161, 0\n" \
    "	v_accvgpr_write_b32 a162, 0\n" \
    "	v_accvgpr_write_b32 a163, 0\n" \
    "	v_accvgpr_write_b32 a164, 0\n" \
    "	v_accvgpr_write_b32 a165, 0\n" \
    "	v_accvgpr_write_b32 a166, 0\n" \
    "	v_accvgpr_write_b32 a167, 0\n" \
    "	v_accvgpr_write_b32 a168, 0\n" \
    "	v_accvgpr_write_b32 a169, 0\n" \
    "	v_accvgpr_write_b32 a170, 0\n" \
    "	v_accvgpr_write_b32 a171, 0\n" \
    "	v_accvgpr_write_b32 a172, 0\n" \
    "	v_accvgpr_write_b32 a173, 0\n" \
    "	v_accvgpr_write_b32 a174, 0\n" \
    "	v_accvgpr_write_b32 a175, 0\n" \
    "	v_accvgpr_write_b32 a176, 0\n" \
    "	v_accvgpr_write_b32 a177, 0\n" \
    "	v_accvgpr_write_b32 a178, 0\n" \
    "	v_accvgpr_write_b32 a179, 0\n" \
    "	v_accvgpr_write_b32 a180, 0\n" \
    "	v_accvgpr_write_b32 a181, 0\n" \
    "	v_accvgpr_write_b32 a182, 0\n" \
    "	v_accvgpr_write_b32 a183, 0\n" \
    "	v_accvgpr_write_b32 a184, 0\n" \
    "	v_accvgpr_write_b32 a185, 0\n" \
    "	v_accvgpr_write_b32 a186, 0\n" \
    "	v_accvgpr_write_b32 a187, 0\n" \
    "	v_accvgpr_write_b32 a188, 0\n" \
    "	v_accvgpr_write_b32 a189, 0\n" \
    "	v_accvgpr_write_b32 a190, 0\n" \
    "	v_accvgpr_write_b32 a191, 0\n" \
    "	v_accvgpr_write_b32 a192, 0\n" \
    "	v_accvgpr_write_b32 a193, 0\n" \
    "	v_accvgpr_write_b32 a194, 0\n" \
    "	v_accvgpr_write_b32 a195, 0\n" \
    "	v_accvgpr_write_b32 a196, 0\n" \
    "	v_accvgpr_write_b32 a197, 0\n" \
    "	v_accvgpr_write_b32 a198, 0\n" \
    "	v_accvgpr_write_b32 a199, 0\n" \
    "	v_accvgpr_write_b32 a200, 0\n" \
    "	v_accvgpr_write_b32 a201, 0\n" \
    "	v_accvgpr_write_b32 a202, 0\n" \
    "	v_accvgpr_write_b32 a203, 0\n" \
    "	v_accvgpr_write_b32 a204, 0\n" \
    "	v_accvgpr_write_b32 a205, 0\n" \
    "	v_accvgpr_write_b32 a206, 0\n" \
    "	v_accvgpr_write_b32 a207, 0\n" \
    "	v_accvgpr_write_b32 a208, 0\n" \
    "	v_accvgpr_write_b32 a209, 0\n" \
    "	v_accvgpr_write_b32 a210, 0\n" \
    "	v_accvgpr_write_b32 a211, 0\n" \
    "	v_accvgpr_write_b32 a212, 0\n" \
    "	v_accvgpr_write_b32 a213, 0\n" \
    "	v_accvgpr_write_b32 a214, 0\n" \
    "	v_accvgpr_write_b32 a215, 0\n" \
    "	v_accvgpr_write_b32 a216, 0\n" \
    "	v_accvgpr_write_b32 a217, 0\n" \
    "	v_accvgpr_write_b32 a218, 0\n" \
    "	v_accvgpr_write_b32 a219, 0\n" \
    "	v_accvgpr_write_b32 a220, 0\n" \
    "	v_accvgpr_write_b32 a221, 0\n" \
    "	v_accvgpr_write_b32 a222, 0\n" \
    "	v_accvgpr_write_b32 a223, 0\n" \
    "	v_accvgpr_write_b32 a224, 0\n" \
    "	v_accvgpr_write_b32 a225, 0\n" \
    "	v_accvgpr_write_b32 a226, 0\n" \
    "	v_accvgpr_write_b32 a227, 0\n" \
    "	v_accvgpr_write_b32 a228, 0\n" \
    "	v_accvgpr_write_b32 a229, 0\n" \
    "	v_accvgpr_write_b32 a230, 0\n" \
    "	v_accvgpr_write_b32 a231, 0\n" \
    "	v_accvgpr_write_b32 a232, 0\n" \
    "	v_accvgpr_write_b32 a233, 0\n" \
    "	v_accvgpr_write_b32 a234, 0\n" \
    "	v_accvgpr_write_b32 a235, 0\n" \
    "	v_accvgpr_write_b32 a236, 0\n" \
    "	v_accvgpr_write_b32 a237, 0\n" \
    "	v_accvgpr_write_b32 a238, 0\n" \
    "	v_accvgpr_write_b32 a239, 0\n" \
    "	v_accvgpr_write_b32 a240, 0\n" \
    "	v_accvgpr_write_b32 a241, 0\n" \
    "	v_accvgpr_write_b32 a242, 0\n" \
    "	v_accvgpr_write_b32 a243, 0\n" \
    "	v_accvgpr_write_b32 a244, 0\n" \
    "	v_accvgpr_write_b32 a245, 0\n" \
    "	v_accvgpr_write_b32 a246, 0\n" \
    "	v_accvgpr_write_b32 a247, 0\n" \
    "	v_accvgpr_write_b32 a248, 0\n" \
    "	v_accvgpr_write_b32 a249, 0\n" \
    "	v_accvgpr_write_b32 a250, 0\n" \
    "	v_accvgpr_write_b32 a251, 0\n" \
    "	v_accvgpr_write_b32 a252, 0\n" \
    "	v_accvgpr_write_b32 a253, 0\n" \
    "	v_accvgpr_write_b32 a254, 0\n" \
    "	v_accvgpr_write_b32 a255, 0\n" \
    "KEEP_%=:\n" \
    "	s_add_u32 m0, s61, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v136, s[62:63]\n" \
    "	s_add_u32 m0, s61, 1024\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v137, s[62:63]\n" \
    "	s_add_u32 m0, s61, 2048\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v138, s[62:63]\n" \
    "	s_add_u32 m0, s61, 3072\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v139, s[62:63]\n" \
    "	s_add_u32 m0, s61, 4096\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v140, s[62:63]\n" \
    "	s_add_u32 m0, s61, 5120\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v141, s[62:63]\n" \
    "	s_add_u32 m0, s61, 6144\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v142, s[62:63]\n" \
    "	s_add_u32 m0, s61, 7168\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v143, s[62:63]\n" \
    "	s_add_u32 m0, s69, 32768\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v144, s[64:65]\n" \
    "	s_add_u32 m0, s69, 33792\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v145, s[64:65]\n" \
    "	s_add_u32 m0, s69, 34816\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v146, s[64:65]\n" \
    "	s_add_u32 m0, s69, 35840\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v147, s[64:65]\n" \
    "	s_add_u32 m0, s69, 36864\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v148, s[64:65]\n" \
    "	s_add_u32 m0, s69, 37888\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v149, s[64:65]\n" \
    "	s_add_u32 m0, s69, 38912\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v150, s[64:65]\n" \
    "	s_add_u32 m0, s69, 39936\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v151, s[64:65]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_waitcnt vmcnt(0)\n" \
    "	s_barrier\n" \
    "	ds_read_b128 v[32:35], v132 offset:0\n" \
    "	ds_read_b128 v[0:3], v128 offset:0\n" \
    "	ds_read_b128 v[4:7], v128 offset:2048\n" \
    "	ds_read_b128 v[8:11], v128 offset:4096\n" \
    "	ds_read_b128 v[12:15], v128 offset:6144\n" \
    "	ds_read_b128 v[16:19], v128 offset:8192\n" \
    "	ds_read_b128 v[20:23], v128 offset:10240\n" \
    "	ds_read_b128 v[24:27], v128 offset:12288\n" \
    "	ds_read_b128 v[28:31], v128 offset:14336\n" \
    "	ds_read_b128 v[36:39], v132 offset:2048\n" \
    "	ds_read_b128 v[40:43], v132 offset:4096\n" \
    "	ds_read_b128 v[44:47], v132 offset:6144\n" \
    "	ds_read_b128 v[48:51], v132 offset:8192\n" \
    "	ds_read_b128 v[52:55], v132 offset:10240\n" \
    "	ds_read_b128 v[56:59], v132 offset:12288\n" \
    "	ds_read_b128 v[60:63], v132 offset:14336\n" \
    "	s_mov_b32 s60, %[trips]\n" \
    "	s_cmp_eq_u32 s60, 0\n" \
    "	s_cbranch_scc1 LAST_%=\n" \
    "LOOP_%=:\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[32:35], v[0:3], a[0:3]\n" \
    "	s_add_u32 m0, s61, 65536\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v136, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[32:35], v[4:7], a[32:35]\n" \
    "	ds_read_b128 v[96:99], v133 offset:0\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[32:35], v[8:11], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[32:35], v[12:15], a[96:99]\n" \
    "	ds_read_b128 v[64:67], v129 offset:0\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[32:35], v[16:19], a[128:131]\n" \
    "	s_add_u32 m0, s61, 66560\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v137, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[32:35], v[20:23], a[160:163]\n" \
    "	ds_read_b128 v[68:71], v129 offset:2048\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[32:35], v[24:27], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[32:35], v[28:31], a[224:227]\n" \
    "	ds_read_b128 v[72:75], v129 offset:4096\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[36:39], v[0:3], a[4:7]\n" \
    "	s_add_u32 m0, s61, 67584\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v138, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[36:39], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[76:79], v129 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[36:39], v[8:11], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[36:39], v[12:15], a[100:103]\n" \
    "	ds_read_b128 v[80:83], v129 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[36:39], v[16:19], a[132:135]\n" \
    "	s_add_u32 m0, s61, 68608\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v139, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[36:39], v[20:23], a[164:167]\n" \
    "	ds_read_b128 v[84:87], v129 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[36:39], v[24:27], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[36:39], v[28:31], a[228:231]\n" \
    "	ds_read_b128 v[88:91], v129 offset:12288\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[40:43], v[0:3], a[8:11]\n" \
    "	s_add_u32 m0, s61, 69632\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v140, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[40:43], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[92:95], v129 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[40:43], v[8:11], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[40:43], v[12:15], a[104:107]\n" \
    "	ds_read_b128 v[100:103], v133 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[40:43], v[16:19], a[136:139]\n" \
    "	s_add_u32 m0, s61, 70656\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v141, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[40:43], v[20:23], a[168:171]\n" \
    "	ds_read_b128 v[104:107], v133 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[40:43], v[24:27], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[40:43], v[28:31], a[232:235]\n" \
    "	ds_read_b128 v[108:111], v133 offset:6144\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[44:47], v[0:3], a[12:15]\n" \
    "	s_add_u32 m0, s61, 71680\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v142, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[44:47], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[112:115], v133 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[44:47], v[8:11], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[44:47], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[116:119], v133 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[44:47], v[16:19], a[140:143]\n" \
    "	s_add_u32 m0, s61, 72704\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v143, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[44:47], v[20:23], a[172:175]\n" \
    "	ds_read_b128 v[120:123], v133 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[44:47], v[24:27], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[44:47], v[28:31], a[236:239]\n" \
    "	ds_read_b128 v[124:127], v133 offset:14336\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[48:51], v[0:3], a[16:19]\n" \
    "	s_add_u32 m0, s69, 98304\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v144, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[48:51], v[4:7], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[48:51], v[8:11], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[48:51], v[12:15], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[48:51], v[16:19], a[144:147]\n" \
    "	s_add_u32 m0, s69, 99328\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v145, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[48:51], v[20:23], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[48:51], v[24:27], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[48:51], v[28:31], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[52:55], v[0:3], a[20:23]\n" \
    "	s_add_u32 m0, s69, 100352\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v146, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[52:55], v[4:7], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[52:55], v[8:11], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[52:55], v[12:15], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[52:55], v[16:19], a[148:151]\n" \
    "	s_add_u32 m0, s69, 101376\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v147, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[52:55], v[20:23], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[52:55], v[24:27], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[52:55], v[28:31], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[56:59], v[0:3], a[24:27]\n" \
    "	s_add_u32 m0, s69, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v148, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[56:59], v[4:7], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[56:59], v[8:11], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[56:59], v[12:15], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[56:59], v[16:19], a[152:155]\n" \
    "	s_add_u32 m0, s69, 103424\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v149, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[56:59], v[20:23], a[184:187]\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[56:59], v[24:27], a[216:219]\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[56:59], v[28:31], a[248:251]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[60:63], v[0:3], a[28:31]\n" \
    "	s_add_u32 m0, s69, 104448\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v150, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[60:63], v[4:7], a[60:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[60:63], v[8:11], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[60:63], v[12:15], a[124:127]\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[60:63], v[16:19], a[156:159]\n" \
    "	s_add_u32 m0, s69, 105472\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v151, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[60:63], v[20:23], a[188:191]\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[60:63], v[24:27], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[60:63], v[28:31], a[252:255]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[96:99], v[64:67], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[96:99], v[68:71], a[32:35]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[96:99], v[72:75], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[96:99], v[76:79], a[96:99]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[96:99], v[80:83], a[128:131]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[96:99], v[84:87], a[160:163]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[96:99], v[88:91], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[96:99], v[92:95], a[224:227]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[100:103], v[64:67], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[100:103], v[68:71], a[36:39]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[100:103], v[72:75], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[100:103], v[76:79], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[100:103], v[80:83], a[132:135]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[100:103], v[84:87], a[164:167]\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[100:103], v[88:91], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[100:103], v[92:95], a[228:231]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[104:107], v[64:67], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[104:107], v[68:71], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[104:107], v[72:75], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[104:107], v[76:79], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[104:107], v[80:83], a[136:139]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[104:107], v[84:87], a[168:171]\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[104:107], v[88:91], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[104:107], v[92:95], a[232:235]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[108:111], v[64:67], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[108:111], v[68:71], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[108:111], v[72:75], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[108:111], v[76:79], a[108:111]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[108:111], v[80:83], a[140:143]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[108:111], v[84:87], a[172:175]\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[108:111], v[88:91], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[108:111], v[92:95], a[236:239]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[112:115], v[64:67], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[112:115], v[68:71], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[112:115], v[72:75], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[112:115], v[76:79], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[112:115], v[80:83], a[144:147]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[112:115], v[84:87], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[112:115], v[88:91], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[112:115], v[92:95], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(2)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[116:119], v[64:67], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[116:119], v[68:71], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[116:119], v[72:75], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[116:119], v[76:79], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[116:119], v[80:83], a[148:151]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[116:119], v[84:87], a[180:183]\n" \
    "	s_waitcnt vmcnt(0)\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	s_barrier\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[116:119], v[88:91], a[212:215]\n" \
    "	ds_read_b128 v[32:35], v134 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[116:119], v[92:95], a[244:247]\n" \
    "	ds_read_b128 v[0:3], v130 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[120:123], v[64:67], a[24:27]\n" \
    "	ds_read_b128 v[4:7], v130 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[120:123], v[68:71], a[56:59]\n" \
    "	ds_read_b128 v[8:11], v130 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[120:123], v[72:75], a[88:91]\n" \
    "	ds_read_b128 v[12:15], v130 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[120:123], v[76:79], a[120:123]\n" \
    "	ds_read_b128 v[16:19], v130 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[120:123], v[80:83], a[152:155]\n" \
    "	ds_read_b128 v[20:23], v130 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[120:123], v[84:87], a[184:187]\n" \
    "	ds_read_b128 v[24:27], v130 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[120:123], v[88:91], a[216:219]\n" \
    "	ds_read_b128 v[28:31], v130 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[120:123], v[92:95], a[248:251]\n" \
    "	ds_read_b128 v[36:39], v134 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[124:127], v[64:67], a[28:31]\n" \
    "	ds_read_b128 v[40:43], v134 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[124:127], v[68:71], a[60:63]\n" \
    "	ds_read_b128 v[44:47], v134 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[124:127], v[72:75], a[92:95]\n" \
    "	ds_read_b128 v[48:51], v134 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[124:127], v[76:79], a[124:127]\n" \
    "	ds_read_b128 v[52:55], v134 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[124:127], v[80:83], a[156:159]\n" \
    "	ds_read_b128 v[56:59], v134 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[124:127], v[84:87], a[188:191]\n" \
    "	ds_read_b128 v[60:63], v134 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[124:127], v[88:91], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[124:127], v[92:95], a[252:255]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[32:35], v[0:3], a[0:3]\n" \
    "	s_add_u32 m0, s61, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v136, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[32:35], v[4:7], a[32:35]\n" \
    "	ds_read_b128 v[96:99], v135 offset:0\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[32:35], v[8:11], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[32:35], v[12:15], a[96:99]\n" \
    "	ds_read_b128 v[64:67], v131 offset:0\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[32:35], v[16:19], a[128:131]\n" \
    "	s_add_u32 m0, s61, 1024\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v137, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[32:35], v[20:23], a[160:163]\n" \
    "	ds_read_b128 v[68:71], v131 offset:2048\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[32:35], v[24:27], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[32:35], v[28:31], a[224:227]\n" \
    "	ds_read_b128 v[72:75], v131 offset:4096\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[36:39], v[0:3], a[4:7]\n" \
    "	s_add_u32 m0, s61, 2048\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v138, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[36:39], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[76:79], v131 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[36:39], v[8:11], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[36:39], v[12:15], a[100:103]\n" \
    "	ds_read_b128 v[80:83], v131 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[36:39], v[16:19], a[132:135]\n" \
    "	s_add_u32 m0, s61, 3072\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v139, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[36:39], v[20:23], a[164:167]\n" \
    "	ds_read_b128 v[84:87], v131 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[36:39], v[24:27], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[36:39], v[28:31], a[228:231]\n" \
    "	ds_read_b128 v[88:91], v131 offset:12288\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[40:43], v[0:3], a[8:11]\n" \
    "	s_add_u32 m0, s61, 4096\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v140, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[40:43], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[92:95], v131 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[40:43], v[8:11], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[40:43], v[12:15], a[104:107]\n" \
    "	ds_read_b128 v[100:103], v135 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[40:43], v[16:19], a[136:139]\n" \
    "	s_add_u32 m0, s61, 5120\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v141, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[40:43], v[20:23], a[168:171]\n" \
    "	ds_read_b128 v[104:107], v135 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[40:43], v[24:27], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[40:43], v[28:31], a[232:235]\n" \
    "	ds_read_b128 v[108:111], v135 offset:6144\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[44:47], v[0:3], a[12:15]\n" \
    "	s_add_u32 m0, s61, 6144\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v142, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[44:47], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[112:115], v135 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[44:47], v[8:11], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[44:47], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[116:119], v135 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[44:47], v[16:19], a[140:143]\n" \
    "	s_add_u32 m0, s61, 7168\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v143, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[44:47], v[20:23], a[172:175]\n" \
    "	ds_read_b128 v[120:123], v135 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[44:47], v[24:27], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[44:47], v[28:31], a[236:239]\n" \
    "	ds_read_b128 v[124:127], v135 offset:14336\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[48:51], v[0:3], a[16:19]\n" \
    "	s_add_u32 m0, s69, 32768\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v144, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[48:51], v[4:7], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[48:51], v[8:11], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[48:51], v[12:15], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[48:51], v[16:19], a[144:147]\n" \
    "	s_add_u32 m0, s69, 33792\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v145, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[48:51], v[20:23], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[48:51], v[24:27], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[48:51], v[28:31], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[52:55], v[0:3], a[20:23]\n" \
    "	s_add_u32 m0, s69, 34816\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v146, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[52:55], v[4:7], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[52:55], v[8:11], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[52:55], v[12:15], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[52:55], v[16:19], a[148:151]\n" \
    "	s_add_u32 m0, s69, 35840\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v147, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[52:55], v[20:23], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[52:55], v[24:27], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[52:55], v[28:31], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[56:59], v[0:3], a[24:27]\n" \
    "	s_add_u32 m0, s69, 36864\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v148, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[56:59], v[4:7], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[56:59], v[8:11], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[56:59], v[12:15], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[56:59], v[16:19], a[152:155]\n" \
    "	s_add_u32 m0, s69, 37888\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v149, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[56:59], v[20:23], a[184:187]\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[56:59], v[24:27], a[216:219]\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[56:59], v[28:31], a[248:251]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[60:63], v[0:3], a[28:31]\n" \
    "	s_add_u32 m0, s69, 38912\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v150, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[60:63], v[4:7], a[60:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[60:63], v[8:11], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[60:63], v[12:15], a[124:127]\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[60:63], v[16:19], a[156:159]\n" \
    "	s_add_u32 m0, s69, 39936\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v151, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[60:63], v[20:23], a[188:191]\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[60:63], v[24:27], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[60:63], v[28:31], a[252:255]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[96:99], v[64:67], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[96:99], v[68:71], a[32:35]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[96:99], v[72:75], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[96:99], v[76:79], a[96:99]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[96:99], v[80:83], a[128:131]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[96:99], v[84:87], a[160:163]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[96:99], v[88:91], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[96:99], v[92:95], a[224:227]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[100:103], v[64:67], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[100:103], v[68:71], a[36:39]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[100:103], v[72:75], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[100:103], v[76:79], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[100:103], v[80:83], a[132:135]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[100:103], v[84:87], a[164:167]\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[100:103], v[88:91], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[100:103], v[92:95], a[228:231]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[104:107], v[64:67], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[104:107], v[68:71], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[104:107], v[72:75], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[104:107], v[76:79], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[104:107], v[80:83], a[136:139]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[104:107], v[84:87], a[168:171]\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[104:107], v[88:91], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[104:107], v[92:95], a[232:235]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[108:111], v[64:67], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[108:111], v[68:71], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[108:111], v[72:75], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[108:111], v[76:79], a[108:111]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[108:111], v[80:83], a[140:143]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[108:111], v[84:87], a[172:175]\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[108:111], v[88:91], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[108:111], v[92:95], a[236:239]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[112:115], v[64:67], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[112:115], v[68:71], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[112:115], v[72:75], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[112:115], v[76:79], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[112:115], v[80:83], a[144:147]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[112:115], v[84:87], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[112:115], v[88:91], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[112:115], v[92:95], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(2)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[116:119], v[64:67], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[116:119], v[68:71], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[116:119], v[72:75], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[116:119], v[76:79], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[116:119], v[80:83], a[148:151]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[116:119], v[84:87], a[180:183]\n" \
    "	s_waitcnt vmcnt(0)\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	s_barrier\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[116:119], v[88:91], a[212:215]\n" \
    "	ds_read_b128 v[32:35], v132 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[116:119], v[92:95], a[244:247]\n" \
    "	ds_read_b128 v[0:3], v128 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[120:123], v[64:67], a[24:27]\n" \
    "	ds_read_b128 v[4:7], v128 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[120:123], v[68:71], a[56:59]\n" \
    "	ds_read_b128 v[8:11], v128 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[120:123], v[72:75], a[88:91]\n" \
    "	ds_read_b128 v[12:15], v128 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[120:123], v[76:79], a[120:123]\n" \
    "	ds_read_b128 v[16:19], v128 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[120:123], v[80:83], a[152:155]\n" \
    "	ds_read_b128 v[20:23], v128 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[120:123], v[84:87], a[184:187]\n" \
    "	ds_read_b128 v[24:27], v128 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[120:123], v[88:91], a[216:219]\n" \
    "	ds_read_b128 v[28:31], v128 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[120:123], v[92:95], a[248:251]\n" \
    "	ds_read_b128 v[36:39], v132 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[124:127], v[64:67], a[28:31]\n" \
    "	ds_read_b128 v[40:43], v132 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[124:127], v[68:71], a[60:63]\n" \
    "	ds_read_b128 v[44:47], v132 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[124:127], v[72:75], a[92:95]\n" \
    "	ds_read_b128 v[48:51], v132 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[124:127], v[76:79], a[124:127]\n" \
    "	ds_read_b128 v[52:55], v132 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[124:127], v[80:83], a[156:159]\n" \
    "	ds_read_b128 v[56:59], v132 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[124:127], v[84:87], a[188:191]\n" \
    "	ds_read_b128 v[60:63], v132 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[124:127], v[88:91], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[124:127], v[92:95], a[252:255]\n" \
    "	s_sub_u32 s60, s60, 1\n" \
    "	s_cmp_eq_u32 s60, 0\n" \
    "	s_cbranch_scc0 LOOP_%=\n" \
    "LAST_%=:\n" \
    "	s_cmp_eq_u32 %[rem], 1\n" \
    "	s_cbranch_scc1 LAST1_%=\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[32:35], v[0:3], a[0:3]\n" \
    "	s_add_u32 m0, s61, 65536\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v136, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[32:35], v[4:7], a[32:35]\n" \
    "	ds_read_b128 v[96:99], v133 offset:0\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[32:35], v[8:11], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[32:35], v[12:15], a[96:99]\n" \
    "	ds_read_b128 v[64:67], v129 offset:0\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[32:35], v[16:19], a[128:131]\n" \
    "	s_add_u32 m0, s61, 66560\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v137, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[32:35], v[20:23], a[160:163]\n" \
    "	ds_read_b128 v[68:71], v129 offset:2048\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[32:35], v[24:27], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[32:35], v[28:31], a[224:227]\n" \
    "	ds_read_b128 v[72:75], v129 offset:4096\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[36:39], v[0:3], a[4:7]\n" \
    "	s_add_u32 m0, s61, 67584\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v138, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[36:39], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[76:79], v129 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[36:39], v[8:11], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[36:39], v[12:15], a[100:103]\n" \
    "	ds_read_b128 v[80:83], v129 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[36:39], v[16:19], a[132:135]\n" \
    "	s_add_u32 m0, s61, 68608\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v139, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[36:39], v[20:23], a[164:167]\n" \
    "	ds_read_b128 v[84:87], v129 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[36:39], v[24:27], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[36:39], v[28:31], a[228:231]\n" \
    "	ds_read_b128 v[88:91], v129 offset:12288\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[40:43], v[0:3], a[8:11]\n" \
    "	s_add_u32 m0, s61, 69632\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v140, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[40:43], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[92:95], v129 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[40:43], v[8:11], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[40:43], v[12:15], a[104:107]\n" \
    "	ds_read_b128 v[100:103], v133 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[40:43], v[16:19], a[136:139]\n" \
    "	s_add_u32 m0, s61, 70656\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v141, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[40:43], v[20:23], a[168:171]\n" \
    "	ds_read_b128 v[104:107], v133 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[40:43], v[24:27], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[40:43], v[28:31], a[232:235]\n" \
    "	ds_read_b128 v[108:111], v133 offset:6144\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[44:47], v[0:3], a[12:15]\n" \
    "	s_add_u32 m0, s61, 71680\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v142, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[44:47], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[112:115], v133 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[44:47], v[8:11], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[44:47], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[116:119], v133 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[44:47], v[16:19], a[140:143]\n" \
    "	s_add_u32 m0, s61, 72704\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v143, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[44:47], v[20:23], a[172:175]\n" \
    "	ds_read_b128 v[120:123], v133 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[44:47], v[24:27], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[44:47], v[28:31], a[236:239]\n" \
    "	ds_read_b128 v[124:127], v133 offset:14336\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[48:51], v[0:3], a[16:19]\n" \
    "	s_add_u32 m0, s69, 98304\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v144, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[48:51], v[4:7], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[48:51], v[8:11], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[48:51], v[12:15], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[48:51], v[16:19], a[144:147]\n" \
    "	s_add_u32 m0, s69, 99328\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v145, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[48:51], v[20:23], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[48:51], v[24:27], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[48:51], v[28:31], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[52:55], v[0:3], a[20:23]\n" \
    "	s_add_u32 m0, s69, 100352\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v146, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[52:55], v[4:7], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[52:55], v[8:11], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[52:55], v[12:15], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[52:55], v[16:19], a[148:151]\n" \
    "	s_add_u32 m0, s69, 101376\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v147, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[52:55], v[20:23], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[52:55], v[24:27], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[52:55], v[28:31], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[56:59], v[0:3], a[24:27]\n" \
    "	s_add_u32 m0, s69, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v148, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[56:59], v[4:7], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[56:59], v[8:11], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[56:59], v[12:15], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[56:59], v[16:19], a[152:155]\n" \
    "	s_add_u32 m0, s69, 103424\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v149, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[56:59], v[20:23], a[184:187]\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[56:59], v[24:27], a[216:219]\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[56:59], v[28:31], a[248:251]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[60:63], v[0:3], a[28:31]\n" \
    "	s_add_u32 m0, s69, 104448\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v150, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[60:63], v[4:7], a[60:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[60:63], v[8:11], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[60:63], v[12:15], a[124:127]\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[60:63], v[16:19], a[156:159]\n" \
    "	s_add_u32 m0, s69, 105472\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v151, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[60:63], v[20:23], a[188:191]\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[60:63], v[24:27], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[60:63], v[28:31], a[252:255]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[96:99], v[64:67], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[96:99], v[68:71], a[32:35]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[96:99], v[72:75], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[96:99], v[76:79], a[96:99]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[96:99], v[80:83], a[128:131]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[96:99], v[84:87], a[160:163]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[96:99], v[88:91], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[96:99], v[92:95], a[224:227]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[100:103], v[64:67], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[100:103], v[68:71], a[36:39]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[100:103], v[72:75], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[100:103], v[76:79], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[100:103], v[80:83], a[132:135]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[100:103], v[84:87], a[164:167]\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[100:103], v[88:91], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[100:103], v[92:95], a[228:231]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[104:107], v[64:67], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[104:107], v[68:71], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[104:107], v[72:75], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[104:107], v[76:79], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[104:107], v[80:83], a[136:139]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[104:107], v[84:87], a[168:171]\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[104:107], v[88:91], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[104:107], v[92:95], a[232:235]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[108:111], v[64:67], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[108:111], v[68:71], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[108:111], v[72:75], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[108:111], v[76:79], a[108:111]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[108:111], v[80:83], a[140:143]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[108:111], v[84:87], a[172:175]\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[108:111], v[88:91], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[108:111], v[92:95], a[236:239]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[112:115], v[64:67], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[112:115], v[68:71], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[112:115], v[72:75], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[112:115], v[76:79], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[112:115], v[80:83], a[144:147]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[112:115], v[84:87], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[112:115], v[88:91], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[112:115], v[92:95], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(2)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[116:119], v[64:67], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[116:119], v[68:71], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[116:119], v[72:75], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[116:119], v[76:79], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[116:119], v[80:83], a[148:151]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[116:119], v[84:87], a[180:183]\n" \
    "	s_waitcnt vmcnt(0)\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	s_barrier\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[116:119], v[88:91], a[212:215]\n" \
    "	ds_read_b128 v[32:35], v134 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[116:119], v[92:95], a[244:247]\n" \
    "	ds_read_b128 v[0:3], v130 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[120:123], v[64:67], a[24:27]\n" \
    "	ds_read_b128 v[4:7], v130 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[120:123], v[68:71], a[56:59]\n" \
    "	ds_read_b128 v[8:11], v130 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[120:123], v[72:75], a[88:91]\n" \
    "	ds_read_b128 v[12:15], v130 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[120:123], v[76:79], a[120:123]\n" \
    "	ds_read_b128 v[16:19], v130 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[120:123], v[80:83], a[152:155]\n" \
    "	ds_read_b128 v[20:23], v130 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[120:123], v[84:87], a[184:187]\n" \
    "	ds_read_b128 v[24:27], v130 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[120:123], v[88:91], a[216:219]\n" \
    "	ds_read_b128 v[28:31], v130 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[120:123], v[92:95], a[248:251]\n" \
    "	ds_read_b128 v[36:39], v134 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[124:127], v[64:67], a[28:31]\n" \
    "	ds_read_b128 v[40:43], v134 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[124:127], v[68:71], a[60:63]\n" \
    "	ds_read_b128 v[44:47], v134 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[124:127], v[72:75], a[92:95]\n" \
    "	ds_read_b128 v[48:51], v134 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[124:127], v[76:79], a[124:127]\n" \
    "	ds_read_b128 v[52:55], v134 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[124:127], v[80:83], a[156:159]\n" \
    "	ds_read_b128 v[56:59], v134 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[124:127], v[84:87], a[188:191]\n" \
    "	ds_read_b128 v[60:63], v134 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[124:127], v[88:91], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[124:127], v[92:95], a[252:255]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[32:35], v[0:3], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[32:35], v[4:7], a[32:35]\n" \
    "	ds_read_b128 v[96:99], v135 offset:0\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[32:35], v[8:11], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[32:35], v[12:15], a[96:99]\n" \
    "	ds_read_b128 v[64:67], v131 offset:0\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[32:35], v[16:19], a[128:131]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[32:35], v[20:23], a[160:163]\n" \
    "	ds_read_b128 v[68:71], v131 offset:2048\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[32:35], v[24:27], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[32:35], v[28:31], a[224:227]\n" \
    "	ds_read_b128 v[72:75], v131 offset:4096\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[36:39], v[0:3], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[36:39], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[76:79], v131 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[36:39], v[8:11], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[36:39], v[12:15], a[100:103]\n" \
    "	ds_read_b128 v[80:83], v131 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[36:39], v[16:19], a[132:135]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[36:39], v[20:23], a[164:167]\n" \
    "	ds_read_b128 v[84:87], v131 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[36:39], v[24:27], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[36:39], v[28:31], a[228:231]\n" \
    "	ds_read_b128 v[88:91], v131 offset:12288\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[40:43], v[0:3], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[40:43], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[92:95], v131 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[40:43], v[8:11], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[40:43], v[12:15], a[104:107]\n" \
    "	ds_read_b128 v[100:103], v135 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[40:43], v[16:19], a[136:139]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[40:43], v[20:23], a[168:171]\n" \
    "	ds_read_b128 v[104:107], v135 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[40:43], v[24:27], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[40:43], v[28:31], a[232:235]\n" \
    "	ds_read_b128 v[108:111], v135 offset:6144\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[44:47], v[0:3], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[44:47], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[112:115], v135 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[44:47], v[8:11], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[44:47], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[116:119], v135 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[44:47], v[16:19], a[140:143]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[44:47], v[20:23], a[172:175]\n" \
    "	ds_read_b128 v[120:123], v135 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[44:47], v[24:27], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[44:47], v[28:31], a[236:239]\n" \
    "	ds_read_b128 v[124:127], v135 offset:14336\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[48:51], v[0:3], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[48:51], v[4:7], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[48:51], v[8:11], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[48:51], v[12:15], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[48:51], v[16:19], a[144:147]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[48:51], v[20:23], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[48:51], v[24:27], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[48:51], v[28:31], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[52:55], v[0:3], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[52:55], v[4:7], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[52:55], v[8:11], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[52:55], v[12:15], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[52:55], v[16:19], a[148:151]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[52:55], v[20:23], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[52:55], v[24:27], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[52:55], v[28:31], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[56:59], v[0:3], a[24:27]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[56:59], v[4:7], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[56:59], v[8:11], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[56:59], v[12:15], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[56:59], v[16:19], a[152:155]\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[56:59], v[20:23], a[184:187]\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[56:59], v[24:27], a[216:219]\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[56:59], v[28:31], a[248:251]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[60:63], v[0:3], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[60:63], v[4:7], a[60:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[60:63], v[8:11], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[60:63], v[12:15], a[124:127]\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[60:63], v[16:19], a[156:159]\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[60:63], v[20:23], a[188:191]\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[60:63], v[24:27], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[60:63], v[28:31], a[252:255]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[96:99], v[64:67], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[96:99], v[68:71], a[32:35]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[96:99], v[72:75], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[96:99], v[76:79], a[96:99]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[96:99], v[80:83], a[128:131]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[96:99], v[84:87], a[160:163]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[96:99], v[88:91], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[96:99], v[92:95], a[224:227]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[100:103], v[64:67], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[100:103], v[68:71], a[36:39]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[100:103], v[72:75], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[100:103], v[76:79], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[100:103], v[80:83], a[132:135]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[100:103], v[84:87], a[164:167]\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[100:103], v[88:91], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[100:103], v[92:95], a[228:231]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[104:107], v[64:67], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[104:107], v[68:71], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[104:107], v[72:75], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[104:107], v[76:79], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[104:107], v[80:83], a[136:139]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[104:107], v[84:87], a[168:171]\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[104:107], v[88:91], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[104:107], v[92:95], a[232:235]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[108:111], v[64:67], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[108:111], v[68:71], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[108:111], v[72:75], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[108:111], v[76:79], a[108:111]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[108:111], v[80:83], a[140:143]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[108:111], v[84:87], a[172:175]\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[108:111], v[88:91], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[108:111], v[92:95], a[236:239]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[112:115], v[64:67], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[112:115], v[68:71], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[112:115], v[72:75], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[112:115], v[76:79], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[112:115], v[80:83], a[144:147]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[112:115], v[84:87], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[112:115], v[88:91], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[112:115], v[92:95], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(2)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[116:119], v[64:67], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[116:119], v[68:71], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[116:119], v[72:75], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[116:119], v[76:79], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[116:119], v[80:83], a[148:151]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[116:119], v[84:87], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[116:119], v[88:91], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[116:119], v[92:95], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(1)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[120:123], v[64:67], a[24:27]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[120:123], v[68:71], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[120:123], v[72:75], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[120:123], v[76:79], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[120:123], v[80:83], a[152:155]\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[120:123], v[84:87], a[184:187]\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[120:123], v[88:91], a[216:219]\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[120:123], v[92:95], a[248:251]\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[124:127], v[64:67], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[124:127], v[68:71], a[60:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[124:127], v[72:75], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[124:127], v[76:79], a[124:127]\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[124:127], v[80:83], a[156:159]\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[124:127], v[84:87], a[188:191]\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[124:127], v[88:91], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[124:127], v[92:95], a[252:255]\n" \
    "	s_branch DONE_%=\n" \
    "LAST1_%=:\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[32:35], v[0:3], a[0:3]\n" \
    "	s_add_u32 m0, s61, 65536\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v136, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[32:35], v[4:7], a[32:35]\n" \
    "	ds_read_b128 v[96:99], v133 offset:0\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[32:35], v[8:11], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[32:35], v[12:15], a[96:99]\n" \
    "	ds_read_b128 v[64:67], v129 offset:0\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[32:35], v[16:19], a[128:131]\n" \
    "	s_add_u32 m0, s61, 66560\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v137, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[32:35], v[20:23], a[160:163]\n" \
    "	ds_read_b128 v[68:71], v129 offset:2048\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[32:35], v[24:27], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[32:35], v[28:31], a[224:227]\n" \
    "	ds_read_b128 v[72:75], v129 offset:4096\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[36:39], v[0:3], a[4:7]\n" \
    "	s_add_u32 m0, s61, 67584\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v138, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[36:39], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[76:79], v129 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[36:39], v[8:11], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[36:39], v[12:15], a[100:103]\n" \
    "	ds_read_b128 v[80:83], v129 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[36:39], v[16:19], a[132:135]\n" \
    "	s_add_u32 m0, s61, 68608\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v139, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[36:39], v[20:23], a[164:167]\n" \
    "	ds_read_b128 v[84:87], v129 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[36:39], v[24:27], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[36:39], v[28:31], a[228:231]\n" \
    "	ds_read_b128 v[88:91], v129 offset:12288\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[40:43], v[0:3], a[8:11]\n" \
    "	s_add_u32 m0, s61, 69632\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v140, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[40:43], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[92:95], v129 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[40:43], v[8:11], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[40:43], v[12:15], a[104:107]\n" \
    "	ds_read_b128 v[100:103], v133 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[40:43], v[16:19], a[136:139]\n" \
    "	s_add_u32 m0, s61, 70656\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v141, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[40:43], v[20:23], a[168:171]\n" \
    "	ds_read_b128 v[104:107], v133 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[40:43], v[24:27], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[40:43], v[28:31], a[232:235]\n" \
    "	ds_read_b128 v[108:111], v133 offset:6144\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[44:47], v[0:3], a[12:15]\n" \
    "	s_add_u32 m0, s61, 71680\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v142, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[44:47], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[112:115], v133 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[44:47], v[8:11], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[44:47], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[116:119], v133 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[44:47], v[16:19], a[140:143]\n" \
    "	s_add_u32 m0, s61, 72704\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v143, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[44:47], v[20:23], a[172:175]\n" \
    "	ds_read_b128 v[120:123], v133 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[44:47], v[24:27], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[44:47], v[28:31], a[236:239]\n" \
    "	ds_read_b128 v[124:127], v133 offset:14336\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[48:51], v[0:3], a[16:19]\n" \
    "	s_add_u32 m0, s69, 98304\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v144, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[48:51], v[4:7], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[48:51], v[8:11], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[48:51], v[12:15], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[48:51], v[16:19], a[144:147]\n" \
    "	s_add_u32 m0, s69, 99328\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v145, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[48:51], v[20:23], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[48:51], v[24:27], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[48:51], v[28:31], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[52:55], v[0:3], a[20:23]\n" \
    "	s_add_u32 m0, s69, 100352\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v146, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[52:55], v[4:7], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[52:55], v[8:11], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[52:55], v[12:15], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[52:55], v[16:19], a[148:151]\n" \
    "	s_add_u32 m0, s69, 101376\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v147, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[52:55], v[20:23], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[52:55], v[24:27], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[52:55], v[28:31], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[56:59], v[0:3], a[24:27]\n" \
    "	s_add_u32 m0, s69, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v148, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[56:59], v[4:7], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[56:59], v[8:11], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[56:59], v[12:15], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[56:59], v[16:19], a[152:155]\n" \
    "	s_add_u32 m0, s69, 103424\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v149, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[56:59], v[20:23], a[184:187]\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[56:59], v[24:27], a[216:219]\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[56:59], v[28:31], a[248:251]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[60:63], v[0:3], a[28:31]\n" \
    "	s_add_u32 m0, s69, 104448\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v150, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[60:63], v[4:7], a[60:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[60:63], v[8:11], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[60:63], v[12:15], a[124:127]\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[60:63], v[16:19], a[156:159]\n" \
    "	s_add_u32 m0, s69, 105472\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v151, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[60:63], v[20:23], a[188:191]\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[60:63], v[24:27], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[60:63], v[28:31], a[252:255]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[96:99], v[64:67], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[96:99], v[68:71], a[32:35]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[96:99], v[72:75], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[96:99], v[76:79], a[96:99]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[96:99], v[80:83], a[128:131]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[96:99], v[84:87], a[160:163]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[96:99], v[88:91], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[96:99], v[92:95], a[224:227]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[100:103], v[64:67], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[100:103], v[68:71], a[36:39]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[100:103], v[72:75], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[100:103], v[76:79], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[100:103], v[80:83], a[132:135]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[100:103], v[84:87], a[164:167]\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[100:103], v[88:91], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[100:103], v[92:95], a[228:231]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[104:107], v[64:67], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[104:107], v[68:71], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[104:107], v[72:75], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[104:107], v[76:79], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[104:107], v[80:83], a[136:139]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[104:107], v[84:87], a[168:171]\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[104:107], v[88:91], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[104:107], v[92:95], a[232:235]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[108:111], v[64:67], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[108:111], v[68:71], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[108:111], v[72:75], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[108:111], v[76:79], a[108:111]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[108:111], v[80:83], a[140:143]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[108:111], v[84:87], a[172:175]\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[108:111], v[88:91], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[108:111], v[92:95], a[236:239]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[112:115], v[64:67], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[112:115], v[68:71], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[112:115], v[72:75], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[112:115], v[76:79], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[112:115], v[80:83], a[144:147]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[112:115], v[84:87], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[112:115], v[88:91], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[112:115], v[92:95], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(2)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[116:119], v[64:67], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[116:119], v[68:71], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[116:119], v[72:75], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[116:119], v[76:79], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[116:119], v[80:83], a[148:151]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[116:119], v[84:87], a[180:183]\n" \
    "	s_waitcnt vmcnt(0)\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	s_barrier\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[116:119], v[88:91], a[212:215]\n" \
    "	ds_read_b128 v[32:35], v134 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[116:119], v[92:95], a[244:247]\n" \
    "	ds_read_b128 v[0:3], v130 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[120:123], v[64:67], a[24:27]\n" \
    "	ds_read_b128 v[4:7], v130 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[120:123], v[68:71], a[56:59]\n" \
    "	ds_read_b128 v[8:11], v130 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[120:123], v[72:75], a[88:91]\n" \
    "	ds_read_b128 v[12:15], v130 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[120:123], v[76:79], a[120:123]\n" \
    "	ds_read_b128 v[16:19], v130 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[120:123], v[80:83], a[152:155]\n" \
    "	ds_read_b128 v[20:23], v130 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[120:123], v[84:87], a[184:187]\n" \
    "	ds_read_b128 v[24:27], v130 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[120:123], v[88:91], a[216:219]\n" \
    "	ds_read_b128 v[28:31], v130 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[120:123], v[92:95], a[248:251]\n" \
    "	ds_read_b128 v[36:39], v134 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[124:127], v[64:67], a[28:31]\n" \
    "	ds_read_b128 v[40:43], v134 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[124:127], v[68:71], a[60:63]\n" \
    "	ds_read_b128 v[44:47], v134 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[124:127], v[72:75], a[92:95]\n" \
    "	ds_read_b128 v[48:51], v134 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[124:127], v[76:79], a[124:127]\n" \
    "	ds_read_b128 v[52:55], v134 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[124:127], v[80:83], a[156:159]\n" \
    "	ds_read_b128 v[56:59], v134 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[124:127], v[84:87], a[188:191]\n" \
    "	ds_read_b128 v[60:63], v134 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[124:127], v[88:91], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[124:127], v[92:95], a[252:255]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[32:35], v[0:3], a[0:3]\n" \
    "	s_add_u32 m0, s61, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v136, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[32:35], v[4:7], a[32:35]\n" \
    "	ds_read_b128 v[96:99], v135 offset:0\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[32:35], v[8:11], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[32:35], v[12:15], a[96:99]\n" \
    "	ds_read_b128 v[64:67], v131 offset:0\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[32:35], v[16:19], a[128:131]\n" \
    "	s_add_u32 m0, s61, 1024\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v137, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[32:35], v[20:23], a[160:163]\n" \
    "	ds_read_b128 v[68:71], v131 offset:2048\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[32:35], v[24:27], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[32:35], v[28:31], a[224:227]\n" \
    "	ds_read_b128 v[72:75], v131 offset:4096\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[36:39], v[0:3], a[4:7]\n" \
    "	s_add_u32 m0, s61, 2048\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v138, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[36:39], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[76:79], v131 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[36:39], v[8:11], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[36:39], v[12:15], a[100:103]\n" \
    "	ds_read_b128 v[80:83], v131 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[36:39], v[16:19], a[132:135]\n" \
    "	s_add_u32 m0, s61, 3072\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v139, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[36:39], v[20:23], a[164:167]\n" \
    "	ds_read_b128 v[84:87], v131 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[36:39], v[24:27], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[36:39], v[28:31], a[228:231]\n" \
    "	ds_read_b128 v[88:91], v131 offset:12288\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[40:43], v[0:3], a[8:11]\n" \
    "	s_add_u32 m0, s61, 4096\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v140, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[40:43], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[92:95], v131 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[40:43], v[8:11], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[40:43], v[12:15], a[104:107]\n" \
    "	ds_read_b128 v[100:103], v135 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[40:43], v[16:19], a[136:139]\n" \
    "	s_add_u32 m0, s61, 5120\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v141, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[40:43], v[20:23], a[168:171]\n" \
    "	ds_read_b128 v[104:107], v135 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[40:43], v[24:27], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[40:43], v[28:31], a[232:235]\n" \
    "	ds_read_b128 v[108:111], v135 offset:6144\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[44:47], v[0:3], a[12:15]\n" \
    "	s_add_u32 m0, s61, 6144\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v142, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[44:47], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[112:115], v135 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[44:47], v[8:11], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[44:47], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[116:119], v135 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[44:47], v[16:19], a[140:143]\n" \
    "	s_add_u32 m0, s61, 7168\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v143, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[44:47], v[20:23], a[172:175]\n" \
    "	ds_read_b128 v[120:123], v135 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[44:47], v[24:27], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[44:47], v[28:31], a[236:239]\n" \
    "	ds_read_b128 v[124:127], v135 offset:14336\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[48:51], v[0:3], a[16:19]\n" \
    "	s_add_u32 m0, s69, 32768\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v144, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[48:51], v[4:7], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[48:51], v[8:11], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[48:51], v[12:15], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[48:51], v[16:19], a[144:147]\n" \
    "	s_add_u32 m0, s69, 33792\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v145, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[48:51], v[20:23], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[48:51], v[24:27], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[48:51], v[28:31], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[52:55], v[0:3], a[20:23]\n" \
    "	s_add_u32 m0, s69, 34816\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v146, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[52:55], v[4:7], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[52:55], v[8:11], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[52:55], v[12:15], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[52:55], v[16:19], a[148:151]\n" \
    "	s_add_u32 m0, s69, 35840\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v147, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[52:55], v[20:23], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[52:55], v[24:27], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[52:55], v[28:31], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[56:59], v[0:3], a[24:27]\n" \
    "	s_add_u32 m0, s69, 36864\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v148, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[56:59], v[4:7], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[56:59], v[8:11], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[56:59], v[12:15], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[56:59], v[16:19], a[152:155]\n" \
    "	s_add_u32 m0, s69, 37888\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v149, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[56:59], v[20:23], a[184:187]\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[56:59], v[24:27], a[216:219]\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[56:59], v[28:31], a[248:251]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[60:63], v[0:3], a[28:31]\n" \
    "	s_add_u32 m0, s69, 38912\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v150, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[60:63], v[4:7], a[60:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[60:63], v[8:11], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[60:63], v[12:15], a[124:127]\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[60:63], v[16:19], a[156:159]\n" \
    "	s_add_u32 m0, s69, 39936\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v151, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[60:63], v[20:23], a[188:191]\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[60:63], v[24:27], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[60:63], v[28:31], a[252:255]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[96:99], v[64:67], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[96:99], v[68:71], a[32:35]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[96:99], v[72:75], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[96:99], v[76:79], a[96:99]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[96:99], v[80:83], a[128:131]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[96:99], v[84:87], a[160:163]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[96:99], v[88:91], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[96:99], v[92:95], a[224:227]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[100:103], v[64:67], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[100:103], v[68:71], a[36:39]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[100:103], v[72:75], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[100:103], v[76:79], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[100:103], v[80:83], a[132:135]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[100:103], v[84:87], a[164:167]\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[100:103], v[88:91], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[100:103], v[92:95], a[228:231]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[104:107], v[64:67], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[104:107], v[68:71], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[104:107], v[72:75], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[104:107], v[76:79], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[104:107], v[80:83], a[136:139]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[104:107], v[84:87], a[168:171]\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[104:107], v[88:91], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[104:107], v[92:95], a[232:235]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[108:111], v[64:67], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[108:111], v[68:71], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[108:111], v[72:75], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[108:111], v[76:79], a[108:111]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[108:111], v[80:83], a[140:143]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[108:111], v[84:87], a[172:175]\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[108:111], v[88:91], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[108:111], v[92:95], a[236:239]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[112:115], v[64:67], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[112:115], v[68:71], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[112:115], v[72:75], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[112:115], v[76:79], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[112:115], v[80:83], a[144:147]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[112:115], v[84:87], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[112:115], v[88:91], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[112:115], v[92:95], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(2)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[116:119], v[64:67], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[116:119], v[68:71], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[116:119], v[72:75], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[116:119], v[76:79], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[116:119], v[80:83], a[148:151]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[116:119], v[84:87], a[180:183]\n" \
    "	s_waitcnt vmcnt(0)\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	s_barrier\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[116:119], v[88:91], a[212:215]\n" \
    "	ds_read_b128 v[32:35], v132 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[116:119], v[92:95], a[244:247]\n" \
    "	ds_read_b128 v[0:3], v128 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[120:123], v[64:67], a[24:27]\n" \
    "	ds_read_b128 v[4:7], v128 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[120:123], v[68:71], a[56:59]\n" \
    "	ds_read_b128 v[8:11], v128 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[120:123], v[72:75], a[88:91]\n" \
    "	ds_read_b128 v[12:15], v128 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[120:123], v[76:79], a[120:123]\n" \
    "	ds_read_b128 v[16:19], v128 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[120:123], v[80:83], a[152:155]\n" \
    "	ds_read_b128 v[20:23], v128 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[120:123], v[84:87], a[184:187]\n" \
    "	ds_read_b128 v[24:27], v128 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[120:123], v[88:91], a[216:219]\n" \
    "	ds_read_b128 v[28:31], v128 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[120:123], v[92:95], a[248:251]\n" \
    "	ds_read_b128 v[36:39], v132 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[124:127], v[64:67], a[28:31]\n" \
    "	ds_read_b128 v[40:43], v132 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[124:127], v[68:71], a[60:63]\n" \
    "	ds_read_b128 v[44:47], v132 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[124:127], v[72:75], a[92:95]\n" \
    "	ds_read_b128 v[48:51], v132 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[124:127], v[76:79], a[124:127]\n" \
    "	ds_read_b128 v[52:55], v132 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[124:127], v[80:83], a[156:159]\n" \
    "	ds_read_b128 v[56:59], v132 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[124:127], v[84:87], a[188:191]\n" \
    "	ds_read_b128 v[60:63], v132 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[124:127], v[88:91], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[124:127], v[92:95], a[252:255]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[32:35], v[0:3], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[32:35], v[4:7], a[32:35]\n" \
    "	ds_read_b128 v[96:99], v133 offset:0\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[32:35], v[8:11], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[32:35], v[12:15], a[96:99]\n" \
    "	ds_read_b128 v[64:67], v129 offset:0\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[32:35], v[16:19], a[128:131]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[32:35], v[20:23], a[160:163]\n" \
    "	ds_read_b128 v[68:71], v129 offset:2048\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[32:35], v[24:27], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[32:35], v[28:31], a[224:227]\n" \
    "	ds_read_b128 v[72:75], v129 offset:4096\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[36:39], v[0:3], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[36:39], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[76:79], v129 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[36:39], v[8:11], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[36:39], v[12:15], a[100:103]\n" \
    "	ds_read_b128 v[80:83], v129 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[36:39], v[16:19], a[132:135]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[36:39], v[20:23], a[164:167]\n" \
    "	ds_read_b128 v[84:87], v129 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[36:39], v[24:27], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[36:39], v[28:31], a[228:231]\n" \
    "	ds_read_b128 v[88:91], v129 offset:12288\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[40:43], v[0:3], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[40:43], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[92:95], v129 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[40:43], v[8:11], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[40:43], v[12:15], a[104:107]\n" \
    "	ds_read_b128 v[100:103], v133 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[40:43], v[16:19], a[136:139]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[40:43], v[20:23], a[168:171]\n" \
    "	ds_read_b128 v[104:107], v133 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[40:43], v[24:27], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[40:43], v[28:31], a[232:235]\n" \
    "	ds_read_b128 v[108:111], v133 offset:6144\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[44:47], v[0:3], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[44:47], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[112:115], v133 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[44:47], v[8:11], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[44:47], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[116:119], v133 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[44:47], v[16:19], a[140:143]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[44:47], v[20:23], a[172:175]\n" \
    "	ds_read_b128 v[120:123], v133 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[44:47], v[24:27], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[44:47], v[28:31], a[236:239]\n" \
    "	ds_read_b128 v[124:127], v133 offset:14336\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[48:51], v[0:3], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[48:51], v[4:7], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[48:51], v[8:11], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[48:51], v[12:15], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[48:51], v[16:19], a[144:147]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[48:51], v[20:23], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[48:51], v[24:27], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[48:51], v[28:31], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[52:55], v[0:3], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[52:55], v[4:7], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[52:55], v[8:11], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[52:55], v[12:15], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[52:55], v[16:19], a[148:151]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[52:55], v[20:23], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[52:55], v[24:27], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[52:55], v[28:31], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[56:59], v[0:3], a[24:27]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[56:59], v[4:7], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[56:59], v[8:11], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[56:59], v[12:15], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[56:59], v[16:19], a[152:155]\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[56:59], v[20:23], a[184:187]\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[56:59], v[24:27], a[216:219]\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[56:59], v[28:31], a[248:251]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[60:63], v[0:3], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[60:63], v[4:7], a[60:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[60:63], v[8:11], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[60:63], v[12:15], a[124:127]\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[60:63], v[16:19], a[156:159]\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[60:63], v[20:23], a[188:191]\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[60:63], v[24:27], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[60:63], v[28:31], a[252:255]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[96:99], v[64:67], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[96:99], v[68:71], a[32:35]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[96:99], v[72:75], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[96:99], v[76:79], a[96:99]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[96:99], v[80:83], a[128:131]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[96:99], v[84:87], a[160:163]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[96:99], v[88:91], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[96:99], v[92:95], a[224:227]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[100:103], v[64:67], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[100:103], v[68:71], a[36:39]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[100:103], v[72:75], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[100:103], v[76:79], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[100:103], v[80:83], a[132:135]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[100:103], v[84:87], a[164:167]\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[100:103], v[88:91], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[100:103], v[92:95], a[228:231]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[104:107], v[64:67], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[104:107], v[68:71], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[104:107], v[72:75], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[104:107], v[76:79], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[104:107], v[80:83], a[136:139]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[104:107], v[84:87], a[168:171]\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[104:107], v[88:91], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[104:107], v[92:95], a[232:235]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[108:111], v[64:67], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[108:111], v[68:71], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[108:111], v[72:75], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[108:111], v[76:79], a[108:111]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[108:111], v[80:83], a[140:143]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[108:111], v[84:87], a[172:175]\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[108:111], v[88:91], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[108:111], v[92:95], a[236:239]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[112:115], v[64:67], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[112:115], v[68:71], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[112:115], v[72:75], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[112:115], v[76:79], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[112:115], v[80:83], a[144:147]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[112:115], v[84:87], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[112:115], v[88:91], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[112:115], v[92:95], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(2)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[116:119], v[64:67], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[116:119], v[68:71], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[116:119], v[72:75], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[116:119], v[76:79], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[116:119], v[80:83], a[148:151]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[116:119], v[84:87], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[116:119], v[88:91], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[116:119], v[92:95], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(1)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[120:123], v[64:67], a[24:27]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[120:123], v[68:71], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[120:123], v[72:75], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[120:123], v[76:79], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[120:123], v[80:83], a[152:155]\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[120:123], v[84:87], a[184:187]\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[120:123], v[88:91], a[216:219]\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[120:123], v[92:95], a[248:251]\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[124:127], v[64:67], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[124:127], v[68:71], a[60:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[124:127], v[72:75], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[124:127], v[76:79], a[124:127]\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[124:127], v[80:83], a[156:159]\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[124:127], v[84:87], a[188:191]\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[124:127], v[88:91], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[124:127], v[92:95], a[252:255]\n" \
    "DONE_%=:\n" \
    "	s_nop 15\n" \
    "	s_barrier\n" \
    "	s_mov_b32 m0, s66\n" \
      : /* accumulators stay in AGPRs */ \
      : [ap] "s"(ap), [wp] "s"(wp), [rsa] "s"(rsa), [rsw] "s"(rsw), [ra] "s"(ra), [rw] "s"(rw), [trips] "s"(trips), [rem] "s"(rem), [lds] "s"(lds), [wave] "s"(wave), [zero] "s"(zero) \
      : "memory", "vcc", "scc", "v0", "v1", "v2", "v3", "v4", "v5", "v6", "v7", "v8", "v9", "v10", "v11", "v12", "v13", "v14", "v15", "v16", "v17", "v18", "v19", "v20", "v21", "v22", "v23", "v24", "v25", "v26", "v27", "v28", "v29", "v30", "v31", "v32", "v33", "v34", "v35", "v36", "v37", "v38", "v39", "v40", "v41", "v42", "v43", "v44", "v45", "v46", "v47", "v48", "v49", "v50", "v51", "v52", "v53", "v54", "v55", "v56", "v57", "v58", "v59", "v60", "v61", "v62", "v63", "v64", "v65", "v66", "v67", "v68", "v69", "v70", "v71", "v72", "v73", "v74", "v75", "v76", "v77", "v78", "v79", "v80", "v81", "v82", "v83", "v84", "v85", "v86", "v87", "v88", "v89", "v90", "v91", "v92", "v93", "v94", "v95", "v96", "v97", "v98", "v99", "v100", "v101", "v102", "v103", "v104", "v105", "v106", "v107", "v108", "v109", "v110", "v111", "v112", "v113", "v114", "v115", "v116", "v117", "v118", "v119", "v120", "v121", "v122", "v123", "v124", "v125", "v126", "v127", "v128", "v129", "v130", "v131", "v132", "v133", "v134", "v135", "v136", "v137", "v138", "v139", "v140", "v141", "v142", "v143", "v144", "v145", "v146", "v147", "v148", "v149", "v150", "v151", "v152", "v153", "v154", "v155", "v156", "v157", "v158", "v159", "v160", "a0", "a1", "a2", "a3", "a4", "a5", "a6", "a7", "a8", "a9", "a10", "a11", "a12", "a13", "a14", "a15", "a16", "a17", "a18", "a19", "a20", "a21", "a22", "a23", "a24", "a25", "a26", "a27", "a28", "a29", "a30", "a31", "a32", "a33", "a34", "a35", "a36", "a37", "a38", "a39", "a40", "a41", "a42", "a43", "a44", "a45", "a46", "a47", "a48", "a49", "a50", "a51", "a52", "a53", "a54", "a55", "a56", "a57", "a58", "a59", "a60", "a61", "a62", "a63", "a64", "a65", "a66", "a67", "a68", "a69", "a70", "a71", "a72", "a73", "a74", "a75", "a76", "a77", "a78", "a79", "a80", "a81", "a82", "a83", "a84", "a85", "a86", "a87", "a88", "a89", "a90", "a91", "a92", "a93", "a94", "a95", "a96", "a97", "a98", "a99", "a100", "a101", "a102", "a103", "a104", "a105", "a106", "a107", "a108", "a109", "a110", "a111", "a112", "a113", "a114", "a115", "a116", "a117", "a118", "a119", "a120", "a121", "a122", "a123", "a124", "a125", "a126", "a127", "a128", "a129", "a130", "a131", "a132", "a133", "a134", "a135", "a136", "a137", "a138", "a139", "a140", "a141", "a142", "a143", "a144", "a145", "a146", "a147", "a148", "a149", "a150", "a151", "a152", "a153", "a154", "a155", "a156", "a157", "a158", "a159", "a160", "a161", "a162", "a163", "a164", "a165", "a166", "a167", "a168", "a169", "a170", "a171", "a172", "a173", "a174", "a175", "a176", "a177", "a178", "a179", "a180", "a181", "a182", "a183", "a184", "a185", "a186", "a187", "a188", "a189", "a190", "a191", "a192", "a193", "a194", "a195", "a196", "a197", "a198", "a199", "a200", "a201", "a202", "a203", "a204", "a205", "a206", "a207", "a208", "a209", "a210", "a211", "a212", "a213", "a214", "a215", "a216", "a217", "a218", "a219", "a220", "a221", "a222", "a223", "a224", "a225", "a226", "a227", "a228", "a229", "a230", "a231", "a232", "a233", "a234", "a235", "a236", "a237", "a238", "a239", "a240", "a241", "a242", "a243", "a244", "a245", "a246", "a247", "a248", "a249", "a250", "a251", "a252", "a253", "a254", "a255", "s60", "s61", "s62", "s63", "s64", "s65", "s66", "s67", "s68", "s69")

#define GEMM_I8_PERIOD_144 3  // stages per trip, and the fewest the loop takes
#define GEMM_I8_ASM_144(ap, wp, rsa, rsw, ra, rw, trips, rem, lds, wave, zero) \
  asm volatile( \
    "	s_mov_b32 s66, m0\n" \
    "	v_mbcnt_lo_u32_b32 v129, -1, 0\n" \
    "	v_mbcnt_hi_u32_b32 v129, -1, v129\n" \
    "	v_and_b32_e32 v130, 15, v129\n" \
    "	v_lshrrev_b32_e32 v131, 4, v129\n" \
    "	v_bfe_u32 v132, v129, 1, 3\n" \
    "	v_lshrrev_b32_e32 v133, 3, v129\n" \
    "	v_and_b32_e32 v134, 7, v129\n" \
    "	s_mul_i32 s67, %[wave], 64\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 0\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v135, s68, v131\n" \
    "	v_xor_b32_e32 v135, v135, v134\n" \
    "	v_lshlrev_b32_e32 v135, 4, v135\n" \
    "	v_add_u32_e32 v136, 0, v133\n" \
    "	v_add_u32_e32 v136, s67, v136\n" \
    "	v_min_u32_e32 v136, %[ra], v136\n" \
    "	v_mad_u32_u24 v116, v136, %[rsa], v135\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 4\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v135, s68, v131\n" \
    "	v_xor_b32_e32 v135, v135, v134\n" \
    "	v_lshlrev_b32_e32 v135, 4, v135\n" \
    "	v_add_u32_e32 v136, 8, v133\n" \
    "	v_add_u32_e32 v136, s67, v136\n" \
    "	v_min_u32_e32 v136, %[ra], v136\n" \
    "	v_mad_u32_u24 v117, v136, %[rsa], v135\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 8\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v135, s68, v131\n" \
    "	v_xor_b32_e32 v135, v135, v134\n" \
    "	v_lshlrev_b32_e32 v135, 4, v135\n" \
    "	v_add_u32_e32 v136, 16, v133\n" \
    "	v_add_u32_e32 v136, s67, v136\n" \
    "	v_min_u32_e32 v136, %[ra], v136\n" \
    "	v_mad_u32_u24 v118, v136, %[rsa], v135\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 12\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v135, s68, v131\n" \
    "	v_xor_b32_e32 v135, v135, v134\n" \
    "	v_lshlrev_b32_e32 v135, 4, v135\n" \
    "	v_add_u32_e32 v136, 24, v133\n" \
    "	v_add_u32_e32 v136, s67, v136\n" \
    "	v_min_u32_e32 v136, %[ra], v136\n" \
    "	v_mad_u32_u24 v119, v136, %[rsa], v135\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 16\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v135, s68, v131\n" \
    "	v_xor_b32_e32 v135, v135, v134\n" \
    "	v_lshlrev_b32_e32 v135, 4, v135\n" \
    "	v_add_u32_e32 v136, 32, v133\n" \
    "	v_add_u32_e32 v136, s67, v136\n" \
    "	v_min_u32_e32 v136, %[ra], v136\n" \
    "	v_mad_u32_u24 v120, v136, %[rsa], v135\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 20\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v135, s68, v131\n" \
    "	v_xor_b32_e32 v135, v135, v134\n" \
    "	v_lshlrev_b32_e32 v135, 4, v135\n" \
    "	v_add_u32_e32 v136, 40, v133\n" \
    "	v_add_u32_e32 v136, s67, v136\n" \
    "	v_min_u32_e32 v136, %[ra], v136\n" \
    "	v_mad_u32_u24 v121, v136, %[rsa], v135\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 24\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v135, s68, v131\n" \
    "	v_xor_b32_e32 v135, v135, v134\n" \
    "	v_lshlrev_b32_e32 v135, 4, v135\n" \
    "	v_add_u32_e32 v136, 48, v133\n" \
    "	v_add_u32_e32 v136, s67, v136\n" \
    "	v_min_u32_e32 v136, %[ra], v136\n" \
    "	v_mad_u32_u24 v122, v136, %[rsa], v135\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 28\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v135, s68, v131\n" \
    "	v_xor_b32_e32 v135, v135, v134\n" \
    "	v_lshlrev_b32_e32 v135, 4, v135\n" \
    "	v_add_u32_e32 v136, 56, v133\n" \
    "	v_add_u32_e32 v136, s67, v136\n" \
    "	v_min_u32_e32 v136, %[ra], v136\n" \
    "	v_mad_u32_u24 v123, v136, %[rsa], v135\n" \
    "	s_mul_i32 s68, %[wave], 5\n" \
    "	s_add_u32 s68, s68, 0\n" \
    "	s_sub_u32 s67, s68, 18\n" \
    "	s_cmp_ge_u32 s68, 18\n" \
    "	s_cselect_b32 s68, s67, s68\n" \
    "	s_lshl_b32 s67, s68, 10\n" \
    "	s_add_u32 s70, %[lds], s67\n" \
    "	s_add_u32 s70, s70, 32768\n" \
    "	s_lshl_b32 s67, s68, 3\n" \
    "	s_lshl_b32 s68, s68, 2\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v135, s68, v131\n" \
    "	v_xor_b32_e32 v135, v135, v134\n" \
    "	v_lshlrev_b32_e32 v135, 4, v135\n" \
    "	v_add_u32_e32 v136, s67, v133\n" \
    "	v_min_u32_e32 v136, %[rw], v136\n" \
    "	v_mad_u32_u24 v124, v136, %[rsw], v135\n" \
    "	s_mul_i32 s68, %[wave], 5\n" \
    "	s_add_u32 s68, s68, 1\n" \
    "	s_sub_u32 s67, s68, 18\n" \
    "	s_cmp_ge_u32 s68, 18\n" \
    "	s_cselect_b32 s68, s67, s68\n" \
    "	s_lshl_b32 s67, s68, 10\n" \
    "	s_add_u32 s71, %[lds], s67\n" \
    "	s_add_u32 s71, s71, 32768\n" \
    "	s_lshl_b32 s67, s68, 3\n" \
    "	s_lshl_b32 s68, s68, 2\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v135, s68, v131\n" \
    "	v_xor_b32_e32 v135, v135, v134\n" \
    "	v_lshlrev_b32_e32 v135, 4, v135\n" \
    "	v_add_u32_e32 v136, s67, v133\n" \
    "	v_min_u32_e32 v136, %[rw], v136\n" \
    "	v_mad_u32_u24 v125, v136, %[rsw], v135\n" \
    "	s_mul_i32 s68, %[wave], 5\n" \
    "	s_add_u32 s68, s68, 2\n" \
    "	s_sub_u32 s67, s68, 18\n" \
    "	s_cmp_ge_u32 s68, 18\n" \
    "	s_cselect_b32 s68, s67, s68\n" \
    "	s_lshl_b32 s67, s68, 10\n" \
    "	s_add_u32 s72, %[lds], s67\n" \
    "	s_add_u32 s72, s72, 32768\n" \
    "	s_lshl_b32 s67, s68, 3\n" \
    "	s_lshl_b32 s68, s68, 2\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v135, s68, v131\n" \
    "	v_xor_b32_e32 v135, v135, v134\n" \
    "	v_lshlrev_b32_e32 v135, 4, v135\n" \
    "	v_add_u32_e32 v136, s67, v133\n" \
    "	v_min_u32_e32 v136, %[rw], v136\n" \
    "	v_mad_u32_u24 v126, v136, %[rsw], v135\n" \
    "	s_mul_i32 s68, %[wave], 5\n" \
    "	s_add_u32 s68, s68, 3\n" \
    "	s_sub_u32 s67, s68, 18\n" \
    "	s_cmp_ge_u32 s68, 18\n" \
    "	s_cselect_b32 s68, s67, s68\n" \
    "	s_lshl_b32 s67, s68, 10\n" \
    "	s_add_u32 s73, %[lds], s67\n" \
    "	s_add_u32 s73, s73, 32768\n" \
    "	s_lshl_b32 s67, s68, 3\n" \
    "	s_lshl_b32 s68, s68, 2\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v135, s68, v131\n" \
    "	v_xor_b32_e32 v135, v135, v134\n" \
    "	v_lshlrev_b32_e32 v135, 4, v135\n" \
    "	v_add_u32_e32 v136, s67, v133\n" \
    "	v_min_u32_e32 v136, %[rw], v136\n" \
    "	v_mad_u32_u24 v127, v136, %[rsw], v135\n" \
    "	s_mul_i32 s68, %[wave], 5\n" \
    "	s_add_u32 s68, s68, 4\n" \
    "	s_sub_u32 s67, s68, 18\n" \
    "	s_cmp_ge_u32 s68, 18\n" \
    "	s_cselect_b32 s68, s67, s68\n" \
    "	s_lshl_b32 s67, s68, 10\n" \
    "	s_add_u32 s74, %[lds], s67\n" \
    "	s_add_u32 s74, s74, 32768\n" \
    "	s_lshl_b32 s67, s68, 3\n" \
    "	s_lshl_b32 s68, s68, 2\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v135, s68, v131\n" \
    "	v_xor_b32_e32 v135, v135, v134\n" \
    "	v_lshlrev_b32_e32 v135, 4, v135\n" \
    "	v_add_u32_e32 v136, s67, v133\n" \
    "	v_min_u32_e32 v136, %[rw], v136\n" \
    "	v_mad_u32_u24 v128, v136, %[rsw], v135\n" \
    "	s_lshl_b32 s67, %[wave], 13\n" \
    "	s_add_u32 s61, %[lds], s67\n" \
    "	s_mul_i32 s67, %[wave], 5120\n" \
    "	s_add_u32 s69, %[lds], s67\n" \
    "	s_mov_b64 s[62:63], %[ap]\n" \
    "	s_mov_b64 s[64:65], %[wp]\n" \
    "	s_add_u32 m0, s61, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v116, s[62:63]\n" \
    "	s_add_u32 m0, s61, 1024\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v117, s[62:63]\n" \
    "	s_add_u32 m0, s61, 2048\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v118, s[62:63]\n" \
    "	s_add_u32 m0, s61, 3072\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v119, s[62:63]\n" \
    "	s_add_u32 m0, s61, 4096\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v120, s[62:63]\n" \
    "	s_add_u32 m0, s61, 5120\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v121, s[62:63]\n" \
    "	s_add_u32 m0, s61, 6144\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v122, s[62:63]\n" \
    "	s_add_u32 m0, s61, 7168\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v123, s[62:63]\n" \
    "	s_add_u32 m0, s70, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v124, s[64:65]\n" \
    "	s_add_u32 m0, s71, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v125, s[64:65]\n" \
    "	s_add_u32 m0, s72, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v126, s[64:65]\n" \
    "	s_add_u32 m0, s73, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v127, s[64:65]\n" \
    "	s_add_u32 m0, s74, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v128, s[64:65]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_add_u32 m0, s61, 51200\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v116, s[62:63]\n" \
    "	s_add_u32 m0, s61, 52224\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v117, s[62:63]\n" \
    "	s_add_u32 m0, s61, 53248\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v118, s[62:63]\n" \
    "	s_add_u32 m0, s61, 54272\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v119, s[62:63]\n" \
    "	s_add_u32 m0, s61, 55296\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v120, s[62:63]\n" \
    "	s_add_u32 m0, s61, 56320\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v121, s[62:63]\n" \
    "	s_add_u32 m0, s61, 57344\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v122, s[62:63]\n" \
    "	s_add_u32 m0, s61, 58368\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v123, s[62:63]\n" \
    "	s_add_u32 m0, s70, 51200\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v124, s[64:65]\n" \
    "	s_add_u32 m0, s71, 51200\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v125, s[64:65]\n" \
    "	s_add_u32 m0, s72, 51200\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v126, s[64:65]\n" \
    "	s_add_u32 m0, s73, 51200\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v127, s[64:65]\n" \
    "	s_add_u32 m0, s74, 51200\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v128, s[64:65]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_lshl_b32 s67, %[wave], 13\n" \
    "	s_mov_b32 s68, 0\n" \
    "	v_lshlrev_b32_e32 v133, 7, v130\n" \
    "	v_add_u32_e32 v133, %[lds], v133\n" \
    "	v_add_u32_e32 v134, 0, v131\n" \
    "	v_xor_b32_e32 v134, v134, v132\n" \
    "	v_lshl_add_u32 v134, v134, 4, v133\n" \
    "	v_add_u32_e32 v104, s67, v134\n" \
    "	v_add_u32_e32 v110, s68, v134\n" \
    "	v_add_u32_e32 v110, 32768, v110\n" \
    "	v_add_u32_e32 v134, 4, v131\n" \
    "	v_xor_b32_e32 v134, v134, v132\n" \
    "	v_lshl_add_u32 v134, v134, 4, v133\n" \
    "	v_add_u32_e32 v105, s67, v134\n" \
    "	v_add_u32_e32 v111, s68, v134\n" \
    "	v_add_u32_e32 v111, 32768, v111\n" \
    "	v_add_u32_e32 v134, 0, v131\n" \
    "	v_xor_b32_e32 v134, v134, v132\n" \
    "	v_lshl_add_u32 v134, v134, 4, v133\n" \
    "	v_add_u32_e32 v106, s67, v134\n" \
    "	v_add_u32_e32 v112, s68, v134\n" \
    "	v_add_u32_e32 v106, 51200, v106\n" \
    "	v_add_u32_e32 v112, 83968, v112\n" \
    "	v_add_u32_e32 v134, 4, v131\n" \
    "	v_xor_b32_e32 v134, v134, v132\n" \
    "	v_lshl_add_u32 v134, v134, 4, v133\n" \
    "	v_add_u32_e32 v107, s67, v134\n" \
    "	v_add_u32_e32 v113, s68, v134\n" \
    "	v_add_u32_e32 v107, 51200, v107\n" \
    "	v_add_u32_e32 v113, 83968, v113\n" \
    "	v_add_u32_e32 v134, 0, v131\n" \
    "	v_xor_b32_e32 v134, v134, v132\n" \
    "	v_lshl_add_u32 v134, v134, 4, v133\n" \
    "	v_add_u32_e32 v108, s67, v134\n" \
    "	v_add_u32_e32 v114, s68, v134\n" \
    "	v_add_u32_e32 v108, 102400, v108\n" \
    "	v_add_u32_e32 v114, 135168, v114\n" \
    "	v_add_u32_e32 v134, 4, v131\n" \
    "	v_xor_b32_e32 v134, v134, v132\n" \
    "	v_lshl_add_u32 v134, v134, 4, v133\n" \
    "	v_add_u32_e32 v109, s67, v134\n" \
    "	v_add_u32_e32 v115, s68, v134\n" \
    "	v_add_u32_e32 v109, 102400, v109\n" \
    "	v_add_u32_e32 v115, 135168, v115\n" \
    "	s_cmp_eq_u32 %[zero], 0\n" \
    "	s_cbranch_scc1 KEEP_%=\n" \
    "	v_accvgpr_write_b32 a0, 0\n" \
    "	v_accvgpr_write_b32 a1, 0\n" \
    "	v_accvgpr_write_b32 a2, 0\n" \
    "	v_accvgpr_write_b32 a3, 0\n" \
    "	v_accvgpr_write_b32 a4, 0\n" \
    "	v_accvgpr_write_b32 a5, 0\n" \
    "	v_accvgpr_write_b32 a6, 0\n" \
    "	v_accvgpr_write_b32 a7, 0\n" \
    "	v_accvgpr_write_b32 a8, 0\n" \
    "	v_accvgpr_write_b32 a9, 0\n" \
    "	v_accvgpr_write_b32 a10, 0\n" \
    "	v_accvgpr_write_b32 a11, 0\n" \
    "	v_accvgpr_write_b32 a12, 0\n" \
    "	v_accvgpr_write_b32 a13, 0\n" \
    "	v_accvgpr_write_b32 a14, 0\n" \
    "	v_accvgpr_write_b32 a15, 0\n" \
    "	v_accvgpr_write_b32 a16, 0\n" \
    "	v_accvgpr_write_b32 a17, 0\n" \
    "	v_accvgpr_write_b32 a18, 0\n" \
    "	v_accvgpr_write_b32 a19, 0\n" \
    "	v_accvgpr_write_b32 a20, 0\n" \
    "	v_accvgpr_write_b32 a21, 0\n" \
    "	v_accvgpr_write_b32 a22, 0\n" \
    "	v_accvgpr_write_b32 a23, 0\n" \
    "	v_accvgpr_write_b32 a24, 0\n" \
    "	v_accvgpr_write_b32 a25, 0\n" \
    "	v_accvgpr_write_b32 a26, 0\n" \
    "	v_accvgpr_write_b32 a27, 0\n" \
    "	v_accvgpr_write_b32 a28, 0\n" \
    "	v_accvgpr_write_b32 a29, 0\n" \
    "	v_accvgpr_write_b32 a30, 0\n" \
    "	v_accvgpr_write_b32 a31, 0\n" \
    "	v_accvgpr_write_b32 a32, 0\n" \
    "	v_accvgpr_write_b32 a33, 0\n" \
    "	v_accvgpr_write_b32 a34, 0\n" \
    "	v_accvgpr_write_b32 a35, 0\n" \
    "	v_accvgpr_write_b32 a36, 0\n" \
    "	v_accvgpr_write_b32 a37, 0\n" \
    "	v_accvgpr_write_b32 a38, 0\n" \
    "	v_accvgpr_write_b32 a39, 0\n" \
    "	v_accvgpr_write_b32 a40, 0\n" \
    "	v_accvgpr_write_b32 a41, 0\n" \
    "	v_accvgpr_write_b32 a42, 0\n" \
    "	v_accvgpr_write_b32 a43, 0\n" \
    "	v_accvgpr_write_b32 a44, 0\n" \
    "	v_accvgpr_write_b32 a45, 0\n" \
    "	v_accvgpr_write_b32 a46, 0\n" \
    "	v_accvgpr_write_b32 a47, 0\n" \
    "	v_accvgpr_write_b32 a48, 0\n" \
    "	v_accvgpr_write_b32 a49, 0\n" \
    "	v_accvgpr_write_b32 a50, 0\n" \
    "	v_accvgpr_write_b32 a51, 0\n" \
    "	v_accvgpr_write_b32 a52, 0\n" \
    "	v_accvgpr_write_b32 a53, 0\n" \
    "	v_accvgpr_write_b32 a54, 0\n" \
    "	v_accvgpr_write_b32 a55, 0\n" \
    "	v_accvgpr_write_b32 a56, 0\n" \
    "	v_accvgpr_write_b32 a57, 0\n" \
    "	v_accvgpr_write_b32 a58, 0\n" \
    "	v_accvgpr_write_b32 a59, 0\n" \
    "	v_accvgpr_write_b32 a60, 0\n" \
    "	v_accvgpr_write_b32 a61, 0\n" \
    "	v_accvgpr_write_b32 a62, 0\n" \
    "	v_accvgpr_write_b32 a63, 0\n" \
    "	v_accvgpr_write_b32 a64, 0\n" \
    "	v_accvgpr_write_b32 a65, 0\n" \
    "	v_accvgpr_write_b32 a66, 0\n" \
    "	v_accvgpr_write_b32 a67, 0\n" \
    "	v_accvgpr_write_b32 a68, 0\n" \
    "	v_accvgpr_write_b32 a69, 0\n" \
    "	v_accvgpr_write_b32 a70, 0\n" \
    "	v_accvgpr_write_b32 a71, 0\n" \
    "	v_accvgpr_write_b32 a72, 0\n" \
    "	v_accvgpr_write_b32 a73, 0\n" \
    "	v_accvgpr_write_b32 a74, 0\n" \
    "	v_accvgpr_write_b32 a75, 0\n" \
    "	v_accvgpr_write_b32 a76, 0\n" \
    "	v_accvgpr_write_b32 a77, 0\n" \
    "	v_accvgpr_write_b32 a78, 0\n" \
    "	v_accvgpr_write_b32 a79, 0\n" \
    "	v_accvgpr_write_b32 a80, 0\n" \
    "	v_accvgpr_write_b32 a81, 0\n" \
    "	v_accvgpr_write_b32 a82, 0\n" \
    "	v_accvgpr_write_b32 a83, 0\n" \
    "	v_accvgpr_write_b32 a84, 0\n" \
    "	v_accvgpr_write_b32 a85, 0\n" \
    "	v_accvgpr_write_b32 a86, 0\n" \
    "	v_accvgpr_write_b32 a87, 0\n" \
    "	v_accvgpr_write_b32 a88, 0\n" \
    "	v_accvgpr_write_b32 a89, 0\n" \
    "	v_accvgpr_write_b32 a90, 0\n" \
    "	v_accvgpr_write_b32 a91, 0\n" \
    "	v_accvgpr_write_b32 a92, 0\n" \
    "	v_accvgpr_write_b32 a93, 0\n" \
    "	v_accvgpr_write_b32 a94, 0\n" \
    "	v_accvgpr_write_b32 a95, 0\n" \
    "	v_accvgpr_write_b32 a96, 0\n" \
    "	v_accvgpr_write_b32 a97, 0\n" \
    "	v_accvgpr_write_b32 a98, 0\n" \
    "	v_accvgpr_write_b32 a99, 0\n" \
    "	v_accvgpr_write_b32 a100, 0\n" \
    "	v_accvgpr_write_b32 a101, 0\n" \
    "	v_accvgpr_write_b32 a102, 0\n" \
    "	v_accvgpr_write_b32 a103, 0\n" \
    "	v_accvgpr_write_b32 a104, 0\n" \
    "	v_accvgpr_write_b32 a105, 0\n" \
    "	v_accvgpr_write_b32 a106, 0\n" \
    "	v_accvgpr_write_b32 a107, 0\n" \
    "	v_accvgpr_write_b32 a108, 0\n" \
    "	v_accvgpr_write_b32 a109, 0\n" \
    "	v_accvgpr_write_b32 a110, 0\n" \
    "	v_accvgpr_write_b32 a111, 0\n" \
    "	v_accvgpr_write_b32 a112, 0\n" \
    "	v_accvgpr_write_b32 a113, 0\n" \
    "	v_accvgpr_write_b32 a114, 0\n" \
    "	v_accvgpr_write_b32 a115, 0\n" \
    "	v_accvgpr_write_b32 a116, 0\n" \
    "	v_accvgpr_write_b32 a117, 0\n" \
    "	v_accvgpr_write_b32 a118, 0\n" \
    "	v_accvgpr_write_b32 a119, 0\n" \
    "	v_accvgpr_write_b32 a120, 0\n" \
    "	v_accvgpr_write_b32 a121, 0\n" \
    "	v_accvgpr_write_b32 a122, 0\n" \
    "	v_accvgpr_write_b32 a123, 0\n" \
    "	v_accvgpr_write_b32 a124, 0\n" \
    "	v_accvgpr_write_b32 a125, 0\n" \
    "	v_accvgpr_write_b32 a126, 0\n" \
    "	v_accvgpr_write_b32 a127, 0\n" \
    "	v_accvgpr_write_b32 a128, 0\n" \
    "	v_accvgpr_write_b32 a129, 0\n" \
    "	v_accvgpr_write_b32 a130, 0\n" \
    "	v_accvgpr_write_b32 a131, 0\n" \
    "	v_accvgpr_write_b32 a132, 0\n" \
    "	v_accvgpr_write_b32 a133, 0\n" \
    "	v_accvgpr_write_b32 a134, 0\n" \
    "	v_accvgpr_write_b32 a135, 0\n" \
    "	v_accvgpr_write_b32 a136, 0\n" \
    "	v_accvgpr_write_b32 a137, 0\n" \
    "	v_accvgpr_write_b32 a138, 0\n" \
    "	v_accvgpr_write_b32 a139, 0\n" \
    "	v_accvgpr_write_b32 a140, 0\n" \
    "	v_accvgpr_write_b32 a141, 0\n" \
    "	v_accvgpr_write_b32 a142, 0\n" \
    "	v_accvgpr_write_b32 a143, 0\n" \
    "KEEP_%=:\n" \
    "	s_waitcnt vmcnt(13)\n" \
    "	s_barrier\n" \
    "	ds_read_b128 v[16:19], v110 offset:0\n" \
    "	ds_read_b128 v[0:3], v104 offset:0\n" \
    "	ds_read_b128 v[4:7], v104 offset:2048\n" \
    "	ds_read_b128 v[8:11], v104 offset:4096\n" \
    "	ds_read_b128 v[12:15], v104 offset:6144\n" \
    "	ds_read_b128 v[20:23], v110 offset:2048\n" \
    "	ds_read_b128 v[24:27], v110 offset:4096\n" \
    "	ds_read_b128 v[28:31], v110 offset:6144\n" \
    "	ds_read_b128 v[32:35], v110 offset:8192\n" \
    "	ds_read_b128 v[36:39], v110 offset:10240\n" \
    "	ds_read_b128 v[40:43], v110 offset:12288\n" \
    "	ds_read_b128 v[44:47], v110 offset:14336\n" \
    "	ds_read_b128 v[48:51], v110 offset:16384\n" \
    "	s_mov_b32 s60, %[trips]\n" \
    "	s_cmp_eq_u32 s60, 0\n" \
    "	s_cbranch_scc1 LAST_%=\n" \
    "LOOP_%=:\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[16:19], v[0:3], a[0:3]\n" \
    "	s_add_u32 m0, s61, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v116, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[16:19], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[68:71], v111 offset:0\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[16:19], v[8:11], a[72:75]\n" \
    "	s_add_u32 m0, s61, 103424\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v117, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[16:19], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[52:55], v105 offset:0\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[20:23], v[0:3], a[4:7]\n" \
    "	s_add_u32 m0, s61, 104448\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v118, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[20:23], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[56:59], v105 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[20:23], v[8:11], a[76:79]\n" \
    "	s_add_u32 m0, s61, 105472\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v119, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[20:23], v[12:15], a[112:115]\n" \
    "	ds_read_b128 v[60:63], v105 offset:4096\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[24:27], v[0:3], a[8:11]\n" \
    "	s_add_u32 m0, s61, 106496\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v120, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[24:27], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[64:67], v105 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[24:27], v[8:11], a[80:83]\n" \
    "	s_add_u32 m0, s61, 107520\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v121, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[24:27], v[12:15], a[116:119]\n" \
    "	ds_read_b128 v[72:75], v111 offset:2048\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[28:31], v[0:3], a[12:15]\n" \
    "	s_add_u32 m0, s61, 108544\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v122, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[28:31], v[4:7], a[48:51]\n" \
    "	ds_read_b128 v[76:79], v111 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[28:31], v[8:11], a[84:87]\n" \
    "	s_add_u32 m0, s61, 109568\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v123, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[28:31], v[12:15], a[120:123]\n" \
    "	ds_read_b128 v[80:83], v111 offset:6144\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[32:35], v[0:3], a[16:19]\n" \
    "	s_add_u32 m0, s70, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v124, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[32:35], v[4:7], a[52:55]\n" \
    "	ds_read_b128 v[84:87], v111 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[32:35], v[8:11], a[88:91]\n" \
    "	s_add_u32 m0, s71, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v125, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[32:35], v[12:15], a[124:127]\n" \
    "	ds_read_b128 v[88:91], v111 offset:10240\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[36:39], v[0:3], a[20:23]\n" \
    "	s_add_u32 m0, s72, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v126, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[36:39], v[4:7], a[56:59]\n" \
    "	ds_read_b128 v[92:95], v111 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[36:39], v[8:11], a[92:95]\n" \
    "	s_add_u32 m0, s73, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v127, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[36:39], v[12:15], a[128:131]\n" \
    "	ds_read_b128 v[96:99], v111 offset:14336\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[40:43], v[0:3], a[24:27]\n" \
    "	s_add_u32 m0, s74, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v128, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[40:43], v[4:7], a[60:63]\n" \
    "	ds_read_b128 v[100:103], v111 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[40:43], v[8:11], a[96:99]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[40:43], v[12:15], a[132:135]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[44:47], v[0:3], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[44:47], v[4:7], a[64:67]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[44:47], v[8:11], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[44:47], v[12:15], a[136:139]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[48:51], v[0:3], a[32:35]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[48:51], v[4:7], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[48:51], v[8:11], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[48:51], v[12:15], a[140:143]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[68:71], v[52:55], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[68:71], v[56:59], a[36:39]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[68:71], v[60:63], a[72:75]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[68:71], v[64:67], a[108:111]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[72:75], v[52:55], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[72:75], v[56:59], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[72:75], v[60:63], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[72:75], v[64:67], a[112:115]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[76:79], v[52:55], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[76:79], v[56:59], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[76:79], v[60:63], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[76:79], v[64:67], a[116:119]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[80:83], v[52:55], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[80:83], v[56:59], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[80:83], v[60:63], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[80:83], v[64:67], a[120:123]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[84:87], v[52:55], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[84:87], v[56:59], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[84:87], v[60:63], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[84:87], v[64:67], a[124:127]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[88:91], v[52:55], a[20:23]\n" \
    "	s_waitcnt vmcnt(13)\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	s_barrier\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[88:91], v[56:59], a[56:59]\n" \
    "	ds_read_b128 v[16:19], v112 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[88:91], v[60:63], a[92:95]\n" \
    "	ds_read_b128 v[0:3], v106 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[88:91], v[64:67], a[128:131]\n" \
    "	ds_read_b128 v[4:7], v106 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[92:95], v[52:55], a[24:27]\n" \
    "	ds_read_b128 v[8:11], v106 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[92:95], v[56:59], a[60:63]\n" \
    "	ds_read_b128 v[12:15], v106 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[92:95], v[60:63], a[96:99]\n" \
    "	ds_read_b128 v[20:23], v112 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[92:95], v[64:67], a[132:135]\n" \
    "	ds_read_b128 v[24:27], v112 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[96:99], v[52:55], a[28:31]\n" \
    "	ds_read_b128 v[28:31], v112 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[96:99], v[56:59], a[64:67]\n" \
    "	ds_read_b128 v[32:35], v112 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[96:99], v[60:63], a[100:103]\n" \
    "	ds_read_b128 v[36:39], v112 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[96:99], v[64:67], a[136:139]\n" \
    "	ds_read_b128 v[40:43], v112 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[100:103], v[52:55], a[32:35]\n" \
    "	ds_read_b128 v[44:47], v112 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[100:103], v[56:59], a[68:71]\n" \
    "	ds_read_b128 v[48:51], v112 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[100:103], v[60:63], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[100:103], v[64:67], a[140:143]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[16:19], v[0:3], a[0:3]\n" \
    "	s_add_u32 m0, s61, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v116, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[16:19], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[68:71], v113 offset:0\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[16:19], v[8:11], a[72:75]\n" \
    "	s_add_u32 m0, s61, 1024\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v117, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[16:19], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[52:55], v107 offset:0\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[20:23], v[0:3], a[4:7]\n" \
    "	s_add_u32 m0, s61, 2048\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v118, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[20:23], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[56:59], v107 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[20:23], v[8:11], a[76:79]\n" \
    "	s_add_u32 m0, s61, 3072\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v119, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[20:23], v[12:15], a[112:115]\n" \
    "	ds_read_b128 v[60:63], v107 offset:4096\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[24:27], v[0:3], a[8:11]\n" \
    "	s_add_u32 m0, s61, 4096\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v120, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[24:27], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[64:67], v107 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[24:27], v[8:11], a[80:83]\n" \
    "	s_add_u32 m0, s61, 5120\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v121, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[24:27], v[12:15], a[116:119]\n" \
    "	ds_read_b128 v[72:75], v113 offset:2048\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[28:31], v[0:3], a[12:15]\n" \
    "	s_add_u32 m0, s61, 6144\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v122, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[28:31], v[4:7], a[48:51]\n" \
    "	ds_read_b128 v[76:79], v113 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[28:31], v[8:11], a[84:87]\n" \
    "	s_add_u32 m0, s61, 7168\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v123, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[28:31], v[12:15], a[120:123]\n" \
    "	ds_read_b128 v[80:83], v113 offset:6144\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[32:35], v[0:3], a[16:19]\n" \
    "	s_add_u32 m0, s70, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v124, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[32:35], v[4:7], a[52:55]\n" \
    "	ds_read_b128 v[84:87], v113 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[32:35], v[8:11], a[88:91]\n" \
    "	s_add_u32 m0, s71, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v125, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[32:35], v[12:15], a[124:127]\n" \
    "	ds_read_b128 v[88:91], v113 offset:10240\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[36:39], v[0:3], a[20:23]\n" \
    "	s_add_u32 m0, s72, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v126, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[36:39], v[4:7], a[56:59]\n" \
    "	ds_read_b128 v[92:95], v113 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[36:39], v[8:11], a[92:95]\n" \
    "	s_add_u32 m0, s73, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v127, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[36:39], v[12:15], a[128:131]\n" \
    "	ds_read_b128 v[96:99], v113 offset:14336\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[40:43], v[0:3], a[24:27]\n" \
    "	s_add_u32 m0, s74, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v128, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[40:43], v[4:7], a[60:63]\n" \
    "	ds_read_b128 v[100:103], v113 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[40:43], v[8:11], a[96:99]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[40:43], v[12:15], a[132:135]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[44:47], v[0:3], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[44:47], v[4:7], a[64:67]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[44:47], v[8:11], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[44:47], v[12:15], a[136:139]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[48:51], v[0:3], a[32:35]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[48:51], v[4:7], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[48:51], v[8:11], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[48:51], v[12:15], a[140:143]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[68:71], v[52:55], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[68:71], v[56:59], a[36:39]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[68:71], v[60:63], a[72:75]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[68:71], v[64:67], a[108:111]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[72:75], v[52:55], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[72:75], v[56:59], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[72:75], v[60:63], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[72:75], v[64:67], a[112:115]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[76:79], v[52:55], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[76:79], v[56:59], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[76:79], v[60:63], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[76:79], v[64:67], a[116:119]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[80:83], v[52:55], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[80:83], v[56:59], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[80:83], v[60:63], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[80:83], v[64:67], a[120:123]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[84:87], v[52:55], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[84:87], v[56:59], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[84:87], v[60:63], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[84:87], v[64:67], a[124:127]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[88:91], v[52:55], a[20:23]\n" \
    "	s_waitcnt vmcnt(13)\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	s_barrier\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[88:91], v[56:59], a[56:59]\n" \
    "	ds_read_b128 v[16:19], v114 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[88:91], v[60:63], a[92:95]\n" \
    "	ds_read_b128 v[0:3], v108 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[88:91], v[64:67], a[128:131]\n" \
    "	ds_read_b128 v[4:7], v108 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[92:95], v[52:55], a[24:27]\n" \
    "	ds_read_b128 v[8:11], v108 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[92:95], v[56:59], a[60:63]\n" \
    "	ds_read_b128 v[12:15], v108 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[92:95], v[60:63], a[96:99]\n" \
    "	ds_read_b128 v[20:23], v114 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[92:95], v[64:67], a[132:135]\n" \
    "	ds_read_b128 v[24:27], v114 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[96:99], v[52:55], a[28:31]\n" \
    "	ds_read_b128 v[28:31], v114 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[96:99], v[56:59], a[64:67]\n" \
    "	ds_read_b128 v[32:35], v114 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[96:99], v[60:63], a[100:103]\n" \
    "	ds_read_b128 v[36:39], v114 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[96:99], v[64:67], a[136:139]\n" \
    "	ds_read_b128 v[40:43], v114 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[100:103], v[52:55], a[32:35]\n" \
    "	ds_read_b128 v[44:47], v114 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[100:103], v[56:59], a[68:71]\n" \
    "	ds_read_b128 v[48:51], v114 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[100:103], v[60:63], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[100:103], v[64:67], a[140:143]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[16:19], v[0:3], a[0:3]\n" \
    "	s_add_u32 m0, s61, 51200\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v116, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[16:19], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[68:71], v115 offset:0\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[16:19], v[8:11], a[72:75]\n" \
    "	s_add_u32 m0, s61, 52224\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v117, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[16:19], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[52:55], v109 offset:0\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[20:23], v[0:3], a[4:7]\n" \
    "	s_add_u32 m0, s61, 53248\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v118, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[20:23], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[56:59], v109 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[20:23], v[8:11], a[76:79]\n" \
    "	s_add_u32 m0, s61, 54272\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v119, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[20:23], v[12:15], a[112:115]\n" \
    "	ds_read_b128 v[60:63], v109 offset:4096\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[24:27], v[0:3], a[8:11]\n" \
    "	s_add_u32 m0, s61, 55296\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v120, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[24:27], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[64:67], v109 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[24:27], v[8:11], a[80:83]\n" \
    "	s_add_u32 m0, s61, 56320\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v121, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[24:27], v[12:15], a[116:119]\n" \
    "	ds_read_b128 v[72:75], v115 offset:2048\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[28:31], v[0:3], a[12:15]\n" \
    "	s_add_u32 m0, s61, 57344\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v122, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[28:31], v[4:7], a[48:51]\n" \
    "	ds_read_b128 v[76:79], v115 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[28:31], v[8:11], a[84:87]\n" \
    "	s_add_u32 m0, s61, 58368\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v123, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[28:31], v[12:15], a[120:123]\n" \
    "	ds_read_b128 v[80:83], v115 offset:6144\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[32:35], v[0:3], a[16:19]\n" \
    "	s_add_u32 m0, s70, 51200\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v124, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[32:35], v[4:7], a[52:55]\n" \
    "	ds_read_b128 v[84:87], v115 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[32:35], v[8:11], a[88:91]\n" \
    "	s_add_u32 m0, s71, 51200\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v125, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[32:35], v[12:15], a[124:127]\n" \
    "	ds_read_b128 v[88:91], v115 offset:10240\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[36:39], v[0:3], a[20:23]\n" \
    "	s_add_u32 m0, s72, 51200\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v126, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[36:39], v[4:7], a[56:59]\n" \
    "	ds_read_b128 v[92:95], v115 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[36:39], v[8:11], a[92:95]\n" \
    "	s_add_u32 m0, s73, 51200\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v127, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[36:39], v[12:15], a[128:131]\n" \
    "	ds_read_b128 v[96:99], v115 offset:14336\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[40:43], v[0:3], a[24:27]\n" \
    "	s_add_u32 m0, s74, 51200\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v128, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[40:43], v[4:7], a[60:63]\n" \
    "	ds_read_b128 v[100:103], v115 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[40:43], v[8:11], a[96:99]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[40:43], v[12:15], a[132:135]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[44:47], v[0:3], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[44:47], v[4:7], a[64:67]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[44:47], v[8:11], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[44:47], v[12:15], a[136:139]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[48:51], v[0:3], a[32:35]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[48:51], v[4:7], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[48:51], v[8:11], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[48:51], v[12:15], a[140:143]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[68:71], v[52:55], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[68:71], v[56:59], a[36:39]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[68:71], v[60:63], a[72:75]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[68:71], v[64:67], a[108:111]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[72:75], v[52:55], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[72:75], v[56:59], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[72:75], v[60:63], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[72:75], v[64:67], a[112:115]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[76:79], v[52:55], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[76:79], v[56:59], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[76:79], v[60:63], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[76:79], v[64:67], a[116:119]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[80:83], v[52:55], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[80:83], v[56:59], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[80:83], v[60:63], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[80:83], v[64:67], a[120:123]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[84:87], v[52:55], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[84:87], v[56:59], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[84:87], v[60:63], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[84:87], v[64:67], a[124:127]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[88:91], v[52:55], a[20:23]\n" \
    "	s_waitcnt vmcnt(13)\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	s_barrier\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[88:91], v[56:59], a[56:59]\n" \
    "	ds_read_b128 v[16:19], v110 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[88:91], v[60:63], a[92:95]\n" \
    "	ds_read_b128 v[0:3], v104 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[88:91], v[64:67], a[128:131]\n" \
    "	ds_read_b128 v[4:7], v104 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[92:95], v[52:55], a[24:27]\n" \
    "	ds_read_b128 v[8:11], v104 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[92:95], v[56:59], a[60:63]\n" \
    "	ds_read_b128 v[12:15], v104 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[92:95], v[60:63], a[96:99]\n" \
    "	ds_read_b128 v[20:23], v110 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[92:95], v[64:67], a[132:135]\n" \
    "	ds_read_b128 v[24:27], v110 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[96:99], v[52:55], a[28:31]\n" \
    "	ds_read_b128 v[28:31], v110 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[96:99], v[56:59], a[64:67]\n" \
    "	ds_read_b128 v[32:35], v110 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[96:99], v[60:63], a[100:103]\n" \
    "	ds_read_b128 v[36:39], v110 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[96:99], v[64:67], a[136:139]\n" \
    "	ds_read_b128 v[40:43], v110 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[100:103], v[52:55], a[32:35]\n" \
    "	ds_read_b128 v[44:47], v110 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[100:103], v[56:59], a[68:71]\n" \
    "	ds_read_b128 v[48:51], v110 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[100:103], v[60:63], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[100:103], v[64:67], a[140:143]\n" \
    "	s_sub_u32 s60, s60, 1\n" \
    "	s_cmp_eq_u32 s60, 0\n" \
    "	s_cbranch_scc0 LOOP_%=\n" \
    "LAST_%=:\n" \
    "	s_cmp_eq_u32 %[rem], 1\n" \
    "	s_cbranch_scc1 LAST1_%=\n" \
    "	s_cmp_eq_u32 %[rem], 2\n" \
    "	s_cbranch_scc1 LAST2_%=\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[16:19], v[0:3], a[0:3]\n" \
    "	s_add_u32 m0, s61, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v116, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[16:19], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[68:71], v111 offset:0\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[16:19], v[8:11], a[72:75]\n" \
    "	s_add_u32 m0, s61, 103424\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v117, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[16:19], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[52:55], v105 offset:0\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[20:23], v[0:3], a[4:7]\n" \
    "	s_add_u32 m0, s61, 104448\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v118, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[20:23], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[56:59], v105 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[20:23], v[8:11], a[76:79]\n" \
    "	s_add_u32 m0, s61, 105472\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v119, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[20:23], v[12:15], a[112:115]\n" \
    "	ds_read_b128 v[60:63], v105 offset:4096\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[24:27], v[0:3], a[8:11]\n" \
    "	s_add_u32 m0, s61, 106496\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v120, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[24:27], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[64:67], v105 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[24:27], v[8:11], a[80:83]\n" \
    "	s_add_u32 m0, s61, 107520\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v121, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[24:27], v[12:15], a[116:119]\n" \
    "	ds_read_b128 v[72:75], v111 offset:2048\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[28:31], v[0:3], a[12:15]\n" \
    "	s_add_u32 m0, s61, 108544\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v122, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[28:31], v[4:7], a[48:51]\n" \
    "	ds_read_b128 v[76:79], v111 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[28:31], v[8:11], a[84:87]\n" \
    "	s_add_u32 m0, s61, 109568\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v123, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[28:31], v[12:15], a[120:123]\n" \
    "	ds_read_b128 v[80:83], v111 offset:6144\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[32:35], v[0:3], a[16:19]\n" \
    "	s_add_u32 m0, s70, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v124, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[32:35], v[4:7], a[52:55]\n" \
    "	ds_read_b128 v[84:87], v111 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[32:35], v[8:11], a[88:91]\n" \
    "	s_add_u32 m0, s71, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v125, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[32:35], v[12:15], a[124:127]\n" \
    "	ds_read_b128 v[88:91], v111 offset:10240\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[36:39], v[0:3], a[20:23]\n" \
    "	s_add_u32 m0, s72, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v126, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[36:39], v[4:7], a[56:59]\n" \
    "	ds_read_b128 v[92:95], v111 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[36:39], v[8:11], a[92:95]\n" \
    "	s_add_u32 m0, s73, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v127, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[36:39], v[12:15], a[128:131]\n" \
    "	ds_read_b128 v[96:99], v111 offset:14336\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[40:43], v[0:3], a[24:27]\n" \
    "	s_add_u32 m0, s74, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v128, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[40:43], v[4:7], a[60:63]\n" \
    "	ds_read_b128 v[100:103], v111 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[40:43], v[8:11], a[96:99]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[40:43], v[12:15], a[132:135]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[44:47], v[0:3], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[44:47], v[4:7], a[64:67]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[44:47], v[8:11], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[44:47], v[12:15], a[136:139]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[48:51], v[0:3], a[32:35]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[48:51], v[4:7], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[48:51], v[8:11], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[48:51], v[12:15], a[140:143]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[68:71], v[52:55], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[68:71], v[56:59], a[36:39]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[68:71], v[60:63], a[72:75]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[68:71], v[64:67], a[108:111]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[72:75], v[52:55], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[72:75], v[56:59], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[72:75], v[60:63], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[72:75], v[64:67], a[112:115]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[76:79], v[52:55], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[76:79], v[56:59], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[76:79], v[60:63], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[76:79], v[64:67], a[116:119]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[80:83], v[52:55], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[80:83], v[56:59], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[80:83], v[60:63], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[80:83], v[64:67], a[120:123]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[84:87], v[52:55], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[84:87], v[56:59], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[84:87], v[60:63], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[84:87], v[64:67], a[124:127]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[88:91], v[52:55], a[20:23]\n" \
    "	s_waitcnt vmcnt(13)\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	s_barrier\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[88:91], v[56:59], a[56:59]\n" \
    "	ds_read_b128 v[16:19], v112 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[88:91], v[60:63], a[92:95]\n" \
    "	ds_read_b128 v[0:3], v106 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[88:91], v[64:67], a[128:131]\n" \
    "	ds_read_b128 v[4:7], v106 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[92:95], v[52:55], a[24:27]\n" \
    "	ds_read_b128 v[8:11], v106 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[92:95], v[56:59], a[60:63]\n" \
    "	ds_read_b128 v[12:15], v106 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[92:95], v[60:63], a[96:99]\n" \
    "	ds_read_b128 v[20:23], v112 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[92:95], v[64:67], a[132:135]\n" \
    "	ds_read_b128 v[24:27], v112 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[96:99], v[52:55], a[28:31]\n" \
    "	ds_read_b128 v[28:31], v112 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[96:99], v[56:59], a[64:67]\n" \
    "	ds_read_b128 v[32:35], v112 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[96:99], v[60:63], a[100:103]\n" \
    "	ds_read_b128 v[36:39], v112 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[96:99], v[64:67], a[136:139]\n" \
    "	ds_read_b128 v[40:43], v112 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[100:103], v[52:55], a[32:35]\n" \
    "	ds_read_b128 v[44:47], v112 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[100:103], v[56:59], a[68:71]\n" \
    "	ds_read_b128 v[48:51], v112 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[100:103], v[60:63], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[100:103], v[64:67], a[140:143]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[16:19], v[0:3], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[16:19], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[68:71], v113 offset:0\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[16:19], v[8:11], a[72:75]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[16:19], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[52:55], v107 offset:0\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[20:23], v[0:3], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[20:23], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[56:59], v107 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[20:23], v[8:11], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[20:23], v[12:15], a[112:115]\n" \
    "	ds_read_b128 v[60:63], v107 offset:4096\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[24:27], v[0:3], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[24:27], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[64:67], v107 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[24:27], v[8:11], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[24:27], v[12:15], a[116:119]\n" \
    "	ds_read_b128 v[72:75], v113 offset:2048\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[28:31], v[0:3], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[28:31], v[4:7], a[48:51]\n" \
    "	ds_read_b128 v[76:79], v113 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[28:31], v[8:11], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[28:31], v[12:15], a[120:123]\n" \
    "	ds_read_b128 v[80:83], v113 offset:6144\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[32:35], v[0:3], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[32:35], v[4:7], a[52:55]\n" \
    "	ds_read_b128 v[84:87], v113 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[32:35], v[8:11], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[32:35], v[12:15], a[124:127]\n" \
    "	ds_read_b128 v[88:91], v113 offset:10240\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[36:39], v[0:3], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[36:39], v[4:7], a[56:59]\n" \
    "	ds_read_b128 v[92:95], v113 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[36:39], v[8:11], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[36:39], v[12:15], a[128:131]\n" \
    "	ds_read_b128 v[96:99], v113 offset:14336\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[40:43], v[0:3], a[24:27]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[40:43], v[4:7], a[60:63]\n" \
    "	ds_read_b128 v[100:103], v113 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[40:43], v[8:11], a[96:99]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[40:43], v[12:15], a[132:135]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[44:47], v[0:3], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[44:47], v[4:7], a[64:67]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[44:47], v[8:11], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[44:47], v[12:15], a[136:139]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[48:51], v[0:3], a[32:35]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[48:51], v[4:7], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[48:51], v[8:11], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[48:51], v[12:15], a[140:143]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[68:71], v[52:55], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[68:71], v[56:59], a[36:39]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[68:71], v[60:63], a[72:75]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[68:71], v[64:67], a[108:111]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[72:75], v[52:55], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[72:75], v[56:59], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[72:75], v[60:63], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[72:75], v[64:67], a[112:115]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[76:79], v[52:55], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[76:79], v[56:59], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[76:79], v[60:63], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[76:79], v[64:67], a[116:119]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[80:83], v[52:55], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[80:83], v[56:59], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[80:83], v[60:63], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[80:83], v[64:67], a[120:123]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[84:87], v[52:55], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[84:87], v[56:59], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[84:87], v[60:63], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[84:87], v[64:67], a[124:127]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[88:91], v[52:55], a[20:23]\n" \
    "	s_waitcnt vmcnt(0)\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	s_barrier\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[88:91], v[56:59], a[56:59]\n" \
    "	ds_read_b128 v[16:19], v114 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[88:91], v[60:63], a[92:95]\n" \
    "	ds_read_b128 v[0:3], v108 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[88:91], v[64:67], a[128:131]\n" \
    "	ds_read_b128 v[4:7], v108 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[92:95], v[52:55], a[24:27]\n" \
    "	ds_read_b128 v[8:11], v108 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[92:95], v[56:59], a[60:63]\n" \
    "	ds_read_b128 v[12:15], v108 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[92:95], v[60:63], a[96:99]\n" \
    "	ds_read_b128 v[20:23], v114 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[92:95], v[64:67], a[132:135]\n" \
    "	ds_read_b128 v[24:27], v114 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[96:99], v[52:55], a[28:31]\n" \
    "	ds_read_b128 v[28:31], v114 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[96:99], v[56:59], a[64:67]\n" \
    "	ds_read_b128 v[32:35], v114 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[96:99], v[60:63], a[100:103]\n" \
    "	ds_read_b128 v[36:39], v114 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[96:99], v[64:67], a[136:139]\n" \
    "	ds_read_b128 v[40:43], v114 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[100:103], v[52:55], a[32:35]\n" \
    "	ds_read_b128 v[44:47], v114 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[100:103], v[56:59], a[68:71]\n" \
    "	ds_read_b128 v[48:51], v114 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[100:103], v[60:63], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[100:103], v[64:67], a[140:143]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[16:19], v[0:3], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[16:19], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[68:71], v115 offset:0\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[16:19], v[8:11], a[72:75]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[16:19], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[52:55], v109 offset:0\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[20:23], v[0:3], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[20:23], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[56:59], v109 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[20:23], v[8:11], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[20:23], v[12:15], a[112:115]\n" \
    "	ds_read_b128 v[60:63], v109 offset:4096\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[24:27], v[0:3], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[24:27], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[64:67], v109 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[24:27], v[8:11], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[24:27], v[12:15], a[116:119]\n" \
    "	ds_read_b128 v[72:75], v115 offset:2048\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[28:31], v[0:3], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[28:31], v[4:7], a[48:51]\n" \
    "	ds_read_b128 v[76:79], v115 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[28:31], v[8:11], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[28:31], v[12:15], a[120:123]\n" \
    "	ds_read_b128 v[80:83], v115 offset:6144\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[32:35], v[0:3], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[32:35], v[4:7], a[52:55]\n" \
    "	ds_read_b128 v[84:87], v115 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[32:35], v[8:11], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[32:35], v[12:15], a[124:127]\n" \
    "	ds_read_b128 v[88:91], v115 offset:10240\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[36:39], v[0:3], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[36:39], v[4:7], a[56:59]\n" \
    "	ds_read_b128 v[92:95], v115 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[36:39], v[8:11], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[36:39], v[12:15], a[128:131]\n" \
    "	ds_read_b128 v[96:99], v115 offset:14336\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[40:43], v[0:3], a[24:27]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[40:43], v[4:7], a[60:63]\n" \
    "	ds_read_b128 v[100:103], v115 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[40:43], v[8:11], a[96:99]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[40:43], v[12:15], a[132:135]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[44:47], v[0:3], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[44:47], v[4:7], a[64:67]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[44:47], v[8:11], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[44:47], v[12:15], a[136:139]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[48:51], v[0:3], a[32:35]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[48:51], v[4:7], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[48:51], v[8:11], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[48:51], v[12:15], a[140:143]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[68:71], v[52:55], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[68:71], v[56:59], a[36:39]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[68:71], v[60:63], a[72:75]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[68:71], v[64:67], a[108:111]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[72:75], v[52:55], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[72:75], v[56:59], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[72:75], v[60:63], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[72:75], v[64:67], a[112:115]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[76:79], v[52:55], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[76:79], v[56:59], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[76:79], v[60:63], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[76:79], v[64:67], a[116:119]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[80:83], v[52:55], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[80:83], v[56:59], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[80:83], v[60:63], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[80:83], v[64:67], a[120:123]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[84:87], v[52:55], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[84:87], v[56:59], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[84:87], v[60:63], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[84:87], v[64:67], a[124:127]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[88:91], v[52:55], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[88:91], v[56:59], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[88:91], v[60:63], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[88:91], v[64:67], a[128:131]\n" \
    "	s_waitcnt lgkmcnt(2)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[92:95], v[52:55], a[24:27]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[92:95], v[56:59], a[60:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[92:95], v[60:63], a[96:99]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[92:95], v[64:67], a[132:135]\n" \
    "	s_waitcnt lgkmcnt(1)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[96:99], v[52:55], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[96:99], v[56:59], a[64:67]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[96:99], v[60:63], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[96:99], v[64:67], a[136:139]\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[100:103], v[52:55], a[32:35]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[100:103], v[56:59], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[100:103], v[60:63], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[100:103], v[64:67], a[140:143]\n" \
    "	s_branch DONE_%=\n" \
    "LAST1_%=:\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[16:19], v[0:3], a[0:3]\n" \
    "	s_add_u32 m0, s61, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v116, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[16:19], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[68:71], v111 offset:0\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[16:19], v[8:11], a[72:75]\n" \
    "	s_add_u32 m0, s61, 103424\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v117, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[16:19], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[52:55], v105 offset:0\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[20:23], v[0:3], a[4:7]\n" \
    "	s_add_u32 m0, s61, 104448\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v118, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[20:23], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[56:59], v105 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[20:23], v[8:11], a[76:79]\n" \
    "	s_add_u32 m0, s61, 105472\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v119, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[20:23], v[12:15], a[112:115]\n" \
    "	ds_read_b128 v[60:63], v105 offset:4096\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[24:27], v[0:3], a[8:11]\n" \
    "	s_add_u32 m0, s61, 106496\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v120, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[24:27], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[64:67], v105 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[24:27], v[8:11], a[80:83]\n" \
    "	s_add_u32 m0, s61, 107520\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v121, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[24:27], v[12:15], a[116:119]\n" \
    "	ds_read_b128 v[72:75], v111 offset:2048\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[28:31], v[0:3], a[12:15]\n" \
    "	s_add_u32 m0, s61, 108544\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v122, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[28:31], v[4:7], a[48:51]\n" \
    "	ds_read_b128 v[76:79], v111 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[28:31], v[8:11], a[84:87]\n" \
    "	s_add_u32 m0, s61, 109568\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v123, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[28:31], v[12:15], a[120:123]\n" \
    "	ds_read_b128 v[80:83], v111 offset:6144\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[32:35], v[0:3], a[16:19]\n" \
    "	s_add_u32 m0, s70, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v124, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[32:35], v[4:7], a[52:55]\n" \
    "	ds_read_b128 v[84:87], v111 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[32:35], v[8:11], a[88:91]\n" \
    "	s_add_u32 m0, s71, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v125, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[32:35], v[12:15], a[124:127]\n" \
    "	ds_read_b128 v[88:91], v111 offset:10240\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[36:39], v[0:3], a[20:23]\n" \
    "	s_add_u32 m0, s72, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v126, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[36:39], v[4:7], a[56:59]\n" \
    "	ds_read_b128 v[92:95], v111 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[36:39], v[8:11], a[92:95]\n" \
    "	s_add_u32 m0, s73, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v127, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[36:39], v[12:15], a[128:131]\n" \
    "	ds_read_b128 v[96:99], v111 offset:14336\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[40:43], v[0:3], a[24:27]\n" \
    "	s_add_u32 m0, s74, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v128, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[40:43], v[4:7], a[60:63]\n" \
    "	ds_read_b128 v[100:103], v111 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[40:43], v[8:11], a[96:99]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[40:43], v[12:15], a[132:135]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[44:47], v[0:3], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[44:47], v[4:7], a[64:67]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[44:47], v[8:11], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[44:47], v[12:15], a[136:139]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[48:51], v[0:3], a[32:35]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[48:51], v[4:7], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[48:51], v[8:11], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[48:51], v[12:15], a[140:143]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[68:71], v[52:55], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[68:71], v[56:59], a[36:39]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[68:71], v[60:63], a[72:75]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[68:71], v[64:67], a[108:111]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[72:75], v[52:55], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[72:75], v[56:59], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[72:75], v[60:63], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[72:75], v[64:67], a[112:115]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[76:79], v[52:55], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[76:79], v[56:59], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[76:79], v[60:63], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[76:79], v[64:67], a[116:119]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[80:83], v[52:55], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[80:83], v[56:59], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[80:83], v[60:63], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[80:83], v[64:67], a[120:123]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[84:87], v[52:55], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[84:87], v[56:59], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[84:87], v[60:63], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[84:87], v[64:67], a[124:127]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[88:91], v[52:55], a[20:23]\n" \
    "	s_waitcnt vmcnt(13)\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	s_barrier\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[88:91], v[56:59], a[56:59]\n" \
    "	ds_read_b128 v[16:19], v112 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[88:91], v[60:63], a[92:95]\n" \
    "	ds_read_b128 v[0:3], v106 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[88:91], v[64:67], a[128:131]\n" \
    "	ds_read_b128 v[4:7], v106 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[92:95], v[52:55], a[24:27]\n" \
    "	ds_read_b128 v[8:11], v106 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[92:95], v[56:59], a[60:63]\n" \
    "	ds_read_b128 v[12:15], v106 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[92:95], v[60:63], a[96:99]\n" \
    "	ds_read_b128 v[20:23], v112 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[92:95], v[64:67], a[132:135]\n" \
    "	ds_read_b128 v[24:27], v112 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[96:99], v[52:55], a[28:31]\n" \
    "	ds_read_b128 v[28:31], v112 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[96:99], v[56:59], a[64:67]\n" \
    "	ds_read_b128 v[32:35], v112 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[96:99], v[60:63], a[100:103]\n" \
    "	ds_read_b128 v[36:39], v112 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[96:99], v[64:67], a[136:139]\n" \
    "	ds_read_b128 v[40:43], v112 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[100:103], v[52:55], a[32:35]\n" \
    "	ds_read_b128 v[44:47], v112 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[100:103], v[56:59], a[68:71]\n" \
    "	ds_read_b128 v[48:51], v112 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[100:103], v[60:63], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[100:103], v[64:67], a[140:143]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[16:19], v[0:3], a[0:3]\n" \
    "	s_add_u32 m0, s61, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v116, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[16:19], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[68:71], v113 offset:0\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[16:19], v[8:11], a[72:75]\n" \
    "	s_add_u32 m0, s61, 1024\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v117, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[16:19], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[52:55], v107 offset:0\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[20:23], v[0:3], a[4:7]\n" \
    "	s_add_u32 m0, s61, 2048\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v118, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[20:23], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[56:59], v107 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[20:23], v[8:11], a[76:79]\n" \
    "	s_add_u32 m0, s61, 3072\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v119, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[20:23], v[12:15], a[112:115]\n" \
    "	ds_read_b128 v[60:63], v107 offset:4096\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[24:27], v[0:3], a[8:11]\n" \
    "	s_add_u32 m0, s61, 4096\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v120, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[24:27], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[64:67], v107 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[24:27], v[8:11], a[80:83]\n" \
    "	s_add_u32 m0, s61, 5120\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v121, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[24:27], v[12:15], a[116:119]\n" \
    "	ds_read_b128 v[72:75], v113 offset:2048\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[28:31], v[0:3], a[12:15]\n" \
    "	s_add_u32 m0, s61, 6144\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v122, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[28:31], v[4:7], a[48:51]\n" \
    "	ds_read_b128 v[76:79], v113 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[28:31], v[8:11], a[84:87]\n" \
    "	s_add_u32 m0, s61, 7168\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v123, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[28:31], v[12:15], a[120:123]\n" \
    "	ds_read_b128 v[80:83], v113 offset:6144\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[32:35], v[0:3], a[16:19]\n" \
    "	s_add_u32 m0, s70, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v124, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[32:35], v[4:7], a[52:55]\n" \
    "	ds_read_b128 v[84:87], v113 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[32:35], v[8:11], a[88:91]\n" \
    "	s_add_u32 m0, s71, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v125, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[32:35], v[12:15], a[124:127]\n" \
    "	ds_read_b128 v[88:91], v113 offset:10240\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[36:39], v[0:3], a[20:23]\n" \
    "	s_add_u32 m0, s72, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v126, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[36:39], v[4:7], a[56:59]\n" \
    "	ds_read_b128 v[92:95], v113 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[36:39], v[8:11], a[92:95]\n" \
    "	s_add_u32 m0, s73, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v127, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[36:39], v[12:15], a[128:131]\n" \
    "	ds_read_b128 v[96:99], v113 offset:14336\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[40:43], v[0:3], a[24:27]\n" \
    "	s_add_u32 m0, s74, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v128, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[40:43], v[4:7], a[60:63]\n" \
    "	ds_read_b128 v[100:103], v113 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[40:43], v[8:11], a[96:99]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[40:43], v[12:15], a[132:135]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[44:47], v[0:3], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[44:47], v[4:7], a[64:67]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[44:47], v[8:11], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[44:47], v[12:15], a[136:139]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[48:51], v[0:3], a[32:35]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[48:51], v[4:7], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[48:51], v[8:11], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[48:51], v[12:15], a[140:143]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[68:71], v[52:55], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[68:71], v[56:59], a[36:39]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[68:71], v[60:63], a[72:75]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[68:71], v[64:67], a[108:111]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[72:75], v[52:55], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[72:75], v[56:59], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[72:75], v[60:63], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[72:75], v[64:67], a[112:115]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[76:79], v[52:55], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[76:79], v[56:59], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[76:79], v[60:63], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[76:79], v[64:67], a[116:119]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[80:83], v[52:55], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[80:83], v[56:59], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[80:83], v[60:63], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[80:83], v[64:67], a[120:123]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[84:87], v[52:55], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[84:87], v[56:59], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[84:87], v[60:63], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[84:87], v[64:67], a[124:127]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[88:91], v[52:55], a[20:23]\n" \
    "	s_waitcnt vmcnt(13)\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	s_barrier\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[88:91], v[56:59], a[56:59]\n" \
    "	ds_read_b128 v[16:19], v114 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[88:91], v[60:63], a[92:95]\n" \
    "	ds_read_b128 v[0:3], v108 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[88:91], v[64:67], a[128:131]\n" \
    "	ds_read_b128 v[4:7], v108 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[92:95], v[52:55], a[24:27]\n" \
    "	ds_read_b128 v[8:11], v108 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[92:95], v[56:59], a[60:63]\n" \
    "	ds_read_b128 v[12:15], v108 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[92:95], v[60:63], a[96:99]\n" \
    "	ds_read_b128 v[20:23], v114 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[92:95], v[64:67], a[132:135]\n" \
    "	ds_read_b128 v[24:27], v114 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[96:99], v[52:55], a[28:31]\n" \
    "	ds_read_b128 v[28:31], v114 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[96:99], v[56:59], a[64:67]\n" \
    "	ds_read_b128 v[32:35], v114 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[96:99], v[60:63], a[100:103]\n" \
    "	ds_read_b128 v[36:39], v114 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[96:99], v[64:67], a[136:139]\n" \
    "	ds_read_b128 v[40:43], v114 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[100:103], v[52:55], a[32:35]\n" \
    "	ds_read_b128 v[44:47], v114 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[100:103], v[56:59], a[68:71]\n" \
    "	ds_read_b128 v[48:51], v114 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[100:103], v[60:63], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[100:103], v[64:67], a[140:143]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[16:19], v[0:3], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[16:19], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[68:71], v115 offset:0\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[16:19], v[8:11], a[72:75]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[16:19], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[52:55], v109 offset:0\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[20:23], v[0:3], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[20:23], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[56:59], v109 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[20:23], v[8:11], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[20:23], v[12:15], a[112:115]\n" \
    "	ds_read_b128 v[60:63], v109 offset:4096\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[24:27], v[0:3], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[24:27], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[64:67], v109 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[24:27], v[8:11], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[24:27], v[12:15], a[116:119]\n" \
    "	ds_read_b128 v[72:75], v115 offset:2048\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[28:31], v[0:3], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[28:31], v[4:7], a[48:51]\n" \
    "	ds_read_b128 v[76:79], v115 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[28:31], v[8:11], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[28:31], v[12:15], a[120:123]\n" \
    "	ds_read_b128 v[80:83], v115 offset:6144\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[32:35], v[0:3], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[32:35], v[4:7], a[52:55]\n" \
    "	ds_read_b128 v[84:87], v115 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[32:35], v[8:11], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[32:35], v[12:15], a[124:127]\n" \
    "	ds_read_b128 v[88:91], v115 offset:10240\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[36:39], v[0:3], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[36:39], v[4:7], a[56:59]\n" \
    "	ds_read_b128 v[92:95], v115 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[36:39], v[8:11], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[36:39], v[12:15], a[128:131]\n" \
    "	ds_read_b128 v[96:99], v115 offset:14336\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[40:43], v[0:3], a[24:27]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[40:43], v[4:7], a[60:63]\n" \
    "	ds_read_b128 v[100:103], v115 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[40:43], v[8:11], a[96:99]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[40:43], v[12:15], a[132:135]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[44:47], v[0:3], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[44:47], v[4:7], a[64:67]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[44:47], v[8:11], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[44:47], v[12:15], a[136:139]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[48:51], v[0:3], a[32:35]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[48:51], v[4:7], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[48:51], v[8:11], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[48:51], v[12:15], a[140:143]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[68:71], v[52:55], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[68:71], v[56:59], a[36:39]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[68:71], v[60:63], a[72:75]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[68:71], v[64:67], a[108:111]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[72:75], v[52:55], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[72:75], v[56:59], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[72:75], v[60:63], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[72:75], v[64:67], a[112:115]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[76:79], v[52:55], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[76:79], v[56:59], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[76:79], v[60:63], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[76:79], v[64:67], a[116:119]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[80:83], v[52:55], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[80:83], v[56:59], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[80:83], v[60:63], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[80:83], v[64:67], a[120:123]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[84:87], v[52:55], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[84:87], v[56:59], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[84:87], v[60:63], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[84:87], v[64:67], a[124:127]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[88:91], v[52:55], a[20:23]\n" \
    "	s_waitcnt vmcnt(0)\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	s_barrier\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[88:91], v[56:59], a[56:59]\n" \
    "	ds_read_b128 v[16:19], v110 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[88:91], v[60:63], a[92:95]\n" \
    "	ds_read_b128 v[0:3], v104 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[88:91], v[64:67], a[128:131]\n" \
    "	ds_read_b128 v[4:7], v104 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[92:95], v[52:55], a[24:27]\n" \
    "	ds_read_b128 v[8:11], v104 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[92:95], v[56:59], a[60:63]\n" \
    "	ds_read_b128 v[12:15], v104 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[92:95], v[60:63], a[96:99]\n" \
    "	ds_read_b128 v[20:23], v110 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[92:95], v[64:67], a[132:135]\n" \
    "	ds_read_b128 v[24:27], v110 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[96:99], v[52:55], a[28:31]\n" \
    "	ds_read_b128 v[28:31], v110 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[96:99], v[56:59], a[64:67]\n" \
    "	ds_read_b128 v[32:35], v110 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[96:99], v[60:63], a[100:103]\n" \
    "	ds_read_b128 v[36:39], v110 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[96:99], v[64:67], a[136:139]\n" \
    "	ds_read_b128 v[40:43], v110 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[100:103], v[52:55], a[32:35]\n" \
    "	ds_read_b128 v[44:47], v110 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[100:103], v[56:59], a[68:71]\n" \
    "	ds_read_b128 v[48:51], v110 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[100:103], v[60:63], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[100:103], v[64:67], a[140:143]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[16:19], v[0:3], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[16:19], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[68:71], v111 offset:0\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[16:19], v[8:11], a[72:75]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[16:19], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[52:55], v105 offset:0\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[20:23], v[0:3], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[20:23], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[56:59], v105 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[20:23], v[8:11], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[20:23], v[12:15], a[112:115]\n" \
    "	ds_read_b128 v[60:63], v105 offset:4096\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[24:27], v[0:3], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[24:27], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[64:67], v105 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[24:27], v[8:11], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[24:27], v[12:15], a[116:119]\n" \
    "	ds_read_b128 v[72:75], v111 offset:2048\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[28:31], v[0:3], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[28:31], v[4:7], a[48:51]\n" \
    "	ds_read_b128 v[76:79], v111 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[28:31], v[8:11], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[28:31], v[12:15], a[120:123]\n" \
    "	ds_read_b128 v[80:83], v111 offset:6144\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[32:35], v[0:3], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[32:35], v[4:7], a[52:55]\n" \
    "	ds_read_b128 v[84:87], v111 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[32:35], v[8:11], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[32:35], v[12:15], a[124:127]\n" \
    "	ds_read_b128 v[88:91], v111 offset:10240\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[36:39], v[0:3], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[36:39], v[4:7], a[56:59]\n" \
    "	ds_read_b128 v[92:95], v111 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[36:39], v[8:11], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[36:39], v[12:15], a[128:131]\n" \
    "	ds_read_b128 v[96:99], v111 offset:14336\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[40:43], v[0:3], a[24:27]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[40:43], v[4:7], a[60:63]\n" \
    "	ds_read_b128 v[100:103], v111 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[40:43], v[8:11], a[96:99]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[40:43], v[12:15], a[132:135]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[44:47], v[0:3], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[44:47], v[4:7], a[64:67]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[44:47], v[8:11], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[44:47], v[12:15], a[136:139]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[48:51], v[0:3], a[32:35]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[48:51], v[4:7], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[48:51], v[8:11], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[48:51], v[12:15], a[140:143]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[68:71], v[52:55], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[68:71], v[56:59], a[36:39]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[68:71], v[60:63], a[72:75]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[68:71], v[64:67], a[108:111]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[72:75], v[52:55], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[72:75], v[56:59], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[72:75], v[60:63], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[72:75], v[64:67], a[112:115]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[76:79], v[52:55], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[76:79], v[56:59], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[76:79], v[60:63], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[76:79], v[64:67], a[116:119]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[80:83], v[52:55], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[80:83], v[56:59], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[80:83], v[60:63], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[80:83], v[64:67], a[120:123]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[84:87], v[52:55], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[84:87], v[56:59], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[84:87], v[60:63], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[84:87], v[64:67], a[124:127]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[88:91], v[52:55], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[88:91], v[56:59], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[88:91], v[60:63], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[88:91], v[64:67], a[128:131]\n" \
    "	s_waitcnt lgkmcnt(2)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[92:95], v[52:55], a[24:27]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[92:95], v[56:59], a[60:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[92:95], v[60:63], a[96:99]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[92:95], v[64:67], a[132:135]\n" \
    "	s_waitcnt lgkmcnt(1)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[96:99], v[52:55], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[96:99], v[56:59], a[64:67]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[96:99], v[60:63], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[96:99], v[64:67], a[136:139]\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[100:103], v[52:55], a[32:35]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[100:103], v[56:59], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[100:103], v[60:63], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[100:103], v[64:67], a[140:143]\n" \
    "	s_branch DONE_%=\n" \
    "LAST2_%=:\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[16:19], v[0:3], a[0:3]\n" \
    "	s_add_u32 m0, s61, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v116, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[16:19], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[68:71], v111 offset:0\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[16:19], v[8:11], a[72:75]\n" \
    "	s_add_u32 m0, s61, 103424\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v117, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[16:19], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[52:55], v105 offset:0\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[20:23], v[0:3], a[4:7]\n" \
    "	s_add_u32 m0, s61, 104448\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v118, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[20:23], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[56:59], v105 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[20:23], v[8:11], a[76:79]\n" \
    "	s_add_u32 m0, s61, 105472\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v119, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[20:23], v[12:15], a[112:115]\n" \
    "	ds_read_b128 v[60:63], v105 offset:4096\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[24:27], v[0:3], a[8:11]\n" \
    "	s_add_u32 m0, s61, 106496\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v120, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[24:27], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[64:67], v105 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[24:27], v[8:11], a[80:83]\n" \
    "	s_add_u32 m0, s61, 107520\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v121, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[24:27], v[12:15], a[116:119]\n" \
    "	ds_read_b128 v[72:75], v111 offset:2048\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[28:31], v[0:3], a[12:15]\n" \
    "	s_add_u32 m0, s61, 108544\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v122, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[28:31], v[4:7], a[48:51]\n" \
    "	ds_read_b128 v[76:79], v111 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[28:31], v[8:11], a[84:87]\n" \
    "	s_add_u32 m0, s61, 109568\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v123, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[28:31], v[12:15], a[120:123]\n" \
    "	ds_read_b128 v[80:83], v111 offset:6144\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[32:35], v[0:3], a[16:19]\n" \
    "	s_add_u32 m0, s70, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v124, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[32:35], v[4:7], a[52:55]\n" \
    "	ds_read_b128 v[84:87], v111 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[32:35], v[8:11], a[88:91]\n" \
    "	s_add_u32 m0, s71, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v125, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[32:35], v[12:15], a[124:127]\n" \
    "	ds_read_b128 v[88:91], v111 offset:10240\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[36:39], v[0:3], a[20:23]\n" \
    "	s_add_u32 m0, s72, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v126, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[36:39], v[4:7], a[56:59]\n" \
    "	ds_read_b128 v[92:95], v111 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[36:39], v[8:11], a[92:95]\n" \
    "	s_add_u32 m0, s73, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v127, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[36:39], v[12:15], a[128:131]\n" \
    "	ds_read_b128 v[96:99], v111 offset:14336\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[40:43], v[0:3], a[24:27]\n" \
    "	s_add_u32 m0, s74, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v128, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[40:43], v[4:7], a[60:63]\n" \
    "	ds_read_b128 v[100:103], v111 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[40:43], v[8:11], a[96:99]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[40:43], v[12:15], a[132:135]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[44:47], v[0:3], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[44:47], v[4:7], a[64:67]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[44:47], v[8:11], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[44:47], v[12:15], a[136:139]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[48:51], v[0:3], a[32:35]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[48:51], v[4:7], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[48:51], v[8:11], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[48:51], v[12:15], a[140:143]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[68:71], v[52:55], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[68:71], v[56:59], a[36:39]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[68:71], v[60:63], a[72:75]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[68:71], v[64:67], a[108:111]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[72:75], v[52:55], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[72:75], v[56:59], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[72:75], v[60:63], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[72:75], v[64:67], a[112:115]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[76:79], v[52:55], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[76:79], v[56:59], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[76:79], v[60:63], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[76:79], v[64:67], a[116:119]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[80:83], v[52:55], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[80:83], v[56:59], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[80:83], v[60:63], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[80:83], v[64:67], a[120:123]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[84:87], v[52:55], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[84:87], v[56:59], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[84:87], v[60:63], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[84:87], v[64:67], a[124:127]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[88:91], v[52:55], a[20:23]\n" \
    "	s_waitcnt vmcnt(13)\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	s_barrier\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[88:91], v[56:59], a[56:59]\n" \
    "	ds_read_b128 v[16:19], v112 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[88:91], v[60:63], a[92:95]\n" \
    "	ds_read_b128 v[0:3], v106 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[88:91], v[64:67], a[128:131]\n" \
    "	ds_read_b128 v[4:7], v106 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[92:95], v[52:55], a[24:27]\n" \
    "	ds_read_b128 v[8:11], v106 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[92:95], v[56:59], a[60:63]\n" \
    "	ds_read_b128 v[12:15], v106 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[92:95], v[60:63], a[96:99]\n" \
    "	ds_read_b128 v[20:23], v112 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[92:95], v[64:67], a[132:135]\n" \
    "	ds_read_b128 v[24:27], v112 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[96:99], v[52:55], a[28:31]\n" \
    "	ds_read_b128 v[28:31], v112 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[96:99], v[56:59], a[64:67]\n" \
    "	ds_read_b128 v[32:35], v112 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[96:99], v[60:63], a[100:103]\n" \
    "	ds_read_b128 v[36:39], v112 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[96:99], v[64:67], a[136:139]\n" \
    "	ds_read_b128 v[40:43], v112 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[100:103], v[52:55], a[32:35]\n" \
    "	ds_read_b128 v[44:47], v112 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[100:103], v[56:59], a[68:71]\n" \
    "	ds_read_b128 v[48:51], v112 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[100:103], v[60:63], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[100:103], v[64:67], a[140:143]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[16:19], v[0:3], a[0:3]\n" \
    "	s_add_u32 m0, s61, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v116, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[16:19], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[68:71], v113 offset:0\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[16:19], v[8:11], a[72:75]\n" \
    "	s_add_u32 m0, s61, 1024\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v117, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[16:19], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[52:55], v107 offset:0\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[20:23], v[0:3], a[4:7]\n" \
    "	s_add_u32 m0, s61, 2048\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v118, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[20:23], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[56:59], v107 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[20:23], v[8:11], a[76:79]\n" \
    "	s_add_u32 m0, s61, 3072\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v119, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[20:23], v[12:15], a[112:115]\n" \
    "	ds_read_b128 v[60:63], v107 offset:4096\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[24:27], v[0:3], a[8:11]\n" \
    "	s_add_u32 m0, s61, 4096\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v120, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[24:27], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[64:67], v107 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[24:27], v[8:11], a[80:83]\n" \
    "	s_add_u32 m0, s61, 5120\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v121, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[24:27], v[12:15], a[116:119]\n" \
    "	ds_read_b128 v[72:75], v113 offset:2048\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[28:31], v[0:3], a[12:15]\n" \
    "	s_add_u32 m0, s61, 6144\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v122, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[28:31], v[4:7], a[48:51]\n" \
    "	ds_read_b128 v[76:79], v113 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[28:31], v[8:11], a[84:87]\n" \
    "	s_add_u32 m0, s61, 7168\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v123, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[28:31], v[12:15], a[120:123]\n" \
    "	ds_read_b128 v[80:83], v113 offset:6144\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[32:35], v[0:3], a[16:19]\n" \
    "	s_add_u32 m0, s70, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v124, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[32:35], v[4:7], a[52:55]\n" \
    "	ds_read_b128 v[84:87], v113 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[32:35], v[8:11], a[88:91]\n" \
    "	s_add_u32 m0, s71, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v125, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[32:35], v[12:15], a[124:127]\n" \
    "	ds_read_b128 v[88:91], v113 offset:10240\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[36:39], v[0:3], a[20:23]\n" \
    "	s_add_u32 m0, s72, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v126, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[36:39], v[4:7], a[56:59]\n" \
    "	ds_read_b128 v[92:95], v113 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[36:39], v[8:11], a[92:95]\n" \
    "	s_add_u32 m0, s73, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v127, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[36:39], v[12:15], a[128:131]\n" \
    "	ds_read_b128 v[96:99], v113 offset:14336\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[40:43], v[0:3], a[24:27]\n" \
    "	s_add_u32 m0, s74, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v128, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[40:43], v[4:7], a[60:63]\n" \
    "	ds_read_b128 v[100:103], v113 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[40:43], v[8:11], a[96:99]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[40:43], v[12:15], a[132:135]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[44:47], v[0:3], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[44:47], v[4:7], a[64:67]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[44:47], v[8:11], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[44:47], v[12:15], a[136:139]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[48:51], v[0:3], a[32:35]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[48:51], v[4:7], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[48:51], v[8:11], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[48:51], v[12:15], a[140:143]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[68:71], v[52:55], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[68:71], v[56:59], a[36:39]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[68:71], v[60:63], a[72:75]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[68:71], v[64:67], a[108:111]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[72:75], v[52:55], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[72:75], v[56:59], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[72:75], v[60:63], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[72:75], v[64:67], a[112:115]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[76:79], v[52:55], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[76:79], v[56:59], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[76:79], v[60:63], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[76:79], v[64:67], a[116:119]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[80:83], v[52:55], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[80:83], v[56:59], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[80:83], v[60:63], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[80:83], v[64:67], a[120:123]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[84:87], v[52:55], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[84:87], v[56:59], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[84:87], v[60:63], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[84:87], v[64:67], a[124:127]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[88:91], v[52:55], a[20:23]\n" \
    "	s_waitcnt vmcnt(13)\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	s_barrier\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[88:91], v[56:59], a[56:59]\n" \
    "	ds_read_b128 v[16:19], v114 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[88:91], v[60:63], a[92:95]\n" \
    "	ds_read_b128 v[0:3], v108 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[88:91], v[64:67], a[128:131]\n" \
    "	ds_read_b128 v[4:7], v108 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[92:95], v[52:55], a[24:27]\n" \
    "	ds_read_b128 v[8:11], v108 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[92:95], v[56:59], a[60:63]\n" \
    "	ds_read_b128 v[12:15], v108 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[92:95], v[60:63], a[96:99]\n" \
    "	ds_read_b128 v[20:23], v114 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[92:95], v[64:67], a[132:135]\n" \
    "	ds_read_b128 v[24:27], v114 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[96:99], v[52:55], a[28:31]\n" \
    "	ds_read_b128 v[28:31], v114 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[96:99], v[56:59], a[64:67]\n" \
    "	ds_read_b128 v[32:35], v114 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[96:99], v[60:63], a[100:103]\n" \
    "	ds_read_b128 v[36:39], v114 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[96:99], v[64:67], a[136:139]\n" \
    "	ds_read_b128 v[40:43], v114 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[100:103], v[52:55], a[32:35]\n" \
    "	ds_read_b128 v[44:47], v114 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[100:103], v[56:59], a[68:71]\n" \
    "	ds_read_b128 v[48:51], v114 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[100:103], v[60:63], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[100:103], v[64:67], a[140:143]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[16:19], v[0:3], a[0:3]\n" \
    "	s_add_u32 m0, s61, 51200\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v116, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[16:19], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[68:71], v115 offset:0\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[16:19], v[8:11], a[72:75]\n" \
    "	s_add_u32 m0, s61, 52224\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v117, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[16:19], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[52:55], v109 offset:0\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[20:23], v[0:3], a[4:7]\n" \
    "	s_add_u32 m0, s61, 53248\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v118, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[20:23], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[56:59], v109 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[20:23], v[8:11], a[76:79]\n" \
    "	s_add_u32 m0, s61, 54272\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v119, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[20:23], v[12:15], a[112:115]\n" \
    "	ds_read_b128 v[60:63], v109 offset:4096\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[24:27], v[0:3], a[8:11]\n" \
    "	s_add_u32 m0, s61, 55296\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v120, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[24:27], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[64:67], v109 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[24:27], v[8:11], a[80:83]\n" \
    "	s_add_u32 m0, s61, 56320\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v121, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[24:27], v[12:15], a[116:119]\n" \
    "	ds_read_b128 v[72:75], v115 offset:2048\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[28:31], v[0:3], a[12:15]\n" \
    "	s_add_u32 m0, s61, 57344\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v122, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[28:31], v[4:7], a[48:51]\n" \
    "	ds_read_b128 v[76:79], v115 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[28:31], v[8:11], a[84:87]\n" \
    "	s_add_u32 m0, s61, 58368\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v123, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[28:31], v[12:15], a[120:123]\n" \
    "	ds_read_b128 v[80:83], v115 offset:6144\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[32:35], v[0:3], a[16:19]\n" \
    "	s_add_u32 m0, s70, 51200\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v124, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[32:35], v[4:7], a[52:55]\n" \
    "	ds_read_b128 v[84:87], v115 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[32:35], v[8:11], a[88:91]\n" \
    "	s_add_u32 m0, s71, 51200\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v125, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[32:35], v[12:15], a[124:127]\n" \
    "	ds_read_b128 v[88:91], v115 offset:10240\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[36:39], v[0:3], a[20:23]\n" \
    "	s_add_u32 m0, s72, 51200\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v126, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[36:39], v[4:7], a[56:59]\n" \
    "	ds_read_b128 v[92:95], v115 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[36:39], v[8:11], a[92:95]\n" \
    "	s_add_u32 m0, s73, 51200\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v127, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[36:39], v[12:15], a[128:131]\n" \
    "	ds_read_b128 v[96:99], v115 offset:14336\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[40:43], v[0:3], a[24:27]\n" \
    "	s_add_u32 m0, s74, 51200\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v128, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[40:43], v[4:7], a[60:63]\n" \
    "	ds_read_b128 v[100:103], v115 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[40:43], v[8:11], a[96:99]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[40:43], v[12:15], a[132:135]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[44:47], v[0:3], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[44:47], v[4:7], a[64:67]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[44:47], v[8:11], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[44:47], v[12:15], a[136:139]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[48:51], v[0:3], a[32:35]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[48:51], v[4:7], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[48:51], v[8:11], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[48:51], v[12:15], a[140:143]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[68:71], v[52:55], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[68:71], v[56:59], a[36:39]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[68:71], v[60:63], a[72:75]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[68:71], v[64:67], a[108:111]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[72:75], v[52:55], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[72:75], v[56:59], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[72:75], v[60:63], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[72:75], v[64:67], a[112:115]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[76:79], v[52:55], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[76:79], v[56:59], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[76:79], v[60:63], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[76:79], v[64:67], a[116:119]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[80:83], v[52:55], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[80:83], v[56:59], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[80:83], v[60:63], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[80:83], v[64:67], a[120:123]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[84:87], v[52:55], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[84:87], v[56:59], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[84:87], v[60:63], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[84:87], v[64:67], a[124:127]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[88:91], v[52:55], a[20:23]\n" \
    "	s_waitcnt vmcnt(13)\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	s_barrier\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[88:91], v[56:59], a[56:59]\n" \
    "	ds_read_b128 v[16:19], v110 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[88:91], v[60:63], a[92:95]\n" \
    "	ds_read_b128 v[0:3], v104 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[88:91], v[64:67], a[128:131]\n" \
    "	ds_read_b128 v[4:7], v104 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[92:95], v[52:55], a[24:27]\n" \
    "	ds_read_b128 v[8:11], v104 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[92:95], v[56:59], a[60:63]\n" \
    "	ds_read_b128 v[12:15], v104 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[92:95], v[60:63], a[96:99]\n" \
    "	ds_read_b128 v[20:23], v110 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[92:95], v[64:67], a[132:135]\n" \
    "	ds_read_b128 v[24:27], v110 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[96:99], v[52:55], a[28:31]\n" \
    "	ds_read_b128 v[28:31], v110 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[96:99], v[56:59], a[64:67]\n" \
    "	ds_read_b128 v[32:35], v110 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[96:99], v[60:63], a[100:103]\n" \
    "	ds_read_b128 v[36:39], v110 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[96:99], v[64:67], a[136:139]\n" \
    "	ds_read_b128 v[40:43], v110 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[100:103], v[52:55], a[32:35]\n" \
    "	ds_read_b128 v[44:47], v110 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[100:103], v[56:59], a[68:71]\n" \
    "	ds_read_b128 v[48:51], v110 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[100:103], v[60:63], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[100:103], v[64:67], a[140:143]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[16:19], v[0:3], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[16:19], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[68:71], v111 offset:0\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[16:19], v[8:11], a[72:75]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[16:19], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[52:55], v105 offset:0\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[20:23], v[0:3], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[20:23], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[56:59], v105 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[20:23], v[8:11], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[20:23], v[12:15], a[112:115]\n" \
    "	ds_read_b128 v[60:63], v105 offset:4096\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[24:27], v[0:3], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[24:27], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[64:67], v105 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[24:27], v[8:11], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[24:27], v[12:15], a[116:119]\n" \
    "	ds_read_b128 v[72:75], v111 offset:2048\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[28:31], v[0:3], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[28:31], v[4:7], a[48:51]\n" \
    "	ds_read_b128 v[76:79], v111 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[28:31], v[8:11], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[28:31], v[12:15], a[120:123]\n" \
    "	ds_read_b128 v[80:83], v111 offset:6144\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[32:35], v[0:3], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[32:35], v[4:7], a[52:55]\n" \
    "	ds_read_b128 v[84:87], v111 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[32:35], v[8:11], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[32:35], v[12:15], a[124:127]\n" \
    "	ds_read_b128 v[88:91], v111 offset:10240\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[36:39], v[0:3], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[36:39], v[4:7], a[56:59]\n" \
    "	ds_read_b128 v[92:95], v111 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[36:39], v[8:11], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[36:39], v[12:15], a[128:131]\n" \
    "	ds_read_b128 v[96:99], v111 offset:14336\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[40:43], v[0:3], a[24:27]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[40:43], v[4:7], a[60:63]\n" \
    "	ds_read_b128 v[100:103], v111 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[40:43], v[8:11], a[96:99]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[40:43], v[12:15], a[132:135]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[44:47], v[0:3], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[44:47], v[4:7], a[64:67]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[44:47], v[8:11], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[44:47], v[12:15], a[136:139]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[48:51], v[0:3], a[32:35]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[48:51], v[4:7], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[48:51], v[8:11], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[48:51], v[12:15], a[140:143]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[68:71], v[52:55], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[68:71], v[56:59], a[36:39]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[68:71], v[60:63], a[72:75]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[68:71], v[64:67], a[108:111]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[72:75], v[52:55], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[72:75], v[56:59], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[72:75], v[60:63], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[72:75], v[64:67], a[112:115]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[76:79], v[52:55], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[76:79], v[56:59], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[76:79], v[60:63], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[76:79], v[64:67], a[116:119]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[80:83], v[52:55], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[80:83], v[56:59], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[80:83], v[60:63], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[80:83], v[64:67], a[120:123]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[84:87], v[52:55], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[84:87], v[56:59], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[84:87], v[60:63], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[84:87], v[64:67], a[124:127]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[88:91], v[52:55], a[20:23]\n" \
    "	s_waitcnt vmcnt(0)\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	s_barrier\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[88:91], v[56:59], a[56:59]\n" \
    "	ds_read_b128 v[16:19], v112 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[88:91], v[60:63], a[92:95]\n" \
    "	ds_read_b128 v[0:3], v106 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[88:91], v[64:67], a[128:131]\n" \
    "	ds_read_b128 v[4:7], v106 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[92:95], v[52:55], a[24:27]\n" \
    "	ds_read_b128 v[8:11], v106 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[92:95], v[56:59], a[60:63]\n" \
    "	ds_read_b128 v[12:15], v106 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[92:95], v[60:63], a[96:99]\n" \
    "	ds_read_b128 v[20:23], v112 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[92:95], v[64:67], a[132:135]\n" \
    "	ds_read_b128 v[24:27], v112 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[96:99], v[52:55], a[28:31]\n" \
    "	ds_read_b128 v[28:31], v112 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[96:99], v[56:59], a[64:67]\n" \
    "	ds_read_b128 v[32:35], v112 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[96:99], v[60:63], a[100:103]\n" \
    "	ds_read_b128 v[36:39], v112 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[96:99], v[64:67], a[136:139]\n" \
    "	ds_read_b128 v[40:43], v112 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[100:103], v[52:55], a[32:35]\n" \
    "	ds_read_b128 v[44:47], v112 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[100:103], v[56:59], a[68:71]\n" \
    "	ds_read_b128 v[48:51], v112 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[100:103], v[60:63], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[100:103], v[64:67], a[140:143]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[16:19], v[0:3], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[16:19], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[68:71], v113 offset:0\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[16:19], v[8:11], a[72:75]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[16:19], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[52:55], v107 offset:0\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[20:23], v[0:3], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[20:23], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[56:59], v107 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[20:23], v[8:11], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[20:23], v[12:15], a[112:115]\n" \
    "	ds_read_b128 v[60:63], v107 offset:4096\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[24:27], v[0:3], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[24:27], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[64:67], v107 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[24:27], v[8:11], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[24:27], v[12:15], a[116:119]\n" \
    "	ds_read_b128 v[72:75], v113 offset:2048\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[28:31], v[0:3], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[28:31], v[4:7], a[48:51]\n" \
    "	ds_read_b128 v[76:79], v113 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[28:31], v[8:11], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[28:31], v[12:15], a[120:123]\n" \
    "	ds_read_b128 v[80:83], v113 offset:6144\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[32:35], v[0:3], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[32:35], v[4:7], a[52:55]\n" \
    "	ds_read_b128 v[84:87], v113 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[32:35], v[8:11], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[32:35], v[12:15], a[124:127]\n" \
    "	ds_read_b128 v[88:91], v113 offset:10240\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[36:39], v[0:3], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[36:39], v[4:7], a[56:59]\n" \
    "	ds_read_b128 v[92:95], v113 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[36:39], v[8:11], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[36:39], v[12:15], a[128:131]\n" \
    "	ds_read_b128 v[96:99], v113 offset:14336\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[40:43], v[0:3], a[24:27]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[40:43], v[4:7], a[60:63]\n" \
    "	ds_read_b128 v[100:103], v113 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[40:43], v[8:11], a[96:99]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[40:43], v[12:15], a[132:135]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[44:47], v[0:3], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[44:47], v[4:7], a[64:67]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[44:47], v[8:11], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[44:47], v[12:15], a[136:139]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[48:51], v[0:3], a[32:35]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[48:51], v[4:7], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[48:51], v[8:11], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[48:51], v[12:15], a[140:143]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[68:71], v[52:55], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[68:71], v[56:59], a[36:39]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[68:71], v[60:63], a[72:75]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[68:71], v[64:67], a[108:111]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[72:75], v[52:55], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[72:75], v[56:59], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[72:75], v[60:63], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[72:75], v[64:67], a[112:115]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[76:79], v[52:55], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[76:79], v[56:59], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[76:79], v[60:63], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[76:79], v[64:67], a[116:119]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[80:83], v[52:55], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[80:83], v[56:59], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[80:83], v[60:63], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[80:83], v[64:67], a[120:123]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[84:87], v[52:55], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[84:87], v[56:59], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[84:87], v[60:63], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[84:87], v[64:67], a[124:127]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[88:91], v[52:55], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[88:91], v[56:59], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[88:91], v[60:63], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[88:91], v[64:67], a[128:131]\n" \
    "	s_waitcnt lgkmcnt(2)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[92:95], v[52:55], a[24:27]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[92:95], v[56:59], a[60:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[92:95], v[60:63], a[96:99]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[92:95], v[64:67], a[132:135]\n" \
    "	s_waitcnt lgkmcnt(1)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[96:99], v[52:55], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[96:99], v[56:59], a[64:67]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[96:99], v[60:63], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[96:99], v[64:67], a[136:139]\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[100:103], v[52:55], a[32:35]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[100:103], v[56:59], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[100:103], v[60:63], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[100:103], v[64:67], a[140:143]\n" \
    "DONE_%=:\n" \
    "	s_nop 15\n" \
    "	s_barrier\n" \
    "	s_mov_b32 m0, s66\n" \
      : /* accumulators stay in AGPRs */ \
      : [ap] "s"(ap), [wp] "s"(wp), [rsa] "s"(rsa), [rsw] "s"(rsw), [ra] "s"(ra), [rw] "s"(rw), [trips] "s"(trips), [rem] "s"(rem), [lds] "s"(lds), [wave] "s"(wave), [zero] "s"(zero) \
      : "memory", "vcc", "scc", "v0", "v1", "v2", "v3", "v4", "v5", "v6", "v7", "v8", "v9", "v10", "v11", "v12", "v13", "v14", "v15", "v16", "v17", "v18", "v19", "v20", "v21", "v22", "v23", "v24", "v25", "v26", "v27", "v28", "v29", "v30", "v31", "v32", "v33", "v34", "v35", "v36", "v37", "v38", "v39", "v40", "v41", "v42", "v43", "v44", "v45", "v46", "v47", "v48", "v49", "v50", "v51", "v52", "v53", "v54", "v55", "v56", "v57", "v58", "v59", "v60", "v61", "v62", "v63", "v64", "v65", "v66", "v67", "v68", "v69", "v70", "v71", "v72", "v73", "v74", "v75", "v76", "v77", "v78", "v79", "v80", "v81", "v82", "v83", "v84", "v85", "v86", "v87", "v88", "v89", "v90", "v91", "v92", "v93", "v94", "v95", "v96", "v97", "v98", "v99", "v100", "v101", "v102", "v103", "v104", "v105", "v106", "v107", "v108", "v109", "v110", "v111", "v112", "v113", "v114", "v115", "v116", "v117", "v118", "v119", "v120", "v121", "v122", "v123", "v124", "v125", "v126", "v127", "v128", "v129", "v130", "v131", "v132", "v133", "v134", "v135", "v136", "v137", "v138", "v139", "a0", "a1", "a2", "a3", "a4", "a5", "a6", "a7", "a8", "a9", "a10", "a11", "a12", "a13", "a14", "a15", "a16", "a17", "a18", "a19", "a20", "a21", "a22", "a23", "a24", "a25", "a26", "a27", "a28", "a29", "a30", "a31", "a32", "a33", "a34", "a35", "a36", "a37", "a38", "a39", "a40", "a41", "a42", "a43", "a44", "a45", "a46", "a47", "a48", "a49", "a50", "a51", "a52", "a53", "a54", "a55", "a56", "a57", "a58", "a59", "a60", "a61", "a62", "a63", "a64", "a65", "a66", "a67", "a68", "a69", "a70", "a71", "a72", "a73", "a74", "a75", "a76", "a77", "a78", "a79", "a80", "a81", "a82", "a83", "a84", "a85", "a86", "a87", "a88", "a89", "a90", "a91", "a92", "a93", "a94", "a95", "a96", "a97", "a98", "a99", "a100", "a101", "a102", "a103", "a104", "a105", "a106", "a107", "a108", "a109", "a110", "a111", "a112", "a113", "a114", "a115", "a116", "a117", "a118", "a119", "a120", "a121", "a122", "a123", "a124", "a125", "a126", "a127", "a128", "a129", "a130", "a131", "a132", "a133", "a134", "a135", "a136", "a137", "a138", "a139", "a140", "a141", "a142", "a143", "a144", "a145", "a146", "a147", "a148", "a149", "a150", "a151", "a152", "a153", "a154", "a155", "a156", "a157", "a158", "a159", "a160", "a161", "a162", "a163", "a164", "a165", "a166", "a167", "a168", "a169", "a170", "a171", "a172", "a173", "a174", "a175", "a176", "a177", "a178", "a179", "a180", "a181", "a182", "a183", "a184", "a185", "a186", "a187", "a188", "a189", "a190", "a191", "a192", "a193", "a194", "a195", "a196", "a197", "a198", "a199", "a200", "a201", "a202", "a203", "a204", "a205", "a206", "a207", "a208", "a209", "a210", "a211", "a212", "a213", "a214", "a215", "a216", "a217", "a218", "a219", "a220", "a221", "a222", "a223", "a224", "a225", "a226", "a227", "a228", "a229", "a230", "a231", "a232", "a233", "a234", "a235", "a236", "a237", "a238", "a239", "a240", "a241", "a242", "a243", "a244", "a245", "a246", "a247", "a248", "a249", "a250", "a251", "a252", "a253", "a254", "a255", "s60", "s61", "s62", "s63", "s64", "s65", "s66", "s67", "s68", "s69", "s70", "s71", "s72", "s73", "s74", "s75")

#define GEMM_I8_PERIOD_288 2  // stages per trip, and the fewest the loop takes
#define GEMM_I8_ASM_288(ap, wp, rsa, rsw, ra, rw, trips, rem, lds, wave, zero, c8) \
  asm volatile( \
    "	s_mov_b32 s66, m0\n" \
    "	v_mbcnt_lo_u32_b32 v161, -1, 0\n" \
    "	v_mbcnt_hi_u32_b32 v161, -1, v161\n" \
    "	v_and_b32_e32 v162, 15, v161\n" \
    "	v_lshrrev_b32_e32 v163, 4, v161\n" \
    "	v_bfe_u32 v164, v161, 1, 3\n" \
    "	s_and_b32 s67, %[wave], 1\n" \
    "	s_lshr_b32 s68, %[wave], 1\n" \
    "	s_lshl_b32 s67, s67, 14\n" \
    "	s_mul_i32 s68, s68, 18432\n" \
    "	v_lshlrev_b32_e32 v165, 7, v162\n" \
    "	v_add_u32_e32 v165, %[lds], v165\n" \
    "	v_add_u32_e32 v166, 0, v163\n" \
    "	v_xor_b32_e32 v166, v166, v164\n" \
    "	v_lshl_add_u32 v166, v166, 4, v165\n" \
    "	v_add_u32_e32 v136, s67, v166\n" \
    "	v_add_u32_e32 v140, s68, v166\n" \
    "	v_add_u32_e32 v140, 32768, v140\n" \
    "	v_add_u32_e32 v166, 4, v163\n" \
    "	v_xor_b32_e32 v166, v166, v164\n" \
    "	v_lshl_add_u32 v166, v166, 4, v165\n" \
    "	v_add_u32_e32 v137, s67, v166\n" \
    "	v_add_u32_e32 v141, s68, v166\n" \
    "	v_add_u32_e32 v141, 32768, v141\n" \
    "	v_add_u32_e32 v166, 0, v163\n" \
    "	v_xor_b32_e32 v166, v166, v164\n" \
    "	v_lshl_add_u32 v166, v166, 4, v165\n" \
    "	v_add_u32_e32 v138, s67, v166\n" \
    "	v_add_u32_e32 v142, s68, v166\n" \
    "	v_add_u32_e32 v138, 69632, v138\n" \
    "	v_add_u32_e32 v142, 102400, v142\n" \
    "	v_add_u32_e32 v166, 4, v163\n" \
    "	v_xor_b32_e32 v166, v166, v164\n" \
    "	v_lshl_add_u32 v166, v166, 4, v165\n" \
    "	v_add_u32_e32 v139, s67, v166\n" \
    "	v_add_u32_e32 v143, s68, v166\n" \
    "	v_add_u32_e32 v139, 69632, v139\n" \
    "	v_add_u32_e32 v143, 102400, v143\n" \
    "	v_lshrrev_b32_e32 v165, 3, v161\n" \
    "	v_and_b32_e32 v166, 7, v161\n" \
    "	s_mul_i32 s67, %[wave], 64\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 0\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v167, s68, v163\n" \
    "	v_xor_b32_e32 v167, v167, v166\n" \
    "	v_lshlrev_b32_e32 v167, 4, v167\n" \
    "	v_add_u32_e32 v168, 0, v165\n" \
    "	v_add_u32_e32 v168, s67, v168\n" \
    "	v_min_u32_e32 v168, %[ra], v168\n" \
    "	v_mad_u32_u24 v144, v168, %[rsa], v167\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 4\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v167, s68, v163\n" \
    "	v_xor_b32_e32 v167, v167, v166\n" \
    "	v_lshlrev_b32_e32 v167, 4, v167\n" \
    "	v_add_u32_e32 v168, 8, v165\n" \
    "	v_add_u32_e32 v168, s67, v168\n" \
    "	v_min_u32_e32 v168, %[ra], v168\n" \
    "	v_mad_u32_u24 v145, v168, %[rsa], v167\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 8\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v167, s68, v163\n" \
    "	v_xor_b32_e32 v167, v167, v166\n" \
    "	v_lshlrev_b32_e32 v167, 4, v167\n" \
    "	v_add_u32_e32 v168, 16, v165\n" \
    "	v_add_u32_e32 v168, s67, v168\n" \
    "	v_min_u32_e32 v168, %[ra], v168\n" \
    "	v_mad_u32_u24 v146, v168, %[rsa], v167\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 12\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v167, s68, v163\n" \
    "	v_xor_b32_e32 v167, v167, v166\n" \
    "	v_lshlrev_b32_e32 v167, 4, v167\n" \
    "	v_add_u32_e32 v168, 24, v165\n" \
    "	v_add_u32_e32 v168, s67, v168\n" \
    "	v_min_u32_e32 v168, %[ra], v168\n" \
    "	v_mad_u32_u24 v147, v168, %[rsa], v167\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 16\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v167, s68, v163\n" \
    "	v_xor_b32_e32 v167, v167, v166\n" \
    "	v_lshlrev_b32_e32 v167, 4, v167\n" \
    "	v_add_u32_e32 v168, 32, v165\n" \
    "	v_add_u32_e32 v168, s67, v168\n" \
    "	v_min_u32_e32 v168, %[ra], v168\n" \
    "	v_mad_u32_u24 v148, v168, %[rsa], v167\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 20\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v167, s68, v163\n" \
    "	v_xor_b32_e32 v167, v167, v166\n" \
    "	v_lshlrev_b32_e32 v167, 4, v167\n" \
    "	v_add_u32_e32 v168, 40, v165\n" \
    "	v_add_u32_e32 v168, s67, v168\n" \
    "	v_min_u32_e32 v168, %[ra], v168\n" \
    "	v_mad_u32_u24 v149, v168, %[rsa], v167\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 24\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v167, s68, v163\n" \
    "	v_xor_b32_e32 v167, v167, v166\n" \
    "	v_lshlrev_b32_e32 v167, 4, v167\n" \
    "	v_add_u32_e32 v168, 48, v165\n" \
    "	v_add_u32_e32 v168, s67, v168\n" \
    "	v_min_u32_e32 v168, %[ra], v168\n" \
    "	v_mad_u32_u24 v150, v168, %[rsa], v167\n" \
    "	s_mul_i32 s68, %[wave], 32\n" \
    "	s_add_u32 s68, s68, 28\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v167, s68, v163\n" \
    "	v_xor_b32_e32 v167, v167, v166\n" \
    "	v_lshlrev_b32_e32 v167, 4, v167\n" \
    "	v_add_u32_e32 v168, 56, v165\n" \
    "	v_add_u32_e32 v168, s67, v168\n" \
    "	v_min_u32_e32 v168, %[ra], v168\n" \
    "	v_mad_u32_u24 v151, v168, %[rsa], v167\n" \
    "	s_mul_i32 s67, %[wave], 72\n" \
    "	s_mul_i32 s68, %[wave], 36\n" \
    "	s_add_u32 s68, s68, 0\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v167, s68, v163\n" \
    "	v_xor_b32_e32 v167, v167, v166\n" \
    "	v_lshlrev_b32_e32 v167, 4, v167\n" \
    "	v_add_u32_e32 v168, 0, v165\n" \
    "	v_add_u32_e32 v168, s67, v168\n" \
    "	v_min_u32_e32 v168, %[rw], v168\n" \
    "	v_mad_u32_u24 v152, v168, %[rsw], v167\n" \
    "	s_mul_i32 s68, %[wave], 36\n" \
    "	s_add_u32 s68, s68, 4\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v167, s68, v163\n" \
    "	v_xor_b32_e32 v167, v167, v166\n" \
    "	v_lshlrev_b32_e32 v167, 4, v167\n" \
    "	v_add_u32_e32 v168, 8, v165\n" \
    "	v_add_u32_e32 v168, s67, v168\n" \
    "	v_min_u32_e32 v168, %[rw], v168\n" \
    "	v_mad_u32_u24 v153, v168, %[rsw], v167\n" \
    "	s_mul_i32 s68, %[wave], 36\n" \
    "	s_add_u32 s68, s68, 8\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v167, s68, v163\n" \
    "	v_xor_b32_e32 v167, v167, v166\n" \
    "	v_lshlrev_b32_e32 v167, 4, v167\n" \
    "	v_add_u32_e32 v168, 16, v165\n" \
    "	v_add_u32_e32 v168, s67, v168\n" \
    "	v_min_u32_e32 v168, %[rw], v168\n" \
    "	v_mad_u32_u24 v154, v168, %[rsw], v167\n" \
    "	s_mul_i32 s68, %[wave], 36\n" \
    "	s_add_u32 s68, s68, 12\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v167, s68, v163\n" \
    "	v_xor_b32_e32 v167, v167, v166\n" \
    "	v_lshlrev_b32_e32 v167, 4, v167\n" \
    "	v_add_u32_e32 v168, 24, v165\n" \
    "	v_add_u32_e32 v168, s67, v168\n" \
    "	v_min_u32_e32 v168, %[rw], v168\n" \
    "	v_mad_u32_u24 v155, v168, %[rsw], v167\n" \
    "	s_mul_i32 s68, %[wave], 36\n" \
    "	s_add_u32 s68, s68, 16\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v167, s68, v163\n" \
    "	v_xor_b32_e32 v167, v167, v166\n" \
    "	v_lshlrev_b32_e32 v167, 4, v167\n" \
    "	v_add_u32_e32 v168, 32, v165\n" \
    "	v_add_u32_e32 v168, s67, v168\n" \
    "	v_min_u32_e32 v168, %[rw], v168\n" \
    "	v_mad_u32_u24 v156, v168, %[rsw], v167\n" \
    "	s_mul_i32 s68, %[wave], 36\n" \
    "	s_add_u32 s68, s68, 20\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v167, s68, v163\n" \
    "	v_xor_b32_e32 v167, v167, v166\n" \
    "	v_lshlrev_b32_e32 v167, 4, v167\n" \
    "	v_add_u32_e32 v168, 40, v165\n" \
    "	v_add_u32_e32 v168, s67, v168\n" \
    "	v_min_u32_e32 v168, %[rw], v168\n" \
    "	v_mad_u32_u24 v157, v168, %[rsw], v167\n" \
    "	s_mul_i32 s68, %[wave], 36\n" \
    "	s_add_u32 s68, s68, 24\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v167, s68, v163\n" \
    "	v_xor_b32_e32 v167, v167, v166\n" \
    "	v_lshlrev_b32_e32 v167, 4, v167\n" \
    "	v_add_u32_e32 v168, 48, v165\n" \
    "	v_add_u32_e32 v168, s67, v168\n" \
    "	v_min_u32_e32 v168, %[rw], v168\n" \
    "	v_mad_u32_u24 v158, v168, %[rsw], v167\n" \
    "	s_mul_i32 s68, %[wave], 36\n" \
    "	s_add_u32 s68, s68, 28\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v167, s68, v163\n" \
    "	v_xor_b32_e32 v167, v167, v166\n" \
    "	v_lshlrev_b32_e32 v167, 4, v167\n" \
    "	v_add_u32_e32 v168, 56, v165\n" \
    "	v_add_u32_e32 v168, s67, v168\n" \
    "	v_min_u32_e32 v168, %[rw], v168\n" \
    "	v_mad_u32_u24 v159, v168, %[rsw], v167\n" \
    "	s_mul_i32 s68, %[wave], 36\n" \
    "	s_add_u32 s68, s68, 32\n" \
    "	s_and_b32 s68, s68, 7\n" \
    "	v_or_b32_e32 v167, s68, v163\n" \
    "	v_xor_b32_e32 v167, v167, v166\n" \
    "	v_lshlrev_b32_e32 v167, 4, v167\n" \
    "	v_add_u32_e32 v168, 64, v165\n" \
    "	v_add_u32_e32 v168, s67, v168\n" \
    "	v_min_u32_e32 v168, %[rw], v168\n" \
    "	v_mad_u32_u24 v160, v168, %[rsw], v167\n" \
    "	s_lshl_b32 s67, %[wave], 13\n" \
    "	s_add_u32 s61, %[lds], s67\n" \
    "	s_mul_i32 s67, %[wave], 9216\n" \
    "	s_add_u32 s69, %[lds], s67\n" \
    "	s_mov_b64 s[62:63], %[ap]\n" \
    "	s_mov_b64 s[64:65], %[wp]\n" \
    "	s_cmp_eq_u32 %[zero], 0\n" \
    "	s_cbranch_scc1 KEEP_%=\n" \
    "	v_accvgpr_write_b32 a0, 0\n" \
    "	v_accvgpr_write_b32 a1, 0\n" \
    "	v_accvgpr_write_b32 a2, 0\n" \
    "	v_accvgpr_write_b32 a3, 0\n" \
    "	v_accvgpr_write_b32 a4, 0\n" \
    "	v_accvgpr_write_b32 a5, 0\n" \
    "	v_accvgpr_write_b32 a6, 0\n" \
    "	v_accvgpr_write_b32 a7, 0\n" \
    "	v_accvgpr_write_b32 a8, 0\n" \
    "	v_accvgpr_write_b32 a9, 0\n" \
    "	v_accvgpr_write_b32 a10, 0\n" \
    "	v_accvgpr_write_b32 a11, 0\n" \
    "	v_accvgpr_write_b32 a12, 0\n" \
    "	v_accvgpr_write_b32 a13, 0\n" \
    "	v_accvgpr_write_b32 a14, 0\n" \
    "	v_accvgpr_write_b32 a15, 0\n" \
    "	v_accvgpr_write_b32 a16, 0\n" \
    "	v_accvgpr_write_b32 a17, 0\n" \
    "	v_accvgpr_write_b32 a18, 0\n" \
    "	v_accvgpr_write_b32 a19, 0\n" \
    "	v_accvgpr_write_b32 a20, 0\n" \
    "	v_accvgpr_write_b32 a21, 0\n" \
    "	v_accvgpr_write_b32 a22, 0\n" \
    "	v_accvgpr_write_b32 a23, 0\n" \
    "	v_accvgpr_write_b32 a24, 0\n" \
    "	v_accvgpr_write_b32 a25, 0\n" \
    "	v_accvgpr_write_b32 a26, 0\n" \
    "	v_accvgpr_write_b32 a27, 0\n" \
    "	v_accvgpr_write_b32 a28, 0\n" \
    "	v_accvgpr_write_b32 a29, 0\n" \
    "	v_accvgpr_write_b32 a30, 0\n" \
    "	v_accvgpr_write_b32 a31, 0\n" \
    "	v_accvgpr_write_b32 a32, 0\n" \
    "	v_accvgpr_write_b32 a33, 0\n" \
    "	v_accvgpr_write_b32 a34, 0\n" \
    "	v_accvgpr_write_b32 a35, 0\n" \
    "	v_accvgpr_write_b32 a36, 0\n" \
    "	v_accvgpr_write_b32 a37, 0\n" \
    "	v_accvgpr_write_b32 a38, 0\n" \
    "	v_accvgpr_write_b32 a39, 0\n" \
    "	v_accvgpr_write_b32 a40, 0\n" \
    "	v_accvgpr_write_b32 a41, 0\n" \
    "	v_accvgpr_write_b32 a42, 0\n" \
    "	v_accvgpr_write_b32 a43, 0\n" \
    "	v_accvgpr_write_b32 a44, 0\n" \
    "	v_accvgpr_write_b32 a45, 0\n" \
    "	v_accvgpr_write_b32 a46, 0\n" \
    "	v_accvgpr_write_b32 a47, 0\n" \
    "	v_accvgpr_write_b32 a48, 0\n" \
    "	v_accvgpr_write_b32 a49, 0\n" \
    "	v_accvgpr_write_b32 a50, 0\n" \
    "	v_accvgpr_write_b32 a51, 0\n" \
    "	v_accvgpr_write_b32 a52, 0\n" \
    "	v_accvgpr_write_b32 a53, 0\n" \
    "	v_accvgpr_write_b32 a54, 0\n" \
    "	v_accvgpr_write_b32 a55, 0\n" \
    "	v_accvgpr_write_b32 a56, 0\n" \
    "	v_accvgpr_write_b32 a57, 0\n" \
    "	v_accvgpr_write_b32 a58, 0\n" \
    "	v_accvgpr_write_b32 a59, 0\n" \
    "	v_accvgpr_write_b32 a60, 0\n" \
    "	v_accvgpr_write_b32 a61, 0\n" \
    "	v_accvgpr_write_b32 a62, 0\n" \
    "	v_accvgpr_write_b32 a63, 0\n" \
    "	v_accvgpr_write_b32 a64, 0\n" \
    "	v_accvgpr_write_b32 a65, 0\n" \
    "	v_accvgpr_write_b32 a66, 0\n" \
    "	v_accvgpr_write_b32 a67, 0\n" \
    "	v_accvgpr_write_b32 a68, 0\n" \
    "	v_accvgpr_write_b32 a69, 0\n" \
    "	v_accvgpr_write_b32 a70, 0\n" \
    "	v_accvgpr_write_b32 a71, 0\n" \
    "	v_accvgpr_write_b32 a72, 0\n" \
    "	v_accvgpr_write_b32 a73, 0\n" \
    "	v_accvgpr_write_b32 a74, 0\n" \
    "	v_accvgpr_write_b32 a75, 0\n" \
    "	v_accvgpr_write_b32 a76, 0\n" \
    "	v_accvgpr_write_b32 a77, 0\n" \
    "	v_accvgpr_write_b32 a78, 0\n" \
    "	v_accvgpr_write_b32 a79, 0\n" \
    "	v_accvgpr_write_b32 a80, 0\n" \
    "	v_accvgpr_write_b32 a81, 0\n" \
    "	v_accvgpr_write_b32 a82, 0\n" \
    "	v_accvgpr_write_b32 a83, 0\n" \
    "	v_accvgpr_write_b32 a84, 0\n" \
    "	v_accvgpr_write_b32 a85, 0\n" \
    "	v_accvgpr_write_b32 a86, 0\n" \
    "	v_accvgpr_write_b32 a87, 0\n" \
    "	v_accvgpr_write_b32 a88, 0\n" \
    "	v_accvgpr_write_b32 a89, 0\n" \
    "	v_accvgpr_write_b32 a90, 0\n" \
    "	v_accvgpr_write_b32 a91, 0\n" \
    "	v_accvgpr_write_b32 a92, 0\n" \
    "	v_accvgpr_write_b32 a93, 0\n" \
    "	v_accvgpr_write_b32 a94, 0\n" \
    "	v_accvgpr_write_b32 a95, 0\n" \
    "	v_accvgpr_write_b32 a96, 0\n" \
    "	v_accvgpr_write_b32 a97, 0\n" \
    "	v_accvgpr_write_b32 a98, 0\n" \
    "	v_accvgpr_write_b32 a99, 0\n" \
    "	v_accvgpr_write_b32 a100, 0\n" \
    "	v_accvgpr_write_b32 a101, 0\n" \
    "	v_accvgpr_write_b32 a102, 0\n" \
    "	v_accvgpr_write_b32 a103, 0\n" \
    "	v_accvgpr_write_b32 a104, 0\n" \
    "	v_accvgpr_write_b32 a105, 0\n" \
    "	v_accvgpr_write_b32 a106, 0\n" \
    "	v_accvgpr_write_b32 a107, 0\n" \
    "	v_accvgpr_write_b32 a108, 0\n" \
    "	v_accvgpr_write_b32 a109, 0\n" \
    "	v_accvgpr_write_b32 a110, 0\n" \
    "	v_accvgpr_write_b32 a111, 0\n" \
    "	v_accvgpr_write_b32 a112, 0\n" \
    "	v_accvgpr_write_b32 a113, 0\n" \
    "	v_accvgpr_write_b32 a114, 0\n" \
    "	v_accvgpr_write_b32 a115, 0\n" \
    "	v_accvgpr_write_b32 a116, 0\n" \
    "	v_accvgpr_write_b32 a117, 0\n" \
    "	v_accvgpr_write_b32 a118, 0\n" \
    "	v_accvgpr_write_b32 a119, 0\n" \
    "	v_accvgpr_write_b32 a120, 0\n" \
    "	v_accvgpr_write_b32 a121, 0\n" \
    "	v_accvgpr_write_b32 a122, 0\n" \
    "	v_accvgpr_write_b32 a123, 0\n" \
    "	v_accvgpr_write_b32 a124, 0\n" \
    "	v_accvgpr_write_b32 a125, 0\n" \
    "	v_accvgpr_write_b32 a126, 0\n" \
    "	v_accvgpr_write_b32 a127, 0\n" \
    "	v_accvgpr_write_b32 a128, 0\n" \
    "	v_accvgpr_write_b32 a129, 0\n" \
    "	v_accvgpr_write_b32 a130, 0\n" \
    "	v_accvgpr_write_b32 a131, 0\n" \
    "	v_accvgpr_write_b32 a132, 0\n" \
    "	v_accvgpr_write_b32 a133, 0\n" \
    "	v_accvgpr_write_b32 a134, 0\n" \
    "	v_accvgpr_write_b32 a135, 0\n" \
    "	v_accvgpr_write_b32 a136, 0\n" \
    "	v_accvgpr_write_b32 a137, 0\n" \
    "	v_accvgpr_write_b32 a138, 0\n" \
    "	v_accvgpr_write_b32 a139, 0\n" \
    "	v_accvgpr_write_b32 a140, 0\n" \
    "	v_accvgpr_write_b32 a141, 0\n" \
    "	v_accvgpr_write_b32 a142, 0\n" \
    "	v_accvgpr_write_b32 a143, 0\n" \
    "	v_accvgpr_write_b32 a144, 0\n" \
    "	v_accvgpr_write_b32 a145, 0\n" \
    "	v_accvgpr_write_b32 a146, 0\n" \
    "	v_accvgpr_write_b32 a147, 0\n" \
    "	v_accvgpr_write_b32 a148, 0\n" \
    "	v_accvgpr_write_b32 a149, 0\n" \
    "	v_accvgpr_write_b32 a150, 0\n" \
    "	v_accvgpr_write_b32 a151, 0\n" \
    "	v_accvgpr_write_b32 a152, 0\n" \
    "	v_accvgpr_write_b32 a153, 0\n" \
    "	v_accvgpr_write_b32 a154, 0\n" \
    "	v_accvgpr_write_b32 a155, 0\n" \
    "	v_accvgpr_write_b32 a156, 0\n" \
    "	v_accvgpr_write_b32 a157, 0\n" \
    "	v_accvgpr_write_b32 a158, 0\n" \
    "	v_accvgpr_write_b32 a159, 0\n" \
    "	v_accvgpr_write_b32 a160, 0\n" \
    "	v_accvgpr_write_b32 a161, 0\n" \
    "	v_accvgpr_write_b32 a162, 0\n" \
    "	v_accvgpr_write_b32 a163, 0\n" \
    "	v_accvgpr_write_b32 a164, 0\n" \
    "	v_accvgpr_write_b32 a165, 0\n" \
    "	v_accvgpr_write_b32 a166, 0\n" \
    "	v_accvgpr_write_b32 a167, 0\n" \
    "	v_accvgpr_write_b32 a168, 0\n" \
    "	v_accvgpr_write_b32 a169, 0\n" \
    "	v_accvgpr_write_b32 a170, 0\n" \
    "	v_accvgpr_write_b32 a171, 0\n" \
    "	v_accvgpr_write_b32 a172, 0\n" \
    "	v_accvgpr_write_b32 a173, 0\n" \
    "	v_accvgpr_write_b32 a174, 0\n" \
    "	v_accvgpr_write_b32 a175, 0\n" \
    "	v_accvgpr_write_b32 a176, 0\n" \
    "	v_accvgpr_write_b32 a177, 0\n" \
    "	v_accvgpr_write_b32 a178, 0\n" \
    "	v_accvgpr_write_b32 a179, 0\n" \
    "	v_accvgpr_write_b32 a180, 0\n" \
    "	v_accvgpr_write_b32 a181, 0\n" \
    "	v_accvgpr_write_b32 a182, 0\n" \
    "	v_accvgpr_write_b32 a183, 0\n" \
    "	v_accvgpr_write_b32 a184, 0\n" \
    "	v_accvgpr_write_b32 a185, 0\n" \
    "	v_accvgpr_write_b32 a186, 0\n" \
    "	v_accvgpr_write_b32 a187, 0\n" \
    "	v_accvgpr_write_b32 a188, 0\n" \
    "	v_accvgpr_write_b32 a189, 0\n" \
    "	v_accvgpr_write_b32 a190, 0\n" \
    "	v_accvgpr_write_b32 a191, 0\n" \
    "	v_accvgpr_write_b32 a192, 0\n" \
    "	v_accvgpr_write_b32 a193, 0\n" \
    "	v_accvgpr_write_b32 a194, 0\n" \
    "	v_accvgpr_write_b32 a195, 0\n" \
    "	v_accvgpr_write_b32 a196, 0\n" \
    "	v_accvgpr_write_b32 a197, 0\n" \
    "	v_accvgpr_write_b32 a198, 0\n" \
    "	v_accvgpr_write_b32 a199, 0\n" \
    "	v_accvgpr_write_b32 a200, 0\n" \
    "	v_accvgpr_write_b32 a201, 0\n" \
    "	v_accvgpr_write_b32 a202, 0\n" \
    "	v_accvgpr_write_b32 a203, 0\n" \
    "	v_accvgpr_write_b32 a204, 0\n" \
    "	v_accvgpr_write_b32 a205, 0\n" \
    "	v_accvgpr_write_b32 a206, 0\n" \
    "	v_accvgpr_write_b32 a207, 0\n" \
    "	v_accvgpr_write_b32 a208, 0\n" \
    "	v_accvgpr_write_b32 a209, 0\n" \
    "	v_accvgpr_write_b32 a210, 0\n" \
    "	v_accvgpr_write_b32 a211, 0\n" \
    "	v_accvgpr_write_b32 a212, 0\n" \
    "	v_accvgpr_write_b32 a213, 0\n" \
    "	v_accvgpr_write_b32 a214, 0\n" \
    "	v_accvgpr_write_b32 a215, 0\n" \
    "	v_accvgpr_write_b32 a216, 0\n" \
    "	v_accvgpr_write_b32 a217, 0\n" \
    "	v_accvgpr_write_b32 a218, 0\n" \
    "	v_accvgpr_write_b32 a219, 0\n" \
    "	v_accvgpr_write_b32 a220, 0\n" \
    "	v_accvgpr_write_b32 a221, 0\n" \
    "	v_accvgpr_write_b32 a222, 0\n" \
    "	v_accvgpr_write_b32 a223, 0\n" \
    "	v_accvgpr_write_b32 a224, 0\n" \
    "	v_accvgpr_write_b32 a225, 0\n" \
    "	v_accvgpr_write_b32 a226, 0\n" \
    "	v_accvgpr_write_b32 a227, 0\n" \
    "	v_accvgpr_write_b32 a228, 0\n" \
    "	v_accvgpr_write_b32 a229, 0\n" \
    "	v_accvgpr_write_b32 a230, 0\n" \
    "	v_accvgpr_write_b32 a231, 0\n" \
    "	v_accvgpr_write_b32 a232, 0\n" \
    "	v_accvgpr_write_b32 a233, 0\n" \
    "	v_accvgpr_write_b32 a234, 0\n" \
    "	v_accvgpr_write_b32 a235, 0\n" \
    "	v_accvgpr_write_b32 a236, 0\n" \
    "	v_accvgpr_write_b32 a237, 0\n" \
    "	v_accvgpr_write_b32 a238, 0\n" \
    "	v_accvgpr_write_b32 a239, 0\n" \
    "	v_accvgpr_write_b32 a240, 0\n" \
    "	v_accvgpr_write_b32 a241, 0\n" \
    "	v_accvgpr_write_b32 a242, 0\n" \
    "	v_accvgpr_write_b32 a243, 0\n" \
    "	v_accvgpr_write_b32 a244, 0\n" \
    "	v_accvgpr_write_b32 a245, 0\n" \
    "	v_accvgpr_write_b32 a246, 0\n" \
    "	v_accvgpr_write_b32 a247, 0\n" \
    "	v_accvgpr_write_b32 a248, 0\n" \
    "	v_accvgpr_write_b32 a249, 0\n" \
    "	v_accvgpr_write_b32 a250, 0\n" \
    "	v_accvgpr_write_b32 a251, 0\n" \
    "	v_accvgpr_write_b32 a252, 0\n" \
    "	v_accvgpr_write_b32 a253, 0\n" \
    "	v_accvgpr_write_b32 a254, 0\n" \
    "	v_accvgpr_write_b32 a255, 0\n" \
    "KEEP_%=:\n" \
    "	s_add_u32 m0, s61, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v144, s[62:63]\n" \
    "	s_add_u32 m0, s61, 1024\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v145, s[62:63]\n" \
    "	s_add_u32 m0, s61, 2048\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v146, s[62:63]\n" \
    "	s_add_u32 m0, s61, 3072\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v147, s[62:63]\n" \
    "	s_add_u32 m0, s61, 4096\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v148, s[62:63]\n" \
    "	s_add_u32 m0, s61, 5120\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v149, s[62:63]\n" \
    "	s_add_u32 m0, s61, 6144\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v150, s[62:63]\n" \
    "	s_add_u32 m0, s61, 7168\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v151, s[62:63]\n" \
    "	s_add_u32 m0, s69, 32768\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v152, s[64:65]\n" \
    "	s_add_u32 m0, s69, 33792\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v153, s[64:65]\n" \
    "	s_add_u32 m0, s69, 34816\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v154, s[64:65]\n" \
    "	s_add_u32 m0, s69, 35840\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v155, s[64:65]\n" \
    "	s_add_u32 m0, s69, 36864\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v156, s[64:65]\n" \
    "	s_add_u32 m0, s69, 37888\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v157, s[64:65]\n" \
    "	s_add_u32 m0, s69, 38912\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v158, s[64:65]\n" \
    "	s_add_u32 m0, s69, 39936\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v159, s[64:65]\n" \
    "	s_add_u32 m0, s69, 40960\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v160, s[64:65]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_waitcnt vmcnt(0)\n" \
    "	s_barrier\n" \
    "	ds_read_b128 v[32:35], v140 offset:0\n" \
    "	ds_read_b128 v[0:3], v136 offset:0\n" \
    "	ds_read_b128 v[4:7], v136 offset:2048\n" \
    "	ds_read_b128 v[8:11], v136 offset:4096\n" \
    "	ds_read_b128 v[12:15], v136 offset:6144\n" \
    "	ds_read_b128 v[16:19], v136 offset:8192\n" \
    "	ds_read_b128 v[20:23], v136 offset:10240\n" \
    "	ds_read_b128 v[24:27], v136 offset:12288\n" \
    "	ds_read_b128 v[28:31], v136 offset:14336\n" \
    "	ds_read_b128 v[36:39], v140 offset:2048\n" \
    "	ds_read_b128 v[40:43], v140 offset:4096\n" \
    "	ds_read_b128 v[44:47], v140 offset:6144\n" \
    "	ds_read_b128 v[48:51], v140 offset:8192\n" \
    "	ds_read_b128 v[52:55], v140 offset:10240\n" \
    "	ds_read_b128 v[56:59], v140 offset:12288\n" \
    "	ds_read_b128 v[60:63], v140 offset:14336\n" \
    "	ds_read_b128 v[64:67], v140 offset:16384\n" \
    "	s_mov_b32 s60, %[trips]\n" \
    "	s_cmp_eq_u32 s60, 0\n" \
    "	s_cbranch_scc1 LAST_%=\n" \
    "LOOP_%=:\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[32:35], v[0:3], a[0:3]\n" \
    "	s_add_u32 m0, s61, 69632\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v144, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[32:35], v[4:7], a[32:35]\n" \
    "	ds_read_b128 v[100:103], v141 offset:0\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[32:35], v[8:11], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[32:35], v[12:15], a[96:99]\n" \
    "	ds_read_b128 v[68:71], v137 offset:0\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[32:35], v[16:19], a[128:131]\n" \
    "	s_add_u32 m0, s61, 70656\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v145, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[32:35], v[20:23], a[160:163]\n" \
    "	ds_read_b128 v[72:75], v137 offset:2048\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[32:35], v[24:27], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[32:35], v[28:31], a[224:227]\n" \
    "	ds_read_b128 v[76:79], v137 offset:4096\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[36:39], v[0:3], a[4:7]\n" \
    "	s_add_u32 m0, s61, 71680\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v146, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[36:39], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[80:83], v137 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[36:39], v[8:11], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[36:39], v[12:15], a[100:103]\n" \
    "	ds_read_b128 v[84:87], v137 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[36:39], v[16:19], a[132:135]\n" \
    "	s_add_u32 m0, s61, 72704\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v147, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[36:39], v[20:23], a[164:167]\n" \
    "	ds_read_b128 v[88:91], v137 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[36:39], v[24:27], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[36:39], v[28:31], a[228:231]\n" \
    "	ds_read_b128 v[92:95], v137 offset:12288\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[40:43], v[0:3], a[8:11]\n" \
    "	s_add_u32 m0, s61, 73728\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v148, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[40:43], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[96:99], v137 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[40:43], v[8:11], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[40:43], v[12:15], a[104:107]\n" \
    "	ds_read_b128 v[104:107], v141 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[40:43], v[16:19], a[136:139]\n" \
    "	s_add_u32 m0, s61, 74752\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v149, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[40:43], v[20:23], a[168:171]\n" \
    "	ds_read_b128 v[108:111], v141 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[40:43], v[24:27], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[40:43], v[28:31], a[232:235]\n" \
    "	ds_read_b128 v[112:115], v141 offset:6144\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[44:47], v[0:3], a[12:15]\n" \
    "	s_add_u32 m0, s61, 75776\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v150, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[44:47], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[116:119], v141 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[44:47], v[8:11], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[44:47], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[120:123], v141 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[44:47], v[16:19], a[140:143]\n" \
    "	s_add_u32 m0, s61, 76800\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v151, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[44:47], v[20:23], a[172:175]\n" \
    "	ds_read_b128 v[124:127], v141 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[44:47], v[24:27], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[44:47], v[28:31], a[236:239]\n" \
    "	ds_read_b128 v[128:131], v141 offset:14336\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[48:51], v[0:3], a[16:19]\n" \
    "	s_add_u32 m0, s69, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v152, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[48:51], v[4:7], a[48:51]\n" \
    "	ds_read_b128 v[132:135], v141 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[48:51], v[8:11], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[48:51], v[12:15], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[48:51], v[16:19], a[144:147]\n" \
    "	s_add_u32 m0, s69, 103424\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v153, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[48:51], v[20:23], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[48:51], v[24:27], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[48:51], v[28:31], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[52:55], v[0:3], a[20:23]\n" \
    "	s_add_u32 m0, s69, 104448\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v154, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[52:55], v[4:7], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[52:55], v[8:11], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[52:55], v[12:15], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[52:55], v[16:19], a[148:151]\n" \
    "	s_add_u32 m0, s69, 105472\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v155, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[52:55], v[20:23], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[52:55], v[24:27], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[52:55], v[28:31], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[56:59], v[0:3], a[24:27]\n" \
    "	s_add_u32 m0, s69, 106496\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v156, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[56:59], v[4:7], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[56:59], v[8:11], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[56:59], v[12:15], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[56:59], v[16:19], a[152:155]\n" \
    "	s_add_u32 m0, s69, 107520\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v157, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[56:59], v[20:23], a[184:187]\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[56:59], v[24:27], a[216:219]\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[56:59], v[28:31], a[248:251]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[60:63], v[0:3], a[28:31]\n" \
    "	s_add_u32 m0, s69, 108544\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v158, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[60:63], v[4:7], a[60:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[60:63], v[8:11], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[60:63], v[12:15], a[124:127]\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[60:63], v[16:19], a[156:159]\n" \
    "	s_add_u32 m0, s69, 109568\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v159, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[60:63], v[20:23], a[188:191]\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[60:63], v[24:27], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[60:63], v[28:31], a[252:255]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_0], v[64:67], v[0:3], %[c8_0]\n" \
    "	s_add_u32 m0, s69, 110592\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v160, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_1], v[64:67], v[4:7], %[c8_1]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_2], v[64:67], v[8:11], %[c8_2]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_3], v[64:67], v[12:15], %[c8_3]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_4], v[64:67], v[16:19], %[c8_4]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_5], v[64:67], v[20:23], %[c8_5]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_6], v[64:67], v[24:27], %[c8_6]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_7], v[64:67], v[28:31], %[c8_7]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[100:103], v[68:71], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[100:103], v[72:75], a[32:35]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[100:103], v[76:79], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[100:103], v[80:83], a[96:99]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[100:103], v[84:87], a[128:131]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[100:103], v[88:91], a[160:163]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[100:103], v[92:95], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[100:103], v[96:99], a[224:227]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[104:107], v[68:71], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[104:107], v[72:75], a[36:39]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[104:107], v[76:79], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[104:107], v[80:83], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[104:107], v[84:87], a[132:135]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[104:107], v[88:91], a[164:167]\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[104:107], v[92:95], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[104:107], v[96:99], a[228:231]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[108:111], v[68:71], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[108:111], v[72:75], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[108:111], v[76:79], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[108:111], v[80:83], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[108:111], v[84:87], a[136:139]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[108:111], v[88:91], a[168:171]\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[108:111], v[92:95], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[108:111], v[96:99], a[232:235]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[112:115], v[68:71], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[112:115], v[72:75], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[112:115], v[76:79], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[112:115], v[80:83], a[108:111]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[112:115], v[84:87], a[140:143]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[112:115], v[88:91], a[172:175]\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[112:115], v[92:95], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[112:115], v[96:99], a[236:239]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[116:119], v[68:71], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[116:119], v[72:75], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[116:119], v[76:79], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[116:119], v[80:83], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[116:119], v[84:87], a[144:147]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[116:119], v[88:91], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[116:119], v[92:95], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[116:119], v[96:99], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[120:123], v[68:71], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[120:123], v[72:75], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[120:123], v[76:79], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[120:123], v[80:83], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[120:123], v[84:87], a[148:151]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[120:123], v[88:91], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[120:123], v[92:95], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[120:123], v[96:99], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(2)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[124:127], v[68:71], a[24:27]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[124:127], v[72:75], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[124:127], v[76:79], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[124:127], v[80:83], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[124:127], v[84:87], a[152:155]\n" \
    "	s_waitcnt vmcnt(0)\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	s_barrier\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[124:127], v[88:91], a[184:187]\n" \
    "	ds_read_b128 v[32:35], v142 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[124:127], v[92:95], a[216:219]\n" \
    "	ds_read_b128 v[0:3], v138 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[124:127], v[96:99], a[248:251]\n" \
    "	ds_read_b128 v[4:7], v138 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[128:131], v[68:71], a[28:31]\n" \
    "	ds_read_b128 v[8:11], v138 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[128:131], v[72:75], a[60:63]\n" \
    "	ds_read_b128 v[12:15], v138 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[128:131], v[76:79], a[92:95]\n" \
    "	ds_read_b128 v[16:19], v138 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[128:131], v[80:83], a[124:127]\n" \
    "	ds_read_b128 v[20:23], v138 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[128:131], v[84:87], a[156:159]\n" \
    "	ds_read_b128 v[24:27], v138 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[128:131], v[88:91], a[188:191]\n" \
    "	ds_read_b128 v[28:31], v138 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[128:131], v[92:95], a[220:223]\n" \
    "	ds_read_b128 v[36:39], v142 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[128:131], v[96:99], a[252:255]\n" \
    "	ds_read_b128 v[40:43], v142 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_0], v[132:135], v[68:71], %[c8_0]\n" \
    "	ds_read_b128 v[44:47], v142 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_1], v[132:135], v[72:75], %[c8_1]\n" \
    "	ds_read_b128 v[48:51], v142 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_2], v[132:135], v[76:79], %[c8_2]\n" \
    "	ds_read_b128 v[52:55], v142 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_3], v[132:135], v[80:83], %[c8_3]\n" \
    "	ds_read_b128 v[56:59], v142 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_4], v[132:135], v[84:87], %[c8_4]\n" \
    "	ds_read_b128 v[60:63], v142 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_5], v[132:135], v[88:91], %[c8_5]\n" \
    "	ds_read_b128 v[64:67], v142 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_6], v[132:135], v[92:95], %[c8_6]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_7], v[132:135], v[96:99], %[c8_7]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[32:35], v[0:3], a[0:3]\n" \
    "	s_add_u32 m0, s61, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v144, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[32:35], v[4:7], a[32:35]\n" \
    "	ds_read_b128 v[100:103], v143 offset:0\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[32:35], v[8:11], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[32:35], v[12:15], a[96:99]\n" \
    "	ds_read_b128 v[68:71], v139 offset:0\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[32:35], v[16:19], a[128:131]\n" \
    "	s_add_u32 m0, s61, 1024\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v145, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[32:35], v[20:23], a[160:163]\n" \
    "	ds_read_b128 v[72:75], v139 offset:2048\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[32:35], v[24:27], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[32:35], v[28:31], a[224:227]\n" \
    "	ds_read_b128 v[76:79], v139 offset:4096\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[36:39], v[0:3], a[4:7]\n" \
    "	s_add_u32 m0, s61, 2048\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v146, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[36:39], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[80:83], v139 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[36:39], v[8:11], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[36:39], v[12:15], a[100:103]\n" \
    "	ds_read_b128 v[84:87], v139 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[36:39], v[16:19], a[132:135]\n" \
    "	s_add_u32 m0, s61, 3072\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v147, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[36:39], v[20:23], a[164:167]\n" \
    "	ds_read_b128 v[88:91], v139 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[36:39], v[24:27], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[36:39], v[28:31], a[228:231]\n" \
    "	ds_read_b128 v[92:95], v139 offset:12288\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[40:43], v[0:3], a[8:11]\n" \
    "	s_add_u32 m0, s61, 4096\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v148, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[40:43], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[96:99], v139 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[40:43], v[8:11], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[40:43], v[12:15], a[104:107]\n" \
    "	ds_read_b128 v[104:107], v143 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[40:43], v[16:19], a[136:139]\n" \
    "	s_add_u32 m0, s61, 5120\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v149, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[40:43], v[20:23], a[168:171]\n" \
    "	ds_read_b128 v[108:111], v143 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[40:43], v[24:27], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[40:43], v[28:31], a[232:235]\n" \
    "	ds_read_b128 v[112:115], v143 offset:6144\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[44:47], v[0:3], a[12:15]\n" \
    "	s_add_u32 m0, s61, 6144\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v150, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[44:47], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[116:119], v143 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[44:47], v[8:11], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[44:47], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[120:123], v143 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[44:47], v[16:19], a[140:143]\n" \
    "	s_add_u32 m0, s61, 7168\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v151, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[44:47], v[20:23], a[172:175]\n" \
    "	ds_read_b128 v[124:127], v143 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[44:47], v[24:27], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[44:47], v[28:31], a[236:239]\n" \
    "	ds_read_b128 v[128:131], v143 offset:14336\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[48:51], v[0:3], a[16:19]\n" \
    "	s_add_u32 m0, s69, 32768\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v152, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[48:51], v[4:7], a[48:51]\n" \
    "	ds_read_b128 v[132:135], v143 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[48:51], v[8:11], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[48:51], v[12:15], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[48:51], v[16:19], a[144:147]\n" \
    "	s_add_u32 m0, s69, 33792\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v153, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[48:51], v[20:23], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[48:51], v[24:27], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[48:51], v[28:31], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[52:55], v[0:3], a[20:23]\n" \
    "	s_add_u32 m0, s69, 34816\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v154, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[52:55], v[4:7], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[52:55], v[8:11], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[52:55], v[12:15], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[52:55], v[16:19], a[148:151]\n" \
    "	s_add_u32 m0, s69, 35840\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v155, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[52:55], v[20:23], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[52:55], v[24:27], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[52:55], v[28:31], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[56:59], v[0:3], a[24:27]\n" \
    "	s_add_u32 m0, s69, 36864\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v156, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[56:59], v[4:7], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[56:59], v[8:11], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[56:59], v[12:15], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[56:59], v[16:19], a[152:155]\n" \
    "	s_add_u32 m0, s69, 37888\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v157, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[56:59], v[20:23], a[184:187]\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[56:59], v[24:27], a[216:219]\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[56:59], v[28:31], a[248:251]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[60:63], v[0:3], a[28:31]\n" \
    "	s_add_u32 m0, s69, 38912\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v158, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[60:63], v[4:7], a[60:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[60:63], v[8:11], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[60:63], v[12:15], a[124:127]\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[60:63], v[16:19], a[156:159]\n" \
    "	s_add_u32 m0, s69, 39936\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v159, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[60:63], v[20:23], a[188:191]\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[60:63], v[24:27], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[60:63], v[28:31], a[252:255]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_0], v[64:67], v[0:3], %[c8_0]\n" \
    "	s_add_u32 m0, s69, 40960\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v160, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_1], v[64:67], v[4:7], %[c8_1]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_2], v[64:67], v[8:11], %[c8_2]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_3], v[64:67], v[12:15], %[c8_3]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_4], v[64:67], v[16:19], %[c8_4]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_5], v[64:67], v[20:23], %[c8_5]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_6], v[64:67], v[24:27], %[c8_6]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_7], v[64:67], v[28:31], %[c8_7]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[100:103], v[68:71], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[100:103], v[72:75], a[32:35]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[100:103], v[76:79], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[100:103], v[80:83], a[96:99]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[100:103], v[84:87], a[128:131]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[100:103], v[88:91], a[160:163]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[100:103], v[92:95], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[100:103], v[96:99], a[224:227]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[104:107], v[68:71], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[104:107], v[72:75], a[36:39]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[104:107], v[76:79], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[104:107], v[80:83], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[104:107], v[84:87], a[132:135]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[104:107], v[88:91], a[164:167]\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[104:107], v[92:95], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[104:107], v[96:99], a[228:231]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[108:111], v[68:71], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[108:111], v[72:75], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[108:111], v[76:79], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[108:111], v[80:83], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[108:111], v[84:87], a[136:139]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[108:111], v[88:91], a[168:171]\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[108:111], v[92:95], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[108:111], v[96:99], a[232:235]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[112:115], v[68:71], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[112:115], v[72:75], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[112:115], v[76:79], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[112:115], v[80:83], a[108:111]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[112:115], v[84:87], a[140:143]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[112:115], v[88:91], a[172:175]\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[112:115], v[92:95], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[112:115], v[96:99], a[236:239]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[116:119], v[68:71], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[116:119], v[72:75], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[116:119], v[76:79], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[116:119], v[80:83], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[116:119], v[84:87], a[144:147]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[116:119], v[88:91], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[116:119], v[92:95], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[116:119], v[96:99], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[120:123], v[68:71], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[120:123], v[72:75], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[120:123], v[76:79], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[120:123], v[80:83], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[120:123], v[84:87], a[148:151]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[120:123], v[88:91], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[120:123], v[92:95], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[120:123], v[96:99], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(2)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[124:127], v[68:71], a[24:27]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[124:127], v[72:75], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[124:127], v[76:79], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[124:127], v[80:83], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[124:127], v[84:87], a[152:155]\n" \
    "	s_waitcnt vmcnt(0)\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	s_barrier\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[124:127], v[88:91], a[184:187]\n" \
    "	ds_read_b128 v[32:35], v140 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[124:127], v[92:95], a[216:219]\n" \
    "	ds_read_b128 v[0:3], v136 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[124:127], v[96:99], a[248:251]\n" \
    "	ds_read_b128 v[4:7], v136 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[128:131], v[68:71], a[28:31]\n" \
    "	ds_read_b128 v[8:11], v136 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[128:131], v[72:75], a[60:63]\n" \
    "	ds_read_b128 v[12:15], v136 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[128:131], v[76:79], a[92:95]\n" \
    "	ds_read_b128 v[16:19], v136 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[128:131], v[80:83], a[124:127]\n" \
    "	ds_read_b128 v[20:23], v136 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[128:131], v[84:87], a[156:159]\n" \
    "	ds_read_b128 v[24:27], v136 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[128:131], v[88:91], a[188:191]\n" \
    "	ds_read_b128 v[28:31], v136 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[128:131], v[92:95], a[220:223]\n" \
    "	ds_read_b128 v[36:39], v140 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[128:131], v[96:99], a[252:255]\n" \
    "	ds_read_b128 v[40:43], v140 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_0], v[132:135], v[68:71], %[c8_0]\n" \
    "	ds_read_b128 v[44:47], v140 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_1], v[132:135], v[72:75], %[c8_1]\n" \
    "	ds_read_b128 v[48:51], v140 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_2], v[132:135], v[76:79], %[c8_2]\n" \
    "	ds_read_b128 v[52:55], v140 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_3], v[132:135], v[80:83], %[c8_3]\n" \
    "	ds_read_b128 v[56:59], v140 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_4], v[132:135], v[84:87], %[c8_4]\n" \
    "	ds_read_b128 v[60:63], v140 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_5], v[132:135], v[88:91], %[c8_5]\n" \
    "	ds_read_b128 v[64:67], v140 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_6], v[132:135], v[92:95], %[c8_6]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_7], v[132:135], v[96:99], %[c8_7]\n" \
    "	s_sub_u32 s60, s60, 1\n" \
    "	s_cmp_eq_u32 s60, 0\n" \
    "	s_cbranch_scc0 LOOP_%=\n" \
    "LAST_%=:\n" \
    "	s_cmp_eq_u32 %[rem], 1\n" \
    "	s_cbranch_scc1 LAST1_%=\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[32:35], v[0:3], a[0:3]\n" \
    "	s_add_u32 m0, s61, 69632\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v144, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[32:35], v[4:7], a[32:35]\n" \
    "	ds_read_b128 v[100:103], v141 offset:0\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[32:35], v[8:11], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[32:35], v[12:15], a[96:99]\n" \
    "	ds_read_b128 v[68:71], v137 offset:0\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[32:35], v[16:19], a[128:131]\n" \
    "	s_add_u32 m0, s61, 70656\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v145, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[32:35], v[20:23], a[160:163]\n" \
    "	ds_read_b128 v[72:75], v137 offset:2048\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[32:35], v[24:27], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[32:35], v[28:31], a[224:227]\n" \
    "	ds_read_b128 v[76:79], v137 offset:4096\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[36:39], v[0:3], a[4:7]\n" \
    "	s_add_u32 m0, s61, 71680\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v146, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[36:39], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[80:83], v137 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[36:39], v[8:11], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[36:39], v[12:15], a[100:103]\n" \
    "	ds_read_b128 v[84:87], v137 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[36:39], v[16:19], a[132:135]\n" \
    "	s_add_u32 m0, s61, 72704\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v147, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[36:39], v[20:23], a[164:167]\n" \
    "	ds_read_b128 v[88:91], v137 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[36:39], v[24:27], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[36:39], v[28:31], a[228:231]\n" \
    "	ds_read_b128 v[92:95], v137 offset:12288\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[40:43], v[0:3], a[8:11]\n" \
    "	s_add_u32 m0, s61, 73728\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v148, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[40:43], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[96:99], v137 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[40:43], v[8:11], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[40:43], v[12:15], a[104:107]\n" \
    "	ds_read_b128 v[104:107], v141 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[40:43], v[16:19], a[136:139]\n" \
    "	s_add_u32 m0, s61, 74752\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v149, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[40:43], v[20:23], a[168:171]\n" \
    "	ds_read_b128 v[108:111], v141 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[40:43], v[24:27], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[40:43], v[28:31], a[232:235]\n" \
    "	ds_read_b128 v[112:115], v141 offset:6144\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[44:47], v[0:3], a[12:15]\n" \
    "	s_add_u32 m0, s61, 75776\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v150, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[44:47], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[116:119], v141 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[44:47], v[8:11], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[44:47], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[120:123], v141 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[44:47], v[16:19], a[140:143]\n" \
    "	s_add_u32 m0, s61, 76800\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v151, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[44:47], v[20:23], a[172:175]\n" \
    "	ds_read_b128 v[124:127], v141 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[44:47], v[24:27], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[44:47], v[28:31], a[236:239]\n" \
    "	ds_read_b128 v[128:131], v141 offset:14336\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[48:51], v[0:3], a[16:19]\n" \
    "	s_add_u32 m0, s69, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v152, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[48:51], v[4:7], a[48:51]\n" \
    "	ds_read_b128 v[132:135], v141 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[48:51], v[8:11], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[48:51], v[12:15], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[48:51], v[16:19], a[144:147]\n" \
    "	s_add_u32 m0, s69, 103424\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v153, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[48:51], v[20:23], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[48:51], v[24:27], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[48:51], v[28:31], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[52:55], v[0:3], a[20:23]\n" \
    "	s_add_u32 m0, s69, 104448\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v154, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[52:55], v[4:7], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[52:55], v[8:11], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[52:55], v[12:15], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[52:55], v[16:19], a[148:151]\n" \
    "	s_add_u32 m0, s69, 105472\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v155, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[52:55], v[20:23], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[52:55], v[24:27], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[52:55], v[28:31], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[56:59], v[0:3], a[24:27]\n" \
    "	s_add_u32 m0, s69, 106496\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v156, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[56:59], v[4:7], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[56:59], v[8:11], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[56:59], v[12:15], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[56:59], v[16:19], a[152:155]\n" \
    "	s_add_u32 m0, s69, 107520\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v157, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[56:59], v[20:23], a[184:187]\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[56:59], v[24:27], a[216:219]\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[56:59], v[28:31], a[248:251]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[60:63], v[0:3], a[28:31]\n" \
    "	s_add_u32 m0, s69, 108544\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v158, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[60:63], v[4:7], a[60:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[60:63], v[8:11], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[60:63], v[12:15], a[124:127]\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[60:63], v[16:19], a[156:159]\n" \
    "	s_add_u32 m0, s69, 109568\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v159, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[60:63], v[20:23], a[188:191]\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[60:63], v[24:27], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[60:63], v[28:31], a[252:255]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_0], v[64:67], v[0:3], %[c8_0]\n" \
    "	s_add_u32 m0, s69, 110592\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v160, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_1], v[64:67], v[4:7], %[c8_1]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_2], v[64:67], v[8:11], %[c8_2]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_3], v[64:67], v[12:15], %[c8_3]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_4], v[64:67], v[16:19], %[c8_4]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_5], v[64:67], v[20:23], %[c8_5]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_6], v[64:67], v[24:27], %[c8_6]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_7], v[64:67], v[28:31], %[c8_7]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[100:103], v[68:71], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[100:103], v[72:75], a[32:35]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[100:103], v[76:79], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[100:103], v[80:83], a[96:99]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[100:103], v[84:87], a[128:131]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[100:103], v[88:91], a[160:163]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[100:103], v[92:95], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[100:103], v[96:99], a[224:227]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[104:107], v[68:71], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[104:107], v[72:75], a[36:39]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[104:107], v[76:79], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[104:107], v[80:83], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[104:107], v[84:87], a[132:135]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[104:107], v[88:91], a[164:167]\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[104:107], v[92:95], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[104:107], v[96:99], a[228:231]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[108:111], v[68:71], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[108:111], v[72:75], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[108:111], v[76:79], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[108:111], v[80:83], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[108:111], v[84:87], a[136:139]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[108:111], v[88:91], a[168:171]\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[108:111], v[92:95], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[108:111], v[96:99], a[232:235]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[112:115], v[68:71], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[112:115], v[72:75], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[112:115], v[76:79], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[112:115], v[80:83], a[108:111]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[112:115], v[84:87], a[140:143]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[112:115], v[88:91], a[172:175]\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[112:115], v[92:95], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[112:115], v[96:99], a[236:239]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[116:119], v[68:71], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[116:119], v[72:75], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[116:119], v[76:79], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[116:119], v[80:83], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[116:119], v[84:87], a[144:147]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[116:119], v[88:91], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[116:119], v[92:95], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[116:119], v[96:99], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[120:123], v[68:71], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[120:123], v[72:75], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[120:123], v[76:79], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[120:123], v[80:83], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[120:123], v[84:87], a[148:151]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[120:123], v[88:91], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[120:123], v[92:95], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[120:123], v[96:99], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(2)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[124:127], v[68:71], a[24:27]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[124:127], v[72:75], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[124:127], v[76:79], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[124:127], v[80:83], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[124:127], v[84:87], a[152:155]\n" \
    "	s_waitcnt vmcnt(0)\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	s_barrier\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[124:127], v[88:91], a[184:187]\n" \
    "	ds_read_b128 v[32:35], v142 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[124:127], v[92:95], a[216:219]\n" \
    "	ds_read_b128 v[0:3], v138 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[124:127], v[96:99], a[248:251]\n" \
    "	ds_read_b128 v[4:7], v138 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[128:131], v[68:71], a[28:31]\n" \
    "	ds_read_b128 v[8:11], v138 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[128:131], v[72:75], a[60:63]\n" \
    "	ds_read_b128 v[12:15], v138 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[128:131], v[76:79], a[92:95]\n" \
    "	ds_read_b128 v[16:19], v138 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[128:131], v[80:83], a[124:127]\n" \
    "	ds_read_b128 v[20:23], v138 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[128:131], v[84:87], a[156:159]\n" \
    "	ds_read_b128 v[24:27], v138 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[128:131], v[88:91], a[188:191]\n" \
    "	ds_read_b128 v[28:31], v138 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[128:131], v[92:95], a[220:223]\n" \
    "	ds_read_b128 v[36:39], v142 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[128:131], v[96:99], a[252:255]\n" \
    "	ds_read_b128 v[40:43], v142 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_0], v[132:135], v[68:71], %[c8_0]\n" \
    "	ds_read_b128 v[44:47], v142 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_1], v[132:135], v[72:75], %[c8_1]\n" \
    "	ds_read_b128 v[48:51], v142 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_2], v[132:135], v[76:79], %[c8_2]\n" \
    "	ds_read_b128 v[52:55], v142 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_3], v[132:135], v[80:83], %[c8_3]\n" \
    "	ds_read_b128 v[56:59], v142 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_4], v[132:135], v[84:87], %[c8_4]\n" \
    "	ds_read_b128 v[60:63], v142 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_5], v[132:135], v[88:91], %[c8_5]\n" \
    "	ds_read_b128 v[64:67], v142 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_6], v[132:135], v[92:95], %[c8_6]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_7], v[132:135], v[96:99], %[c8_7]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[32:35], v[0:3], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[32:35], v[4:7], a[32:35]\n" \
    "	ds_read_b128 v[100:103], v143 offset:0\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[32:35], v[8:11], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[32:35], v[12:15], a[96:99]\n" \
    "	ds_read_b128 v[68:71], v139 offset:0\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[32:35], v[16:19], a[128:131]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[32:35], v[20:23], a[160:163]\n" \
    "	ds_read_b128 v[72:75], v139 offset:2048\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[32:35], v[24:27], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[32:35], v[28:31], a[224:227]\n" \
    "	ds_read_b128 v[76:79], v139 offset:4096\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[36:39], v[0:3], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[36:39], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[80:83], v139 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[36:39], v[8:11], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[36:39], v[12:15], a[100:103]\n" \
    "	ds_read_b128 v[84:87], v139 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[36:39], v[16:19], a[132:135]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[36:39], v[20:23], a[164:167]\n" \
    "	ds_read_b128 v[88:91], v139 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[36:39], v[24:27], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[36:39], v[28:31], a[228:231]\n" \
    "	ds_read_b128 v[92:95], v139 offset:12288\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[40:43], v[0:3], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[40:43], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[96:99], v139 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[40:43], v[8:11], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[40:43], v[12:15], a[104:107]\n" \
    "	ds_read_b128 v[104:107], v143 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[40:43], v[16:19], a[136:139]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[40:43], v[20:23], a[168:171]\n" \
    "	ds_read_b128 v[108:111], v143 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[40:43], v[24:27], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[40:43], v[28:31], a[232:235]\n" \
    "	ds_read_b128 v[112:115], v143 offset:6144\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[44:47], v[0:3], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[44:47], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[116:119], v143 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[44:47], v[8:11], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[44:47], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[120:123], v143 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[44:47], v[16:19], a[140:143]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[44:47], v[20:23], a[172:175]\n" \
    "	ds_read_b128 v[124:127], v143 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[44:47], v[24:27], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[44:47], v[28:31], a[236:239]\n" \
    "	ds_read_b128 v[128:131], v143 offset:14336\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[48:51], v[0:3], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[48:51], v[4:7], a[48:51]\n" \
    "	ds_read_b128 v[132:135], v143 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[48:51], v[8:11], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[48:51], v[12:15], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[48:51], v[16:19], a[144:147]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[48:51], v[20:23], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[48:51], v[24:27], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[48:51], v[28:31], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[52:55], v[0:3], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[52:55], v[4:7], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[52:55], v[8:11], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[52:55], v[12:15], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[52:55], v[16:19], a[148:151]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[52:55], v[20:23], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[52:55], v[24:27], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[52:55], v[28:31], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[56:59], v[0:3], a[24:27]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[56:59], v[4:7], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[56:59], v[8:11], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[56:59], v[12:15], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[56:59], v[16:19], a[152:155]\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[56:59], v[20:23], a[184:187]\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[56:59], v[24:27], a[216:219]\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[56:59], v[28:31], a[248:251]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[60:63], v[0:3], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[60:63], v[4:7], a[60:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[60:63], v[8:11], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[60:63], v[12:15], a[124:127]\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[60:63], v[16:19], a[156:159]\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[60:63], v[20:23], a[188:191]\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[60:63], v[24:27], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[60:63], v[28:31], a[252:255]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_0], v[64:67], v[0:3], %[c8_0]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_1], v[64:67], v[4:7], %[c8_1]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_2], v[64:67], v[8:11], %[c8_2]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_3], v[64:67], v[12:15], %[c8_3]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_4], v[64:67], v[16:19], %[c8_4]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_5], v[64:67], v[20:23], %[c8_5]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_6], v[64:67], v[24:27], %[c8_6]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_7], v[64:67], v[28:31], %[c8_7]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[100:103], v[68:71], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[100:103], v[72:75], a[32:35]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[100:103], v[76:79], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[100:103], v[80:83], a[96:99]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[100:103], v[84:87], a[128:131]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[100:103], v[88:91], a[160:163]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[100:103], v[92:95], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[100:103], v[96:99], a[224:227]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[104:107], v[68:71], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[104:107], v[72:75], a[36:39]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[104:107], v[76:79], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[104:107], v[80:83], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[104:107], v[84:87], a[132:135]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[104:107], v[88:91], a[164:167]\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[104:107], v[92:95], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[104:107], v[96:99], a[228:231]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[108:111], v[68:71], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[108:111], v[72:75], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[108:111], v[76:79], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[108:111], v[80:83], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[108:111], v[84:87], a[136:139]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[108:111], v[88:91], a[168:171]\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[108:111], v[92:95], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[108:111], v[96:99], a[232:235]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[112:115], v[68:71], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[112:115], v[72:75], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[112:115], v[76:79], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[112:115], v[80:83], a[108:111]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[112:115], v[84:87], a[140:143]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[112:115], v[88:91], a[172:175]\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[112:115], v[92:95], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[112:115], v[96:99], a[236:239]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[116:119], v[68:71], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[116:119], v[72:75], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[116:119], v[76:79], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[116:119], v[80:83], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[116:119], v[84:87], a[144:147]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[116:119], v[88:91], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[116:119], v[92:95], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[116:119], v[96:99], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[120:123], v[68:71], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[120:123], v[72:75], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[120:123], v[76:79], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[120:123], v[80:83], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[120:123], v[84:87], a[148:151]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[120:123], v[88:91], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[120:123], v[92:95], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[120:123], v[96:99], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(2)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[124:127], v[68:71], a[24:27]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[124:127], v[72:75], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[124:127], v[76:79], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[124:127], v[80:83], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[124:127], v[84:87], a[152:155]\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[124:127], v[88:91], a[184:187]\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[124:127], v[92:95], a[216:219]\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[124:127], v[96:99], a[248:251]\n" \
    "	s_waitcnt lgkmcnt(1)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[128:131], v[68:71], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[128:131], v[72:75], a[60:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[128:131], v[76:79], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[128:131], v[80:83], a[124:127]\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[128:131], v[84:87], a[156:159]\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[128:131], v[88:91], a[188:191]\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[128:131], v[92:95], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[128:131], v[96:99], a[252:255]\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_0], v[132:135], v[68:71], %[c8_0]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_1], v[132:135], v[72:75], %[c8_1]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_2], v[132:135], v[76:79], %[c8_2]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_3], v[132:135], v[80:83], %[c8_3]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_4], v[132:135], v[84:87], %[c8_4]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_5], v[132:135], v[88:91], %[c8_5]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_6], v[132:135], v[92:95], %[c8_6]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_7], v[132:135], v[96:99], %[c8_7]\n" \
    "	s_branch DONE_%=\n" \
    "LAST1_%=:\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[32:35], v[0:3], a[0:3]\n" \
    "	s_add_u32 m0, s61, 69632\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v144, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[32:35], v[4:7], a[32:35]\n" \
    "	ds_read_b128 v[100:103], v141 offset:0\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[32:35], v[8:11], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[32:35], v[12:15], a[96:99]\n" \
    "	ds_read_b128 v[68:71], v137 offset:0\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[32:35], v[16:19], a[128:131]\n" \
    "	s_add_u32 m0, s61, 70656\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v145, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[32:35], v[20:23], a[160:163]\n" \
    "	ds_read_b128 v[72:75], v137 offset:2048\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[32:35], v[24:27], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[32:35], v[28:31], a[224:227]\n" \
    "	ds_read_b128 v[76:79], v137 offset:4096\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[36:39], v[0:3], a[4:7]\n" \
    "	s_add_u32 m0, s61, 71680\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v146, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[36:39], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[80:83], v137 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[36:39], v[8:11], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[36:39], v[12:15], a[100:103]\n" \
    "	ds_read_b128 v[84:87], v137 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[36:39], v[16:19], a[132:135]\n" \
    "	s_add_u32 m0, s61, 72704\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v147, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[36:39], v[20:23], a[164:167]\n" \
    "	ds_read_b128 v[88:91], v137 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[36:39], v[24:27], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[36:39], v[28:31], a[228:231]\n" \
    "	ds_read_b128 v[92:95], v137 offset:12288\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[40:43], v[0:3], a[8:11]\n" \
    "	s_add_u32 m0, s61, 73728\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v148, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[40:43], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[96:99], v137 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[40:43], v[8:11], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[40:43], v[12:15], a[104:107]\n" \
    "	ds_read_b128 v[104:107], v141 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[40:43], v[16:19], a[136:139]\n" \
    "	s_add_u32 m0, s61, 74752\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v149, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[40:43], v[20:23], a[168:171]\n" \
    "	ds_read_b128 v[108:111], v141 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[40:43], v[24:27], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[40:43], v[28:31], a[232:235]\n" \
    "	ds_read_b128 v[112:115], v141 offset:6144\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[44:47], v[0:3], a[12:15]\n" \
    "	s_add_u32 m0, s61, 75776\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v150, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[44:47], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[116:119], v141 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[44:47], v[8:11], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[44:47], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[120:123], v141 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[44:47], v[16:19], a[140:143]\n" \
    "	s_add_u32 m0, s61, 76800\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v151, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[44:47], v[20:23], a[172:175]\n" \
    "	ds_read_b128 v[124:127], v141 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[44:47], v[24:27], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[44:47], v[28:31], a[236:239]\n" \
    "	ds_read_b128 v[128:131], v141 offset:14336\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[48:51], v[0:3], a[16:19]\n" \
    "	s_add_u32 m0, s69, 102400\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v152, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[48:51], v[4:7], a[48:51]\n" \
    "	ds_read_b128 v[132:135], v141 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[48:51], v[8:11], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[48:51], v[12:15], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[48:51], v[16:19], a[144:147]\n" \
    "	s_add_u32 m0, s69, 103424\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v153, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[48:51], v[20:23], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[48:51], v[24:27], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[48:51], v[28:31], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[52:55], v[0:3], a[20:23]\n" \
    "	s_add_u32 m0, s69, 104448\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v154, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[52:55], v[4:7], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[52:55], v[8:11], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[52:55], v[12:15], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[52:55], v[16:19], a[148:151]\n" \
    "	s_add_u32 m0, s69, 105472\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v155, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[52:55], v[20:23], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[52:55], v[24:27], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[52:55], v[28:31], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[56:59], v[0:3], a[24:27]\n" \
    "	s_add_u32 m0, s69, 106496\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v156, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[56:59], v[4:7], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[56:59], v[8:11], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[56:59], v[12:15], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[56:59], v[16:19], a[152:155]\n" \
    "	s_add_u32 m0, s69, 107520\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v157, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[56:59], v[20:23], a[184:187]\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[56:59], v[24:27], a[216:219]\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[56:59], v[28:31], a[248:251]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[60:63], v[0:3], a[28:31]\n" \
    "	s_add_u32 m0, s69, 108544\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v158, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[60:63], v[4:7], a[60:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[60:63], v[8:11], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[60:63], v[12:15], a[124:127]\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[60:63], v[16:19], a[156:159]\n" \
    "	s_add_u32 m0, s69, 109568\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v159, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[60:63], v[20:23], a[188:191]\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[60:63], v[24:27], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[60:63], v[28:31], a[252:255]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_0], v[64:67], v[0:3], %[c8_0]\n" \
    "	s_add_u32 m0, s69, 110592\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v160, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_1], v[64:67], v[4:7], %[c8_1]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_2], v[64:67], v[8:11], %[c8_2]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_3], v[64:67], v[12:15], %[c8_3]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_4], v[64:67], v[16:19], %[c8_4]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_5], v[64:67], v[20:23], %[c8_5]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_6], v[64:67], v[24:27], %[c8_6]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_7], v[64:67], v[28:31], %[c8_7]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[100:103], v[68:71], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[100:103], v[72:75], a[32:35]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[100:103], v[76:79], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[100:103], v[80:83], a[96:99]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[100:103], v[84:87], a[128:131]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[100:103], v[88:91], a[160:163]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[100:103], v[92:95], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[100:103], v[96:99], a[224:227]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[104:107], v[68:71], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[104:107], v[72:75], a[36:39]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[104:107], v[76:79], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[104:107], v[80:83], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[104:107], v[84:87], a[132:135]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[104:107], v[88:91], a[164:167]\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[104:107], v[92:95], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[104:107], v[96:99], a[228:231]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[108:111], v[68:71], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[108:111], v[72:75], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[108:111], v[76:79], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[108:111], v[80:83], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[108:111], v[84:87], a[136:139]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[108:111], v[88:91], a[168:171]\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[108:111], v[92:95], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[108:111], v[96:99], a[232:235]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[112:115], v[68:71], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[112:115], v[72:75], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[112:115], v[76:79], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[112:115], v[80:83], a[108:111]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[112:115], v[84:87], a[140:143]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[112:115], v[88:91], a[172:175]\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[112:115], v[92:95], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[112:115], v[96:99], a[236:239]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[116:119], v[68:71], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[116:119], v[72:75], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[116:119], v[76:79], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[116:119], v[80:83], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[116:119], v[84:87], a[144:147]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[116:119], v[88:91], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[116:119], v[92:95], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[116:119], v[96:99], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[120:123], v[68:71], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[120:123], v[72:75], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[120:123], v[76:79], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[120:123], v[80:83], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[120:123], v[84:87], a[148:151]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[120:123], v[88:91], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[120:123], v[92:95], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[120:123], v[96:99], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(2)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[124:127], v[68:71], a[24:27]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[124:127], v[72:75], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[124:127], v[76:79], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[124:127], v[80:83], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[124:127], v[84:87], a[152:155]\n" \
    "	s_waitcnt vmcnt(0)\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	s_barrier\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[124:127], v[88:91], a[184:187]\n" \
    "	ds_read_b128 v[32:35], v142 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[124:127], v[92:95], a[216:219]\n" \
    "	ds_read_b128 v[0:3], v138 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[124:127], v[96:99], a[248:251]\n" \
    "	ds_read_b128 v[4:7], v138 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[128:131], v[68:71], a[28:31]\n" \
    "	ds_read_b128 v[8:11], v138 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[128:131], v[72:75], a[60:63]\n" \
    "	ds_read_b128 v[12:15], v138 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[128:131], v[76:79], a[92:95]\n" \
    "	ds_read_b128 v[16:19], v138 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[128:131], v[80:83], a[124:127]\n" \
    "	ds_read_b128 v[20:23], v138 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[128:131], v[84:87], a[156:159]\n" \
    "	ds_read_b128 v[24:27], v138 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[128:131], v[88:91], a[188:191]\n" \
    "	ds_read_b128 v[28:31], v138 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[128:131], v[92:95], a[220:223]\n" \
    "	ds_read_b128 v[36:39], v142 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[128:131], v[96:99], a[252:255]\n" \
    "	ds_read_b128 v[40:43], v142 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_0], v[132:135], v[68:71], %[c8_0]\n" \
    "	ds_read_b128 v[44:47], v142 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_1], v[132:135], v[72:75], %[c8_1]\n" \
    "	ds_read_b128 v[48:51], v142 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_2], v[132:135], v[76:79], %[c8_2]\n" \
    "	ds_read_b128 v[52:55], v142 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_3], v[132:135], v[80:83], %[c8_3]\n" \
    "	ds_read_b128 v[56:59], v142 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_4], v[132:135], v[84:87], %[c8_4]\n" \
    "	ds_read_b128 v[60:63], v142 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_5], v[132:135], v[88:91], %[c8_5]\n" \
    "	ds_read_b128 v[64:67], v142 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_6], v[132:135], v[92:95], %[c8_6]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_7], v[132:135], v[96:99], %[c8_7]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[32:35], v[0:3], a[0:3]\n" \
    "	s_add_u32 m0, s61, 0\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v144, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[32:35], v[4:7], a[32:35]\n" \
    "	ds_read_b128 v[100:103], v143 offset:0\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[32:35], v[8:11], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[32:35], v[12:15], a[96:99]\n" \
    "	ds_read_b128 v[68:71], v139 offset:0\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[32:35], v[16:19], a[128:131]\n" \
    "	s_add_u32 m0, s61, 1024\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v145, s[62:63]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[32:35], v[20:23], a[160:163]\n" \
    "	ds_read_b128 v[72:75], v139 offset:2048\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[32:35], v[24:27], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[32:35], v[28:31], a[224:227]\n" \
    "	ds_read_b128 v[76:79], v139 offset:4096\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[36:39], v[0:3], a[4:7]\n" \
    "	s_add_u32 m0, s61, 2048\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v146, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[36:39], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[80:83], v139 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[36:39], v[8:11], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[36:39], v[12:15], a[100:103]\n" \
    "	ds_read_b128 v[84:87], v139 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[36:39], v[16:19], a[132:135]\n" \
    "	s_add_u32 m0, s61, 3072\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v147, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[36:39], v[20:23], a[164:167]\n" \
    "	ds_read_b128 v[88:91], v139 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[36:39], v[24:27], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[36:39], v[28:31], a[228:231]\n" \
    "	ds_read_b128 v[92:95], v139 offset:12288\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[40:43], v[0:3], a[8:11]\n" \
    "	s_add_u32 m0, s61, 4096\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v148, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[40:43], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[96:99], v139 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[40:43], v[8:11], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[40:43], v[12:15], a[104:107]\n" \
    "	ds_read_b128 v[104:107], v143 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[40:43], v[16:19], a[136:139]\n" \
    "	s_add_u32 m0, s61, 5120\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v149, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[40:43], v[20:23], a[168:171]\n" \
    "	ds_read_b128 v[108:111], v143 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[40:43], v[24:27], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[40:43], v[28:31], a[232:235]\n" \
    "	ds_read_b128 v[112:115], v143 offset:6144\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[44:47], v[0:3], a[12:15]\n" \
    "	s_add_u32 m0, s61, 6144\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v150, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[44:47], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[116:119], v143 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[44:47], v[8:11], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[44:47], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[120:123], v143 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[44:47], v[16:19], a[140:143]\n" \
    "	s_add_u32 m0, s61, 7168\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v151, s[62:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[44:47], v[20:23], a[172:175]\n" \
    "	ds_read_b128 v[124:127], v143 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[44:47], v[24:27], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[44:47], v[28:31], a[236:239]\n" \
    "	ds_read_b128 v[128:131], v143 offset:14336\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[48:51], v[0:3], a[16:19]\n" \
    "	s_add_u32 m0, s69, 32768\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v152, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[48:51], v[4:7], a[48:51]\n" \
    "	ds_read_b128 v[132:135], v143 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[48:51], v[8:11], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[48:51], v[12:15], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[48:51], v[16:19], a[144:147]\n" \
    "	s_add_u32 m0, s69, 33792\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v153, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[48:51], v[20:23], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[48:51], v[24:27], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[48:51], v[28:31], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[52:55], v[0:3], a[20:23]\n" \
    "	s_add_u32 m0, s69, 34816\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v154, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[52:55], v[4:7], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[52:55], v[8:11], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[52:55], v[12:15], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[52:55], v[16:19], a[148:151]\n" \
    "	s_add_u32 m0, s69, 35840\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v155, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[52:55], v[20:23], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[52:55], v[24:27], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[52:55], v[28:31], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[56:59], v[0:3], a[24:27]\n" \
    "	s_add_u32 m0, s69, 36864\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v156, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[56:59], v[4:7], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[56:59], v[8:11], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[56:59], v[12:15], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[56:59], v[16:19], a[152:155]\n" \
    "	s_add_u32 m0, s69, 37888\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v157, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[56:59], v[20:23], a[184:187]\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[56:59], v[24:27], a[216:219]\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[56:59], v[28:31], a[248:251]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[60:63], v[0:3], a[28:31]\n" \
    "	s_add_u32 m0, s69, 38912\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v158, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[60:63], v[4:7], a[60:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[60:63], v[8:11], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[60:63], v[12:15], a[124:127]\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[60:63], v[16:19], a[156:159]\n" \
    "	s_add_u32 m0, s69, 39936\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v159, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[60:63], v[20:23], a[188:191]\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[60:63], v[24:27], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[60:63], v[28:31], a[252:255]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_0], v[64:67], v[0:3], %[c8_0]\n" \
    "	s_add_u32 m0, s69, 40960\n" \
    "	s_nop 0\n" \
    "	global_load_lds_dwordx4 v160, s[64:65]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_1], v[64:67], v[4:7], %[c8_1]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_2], v[64:67], v[8:11], %[c8_2]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_3], v[64:67], v[12:15], %[c8_3]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_4], v[64:67], v[16:19], %[c8_4]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_5], v[64:67], v[20:23], %[c8_5]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_6], v[64:67], v[24:27], %[c8_6]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_7], v[64:67], v[28:31], %[c8_7]\n" \
    "	s_add_u32 s62, s62, 128\n" \
    "	s_addc_u32 s63, s63, 0\n" \
    "	s_add_u32 s64, s64, 128\n" \
    "	s_addc_u32 s65, s65, 0\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[100:103], v[68:71], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[100:103], v[72:75], a[32:35]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[100:103], v[76:79], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[100:103], v[80:83], a[96:99]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[100:103], v[84:87], a[128:131]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[100:103], v[88:91], a[160:163]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[100:103], v[92:95], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[100:103], v[96:99], a[224:227]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[104:107], v[68:71], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[104:107], v[72:75], a[36:39]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[104:107], v[76:79], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[104:107], v[80:83], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[104:107], v[84:87], a[132:135]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[104:107], v[88:91], a[164:167]\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[104:107], v[92:95], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[104:107], v[96:99], a[228:231]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[108:111], v[68:71], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[108:111], v[72:75], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[108:111], v[76:79], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[108:111], v[80:83], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[108:111], v[84:87], a[136:139]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[108:111], v[88:91], a[168:171]\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[108:111], v[92:95], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[108:111], v[96:99], a[232:235]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[112:115], v[68:71], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[112:115], v[72:75], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[112:115], v[76:79], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[112:115], v[80:83], a[108:111]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[112:115], v[84:87], a[140:143]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[112:115], v[88:91], a[172:175]\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[112:115], v[92:95], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[112:115], v[96:99], a[236:239]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[116:119], v[68:71], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[116:119], v[72:75], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[116:119], v[76:79], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[116:119], v[80:83], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[116:119], v[84:87], a[144:147]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[116:119], v[88:91], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[116:119], v[92:95], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[116:119], v[96:99], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[120:123], v[68:71], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[120:123], v[72:75], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[120:123], v[76:79], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[120:123], v[80:83], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[120:123], v[84:87], a[148:151]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[120:123], v[88:91], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[120:123], v[92:95], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[120:123], v[96:99], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(2)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[124:127], v[68:71], a[24:27]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[124:127], v[72:75], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[124:127], v[76:79], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[124:127], v[80:83], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[124:127], v[84:87], a[152:155]\n" \
    "	s_waitcnt vmcnt(0)\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	s_barrier\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[124:127], v[88:91], a[184:187]\n" \
    "	ds_read_b128 v[32:35], v140 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[124:127], v[92:95], a[216:219]\n" \
    "	ds_read_b128 v[0:3], v136 offset:0\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[124:127], v[96:99], a[248:251]\n" \
    "	ds_read_b128 v[4:7], v136 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[128:131], v[68:71], a[28:31]\n" \
    "	ds_read_b128 v[8:11], v136 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[128:131], v[72:75], a[60:63]\n" \
    "	ds_read_b128 v[12:15], v136 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[128:131], v[76:79], a[92:95]\n" \
    "	ds_read_b128 v[16:19], v136 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[128:131], v[80:83], a[124:127]\n" \
    "	ds_read_b128 v[20:23], v136 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[128:131], v[84:87], a[156:159]\n" \
    "	ds_read_b128 v[24:27], v136 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[128:131], v[88:91], a[188:191]\n" \
    "	ds_read_b128 v[28:31], v136 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[128:131], v[92:95], a[220:223]\n" \
    "	ds_read_b128 v[36:39], v140 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[128:131], v[96:99], a[252:255]\n" \
    "	ds_read_b128 v[40:43], v140 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_0], v[132:135], v[68:71], %[c8_0]\n" \
    "	ds_read_b128 v[44:47], v140 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_1], v[132:135], v[72:75], %[c8_1]\n" \
    "	ds_read_b128 v[48:51], v140 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_2], v[132:135], v[76:79], %[c8_2]\n" \
    "	ds_read_b128 v[52:55], v140 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_3], v[132:135], v[80:83], %[c8_3]\n" \
    "	ds_read_b128 v[56:59], v140 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_4], v[132:135], v[84:87], %[c8_4]\n" \
    "	ds_read_b128 v[60:63], v140 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_5], v[132:135], v[88:91], %[c8_5]\n" \
    "	ds_read_b128 v[64:67], v140 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_6], v[132:135], v[92:95], %[c8_6]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_7], v[132:135], v[96:99], %[c8_7]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[32:35], v[0:3], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[32:35], v[4:7], a[32:35]\n" \
    "	ds_read_b128 v[100:103], v141 offset:0\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[32:35], v[8:11], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[32:35], v[12:15], a[96:99]\n" \
    "	ds_read_b128 v[68:71], v137 offset:0\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[32:35], v[16:19], a[128:131]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[32:35], v[20:23], a[160:163]\n" \
    "	ds_read_b128 v[72:75], v137 offset:2048\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[32:35], v[24:27], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[32:35], v[28:31], a[224:227]\n" \
    "	ds_read_b128 v[76:79], v137 offset:4096\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[36:39], v[0:3], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[36:39], v[4:7], a[36:39]\n" \
    "	ds_read_b128 v[80:83], v137 offset:6144\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[36:39], v[8:11], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[36:39], v[12:15], a[100:103]\n" \
    "	ds_read_b128 v[84:87], v137 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[36:39], v[16:19], a[132:135]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[36:39], v[20:23], a[164:167]\n" \
    "	ds_read_b128 v[88:91], v137 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[36:39], v[24:27], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[36:39], v[28:31], a[228:231]\n" \
    "	ds_read_b128 v[92:95], v137 offset:12288\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[40:43], v[0:3], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[40:43], v[4:7], a[40:43]\n" \
    "	ds_read_b128 v[96:99], v137 offset:14336\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[40:43], v[8:11], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[40:43], v[12:15], a[104:107]\n" \
    "	ds_read_b128 v[104:107], v141 offset:2048\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[40:43], v[16:19], a[136:139]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[40:43], v[20:23], a[168:171]\n" \
    "	ds_read_b128 v[108:111], v141 offset:4096\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[40:43], v[24:27], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[40:43], v[28:31], a[232:235]\n" \
    "	ds_read_b128 v[112:115], v141 offset:6144\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[44:47], v[0:3], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[44:47], v[4:7], a[44:47]\n" \
    "	ds_read_b128 v[116:119], v141 offset:8192\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[44:47], v[8:11], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[44:47], v[12:15], a[108:111]\n" \
    "	ds_read_b128 v[120:123], v141 offset:10240\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[44:47], v[16:19], a[140:143]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[44:47], v[20:23], a[172:175]\n" \
    "	ds_read_b128 v[124:127], v141 offset:12288\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[44:47], v[24:27], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[44:47], v[28:31], a[236:239]\n" \
    "	ds_read_b128 v[128:131], v141 offset:14336\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[48:51], v[0:3], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[48:51], v[4:7], a[48:51]\n" \
    "	ds_read_b128 v[132:135], v141 offset:16384\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[48:51], v[8:11], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[48:51], v[12:15], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[48:51], v[16:19], a[144:147]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[48:51], v[20:23], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[48:51], v[24:27], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[48:51], v[28:31], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[52:55], v[0:3], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[52:55], v[4:7], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[52:55], v[8:11], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[52:55], v[12:15], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[52:55], v[16:19], a[148:151]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[52:55], v[20:23], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[52:55], v[24:27], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[52:55], v[28:31], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[56:59], v[0:3], a[24:27]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[56:59], v[4:7], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[56:59], v[8:11], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[56:59], v[12:15], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[56:59], v[16:19], a[152:155]\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[56:59], v[20:23], a[184:187]\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[56:59], v[24:27], a[216:219]\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[56:59], v[28:31], a[248:251]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[60:63], v[0:3], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[60:63], v[4:7], a[60:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[60:63], v[8:11], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[60:63], v[12:15], a[124:127]\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[60:63], v[16:19], a[156:159]\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[60:63], v[20:23], a[188:191]\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[60:63], v[24:27], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[60:63], v[28:31], a[252:255]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_0], v[64:67], v[0:3], %[c8_0]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_1], v[64:67], v[4:7], %[c8_1]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_2], v[64:67], v[8:11], %[c8_2]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_3], v[64:67], v[12:15], %[c8_3]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_4], v[64:67], v[16:19], %[c8_4]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_5], v[64:67], v[20:23], %[c8_5]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_6], v[64:67], v[24:27], %[c8_6]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_7], v[64:67], v[28:31], %[c8_7]\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	s_waitcnt lgkmcnt(15)\n" \
    "	v_mfma_i32_16x16x64_i8 a[0:3], v[100:103], v[68:71], a[0:3]\n" \
    "	s_waitcnt lgkmcnt(14)\n" \
    "	v_mfma_i32_16x16x64_i8 a[32:35], v[100:103], v[72:75], a[32:35]\n" \
    "	s_waitcnt lgkmcnt(13)\n" \
    "	v_mfma_i32_16x16x64_i8 a[64:67], v[100:103], v[76:79], a[64:67]\n" \
    "	s_waitcnt lgkmcnt(12)\n" \
    "	v_mfma_i32_16x16x64_i8 a[96:99], v[100:103], v[80:83], a[96:99]\n" \
    "	s_waitcnt lgkmcnt(11)\n" \
    "	v_mfma_i32_16x16x64_i8 a[128:131], v[100:103], v[84:87], a[128:131]\n" \
    "	s_waitcnt lgkmcnt(10)\n" \
    "	v_mfma_i32_16x16x64_i8 a[160:163], v[100:103], v[88:91], a[160:163]\n" \
    "	s_waitcnt lgkmcnt(9)\n" \
    "	v_mfma_i32_16x16x64_i8 a[192:195], v[100:103], v[92:95], a[192:195]\n" \
    "	s_waitcnt lgkmcnt(8)\n" \
    "	v_mfma_i32_16x16x64_i8 a[224:227], v[100:103], v[96:99], a[224:227]\n" \
    "	s_waitcnt lgkmcnt(7)\n" \
    "	v_mfma_i32_16x16x64_i8 a[4:7], v[104:107], v[68:71], a[4:7]\n" \
    "	v_mfma_i32_16x16x64_i8 a[36:39], v[104:107], v[72:75], a[36:39]\n" \
    "	v_mfma_i32_16x16x64_i8 a[68:71], v[104:107], v[76:79], a[68:71]\n" \
    "	v_mfma_i32_16x16x64_i8 a[100:103], v[104:107], v[80:83], a[100:103]\n" \
    "	v_mfma_i32_16x16x64_i8 a[132:135], v[104:107], v[84:87], a[132:135]\n" \
    "	v_mfma_i32_16x16x64_i8 a[164:167], v[104:107], v[88:91], a[164:167]\n" \
    "	v_mfma_i32_16x16x64_i8 a[196:199], v[104:107], v[92:95], a[196:199]\n" \
    "	v_mfma_i32_16x16x64_i8 a[228:231], v[104:107], v[96:99], a[228:231]\n" \
    "	s_waitcnt lgkmcnt(6)\n" \
    "	v_mfma_i32_16x16x64_i8 a[8:11], v[108:111], v[68:71], a[8:11]\n" \
    "	v_mfma_i32_16x16x64_i8 a[40:43], v[108:111], v[72:75], a[40:43]\n" \
    "	v_mfma_i32_16x16x64_i8 a[72:75], v[108:111], v[76:79], a[72:75]\n" \
    "	v_mfma_i32_16x16x64_i8 a[104:107], v[108:111], v[80:83], a[104:107]\n" \
    "	v_mfma_i32_16x16x64_i8 a[136:139], v[108:111], v[84:87], a[136:139]\n" \
    "	v_mfma_i32_16x16x64_i8 a[168:171], v[108:111], v[88:91], a[168:171]\n" \
    "	v_mfma_i32_16x16x64_i8 a[200:203], v[108:111], v[92:95], a[200:203]\n" \
    "	v_mfma_i32_16x16x64_i8 a[232:235], v[108:111], v[96:99], a[232:235]\n" \
    "	s_waitcnt lgkmcnt(5)\n" \
    "	v_mfma_i32_16x16x64_i8 a[12:15], v[112:115], v[68:71], a[12:15]\n" \
    "	v_mfma_i32_16x16x64_i8 a[44:47], v[112:115], v[72:75], a[44:47]\n" \
    "	v_mfma_i32_16x16x64_i8 a[76:79], v[112:115], v[76:79], a[76:79]\n" \
    "	v_mfma_i32_16x16x64_i8 a[108:111], v[112:115], v[80:83], a[108:111]\n" \
    "	v_mfma_i32_16x16x64_i8 a[140:143], v[112:115], v[84:87], a[140:143]\n" \
    "	v_mfma_i32_16x16x64_i8 a[172:175], v[112:115], v[88:91], a[172:175]\n" \
    "	v_mfma_i32_16x16x64_i8 a[204:207], v[112:115], v[92:95], a[204:207]\n" \
    "	v_mfma_i32_16x16x64_i8 a[236:239], v[112:115], v[96:99], a[236:239]\n" \
    "	s_waitcnt lgkmcnt(4)\n" \
    "	v_mfma_i32_16x16x64_i8 a[16:19], v[116:119], v[68:71], a[16:19]\n" \
    "	v_mfma_i32_16x16x64_i8 a[48:51], v[116:119], v[72:75], a[48:51]\n" \
    "	v_mfma_i32_16x16x64_i8 a[80:83], v[116:119], v[76:79], a[80:83]\n" \
    "	v_mfma_i32_16x16x64_i8 a[112:115], v[116:119], v[80:83], a[112:115]\n" \
    "	v_mfma_i32_16x16x64_i8 a[144:147], v[116:119], v[84:87], a[144:147]\n" \
    "	v_mfma_i32_16x16x64_i8 a[176:179], v[116:119], v[88:91], a[176:179]\n" \
    "	v_mfma_i32_16x16x64_i8 a[208:211], v[116:119], v[92:95], a[208:211]\n" \
    "	v_mfma_i32_16x16x64_i8 a[240:243], v[116:119], v[96:99], a[240:243]\n" \
    "	s_waitcnt lgkmcnt(3)\n" \
    "	v_mfma_i32_16x16x64_i8 a[20:23], v[120:123], v[68:71], a[20:23]\n" \
    "	v_mfma_i32_16x16x64_i8 a[52:55], v[120:123], v[72:75], a[52:55]\n" \
    "	v_mfma_i32_16x16x64_i8 a[84:87], v[120:123], v[76:79], a[84:87]\n" \
    "	v_mfma_i32_16x16x64_i8 a[116:119], v[120:123], v[80:83], a[116:119]\n" \
    "	v_mfma_i32_16x16x64_i8 a[148:151], v[120:123], v[84:87], a[148:151]\n" \
    "	v_mfma_i32_16x16x64_i8 a[180:183], v[120:123], v[88:91], a[180:183]\n" \
    "	v_mfma_i32_16x16x64_i8 a[212:215], v[120:123], v[92:95], a[212:215]\n" \
    "	v_mfma_i32_16x16x64_i8 a[244:247], v[120:123], v[96:99], a[244:247]\n" \
    "	s_waitcnt lgkmcnt(2)\n" \
    "	v_mfma_i32_16x16x64_i8 a[24:27], v[124:127], v[68:71], a[24:27]\n" \
    "	v_mfma_i32_16x16x64_i8 a[56:59], v[124:127], v[72:75], a[56:59]\n" \
    "	v_mfma_i32_16x16x64_i8 a[88:91], v[124:127], v[76:79], a[88:91]\n" \
    "	v_mfma_i32_16x16x64_i8 a[120:123], v[124:127], v[80:83], a[120:123]\n" \
    "	v_mfma_i32_16x16x64_i8 a[152:155], v[124:127], v[84:87], a[152:155]\n" \
    "	v_mfma_i32_16x16x64_i8 a[184:187], v[124:127], v[88:91], a[184:187]\n" \
    "	v_mfma_i32_16x16x64_i8 a[216:219], v[124:127], v[92:95], a[216:219]\n" \
    "	v_mfma_i32_16x16x64_i8 a[248:251], v[124:127], v[96:99], a[248:251]\n" \
    "	s_waitcnt lgkmcnt(1)\n" \
    "	v_mfma_i32_16x16x64_i8 a[28:31], v[128:131], v[68:71], a[28:31]\n" \
    "	v_mfma_i32_16x16x64_i8 a[60:63], v[128:131], v[72:75], a[60:63]\n" \
    "	v_mfma_i32_16x16x64_i8 a[92:95], v[128:131], v[76:79], a[92:95]\n" \
    "	v_mfma_i32_16x16x64_i8 a[124:127], v[128:131], v[80:83], a[124:127]\n" \
    "	v_mfma_i32_16x16x64_i8 a[156:159], v[128:131], v[84:87], a[156:159]\n" \
    "	v_mfma_i32_16x16x64_i8 a[188:191], v[128:131], v[88:91], a[188:191]\n" \
    "	v_mfma_i32_16x16x64_i8 a[220:223], v[128:131], v[92:95], a[220:223]\n" \
    "	v_mfma_i32_16x16x64_i8 a[252:255], v[128:131], v[96:99], a[252:255]\n" \
    "	s_waitcnt lgkmcnt(0)\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_0], v[132:135], v[68:71], %[c8_0]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_1], v[132:135], v[72:75], %[c8_1]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_2], v[132:135], v[76:79], %[c8_2]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_3], v[132:135], v[80:83], %[c8_3]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_4], v[132:135], v[84:87], %[c8_4]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_5], v[132:135], v[88:91], %[c8_5]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_6], v[132:135], v[92:95], %[c8_6]\n" \
    "	v_mfma_i32_16x16x64_i8 %[c8_7], v[132:135], v[96:99], %[c8_7]\n" \
    "DONE_%=:\n" \
    "	s_nop 15\n" \
    "	s_barrier\n" \
    "	s_mov_b32 m0, s66\n" \
      : [c8_0] "+v"(c8[0]), [c8_1] "+v"(c8[1]), [c8_2] "+v"(c8[2]), [c8_3] "+v"(c8[3]), [c8_4] "+v"(c8[4]), [c8_5] "+v"(c8[5]), [c8_6] "+v"(c8[6]), [c8_7] "+v"(c8[7]) \
      : [ap] "s"(ap), [wp] "s"(wp), [rsa] "s"(rsa), [rsw] "s"(rsw), [ra] "s"(ra), [rw] "s"(rw), [trips] "s"(trips), [rem] "s"(rem), [lds] "s"(lds), [wave] "s"(wave), [zero] "s"(zero) \
      : "memory", "vcc", "scc", "v0", "v1", "v2", "v3", "v4", "v5", "v6", "v7", "v8", "v9", "v10", "v11", "v12", "v13", "v14", "v15", "v16", "v17", "v18", "v19", "v20", "v21", "v22", "v23", "v24", "v25", "v26", "v27", "v28", "v29", "v30", "v31", "v32", "v33", "v34", "v35", "v36", "v37", "v38", "v39", "v40", "v41", "v42", "v43", "v44", "v45", "v46", "v47", "v48", "v49", "v50", "v51", "v52", "v53", "v54", "v55", "v56", "v57", "v58", "v59", "v60", "v61", "v62", "v63", "v64", "v65", "v66", "v67", "v68", "v69", "v70", "v71", "v72", "v73", "v74", "v75", "v76", "v77", "v78", "v79", "v80", "v81", "v82", "v83", "v84", "v85", "v86", "v87", "v88", "v89", "v90", "v91", "v92", "v93", "v94", "v95", "v96", "v97", "v98", "v99", "v100", "v101", "v102", "v103", "v104", "v105", "v106", "v107", "v108", "v109", "v110", "v111", "v112", "v113", "v114", "v115", "v116", "v117", "v118", "v119", "v120", "v121", "v122", "v123", "v124", "v125", "v126", "v127", "v128", "v129", "v130", "v131", "v132", "v133", "v134", "v135", "v136", "v137", "v138", "v139", "v140", "v141", "v142", "v143", "v144", "v145", "v146", "v147", "v148", "v149", "v150", "v151", "v152", "v153", "v154", "v155", "v156", "v157", "v158", "v159", "v160", "v161", "v162", "v163", "v164", "v165", "v166", "v167", "v168", "v169", "a0", "a1", "a2", "a3", "a4", "a5", "a6", "a7", "a8", "a9", "a10", "a11", "a12", "a13", "a14", "a15", "a16", "a17", "a18", "a19", "a20", "a21", "a22", "a23", "a24", "a25", "a26", "a27", "a28", "a29", "a30", "a31", "a32", "a33", "a34", "a35", "a36", "a37", "a38", "a39", "a40", "a41", "a42", "a43", "a44", "a45", "a46", "a47", "a48", "a49", "a50", "a51", "a52", "a53", "a54", "a55", "a56", "a57", "a58", "a59", "a60", "a61", "a62", "a63", "a64", "a65", "a66", "a67", "a68", "a69", "a70", "a71", "a72", "a73", "a74", "a75", "a76", "a77", "a78", "a79", "a80", "a81", "a82", "a83", "a84", "a85", "a86", "a87", "a88", "a89", "a90", "a91", "a92", "a93", "a94", "a95", "a96", "a97", "a98", "a99", "a100", "a101", "a102", "a103", "a104", "a105", "a106", "a107", "a108", "a109", "a110", "a111", "a112", "a113", "a114", "a115", "a116", "a117", "a118", "a119", "a120", "a121", "a122", "a123", "a124", "a125", "a126", "a127", "a128", "a129", "a130", "a131", "a132", "a133", "a134", "a135", "a136", "a137", "a138", "a139", "a140", "a141", "a142", "a143", "a144", "a145", "a146", "a147", "a148", "a149", "a150", "a151", "a152", "a153", "a154", "a155", "a156", "a157", "a158", "a159", "a160", "a161", "a162", "a163", "a164", "a165", "a166", "a167", "a168", "a169", "a170", "a171", "a172", "a173", "a174", "a175", "a176", "a177", "a178", "a179", "a180", "a181", "a182", "a183", "a184", "a185", "a186", "a187", "a188", "a189", "a190", "a191", "a192", "a193", "a194", "a195", "a196", "a197", "a198", "a199", "a200", "a201", "a202", "a203", "a204", "a205", "a206", "a207", "a208", "a209", "a210", "a211", "a212", "a213", "a214", "a215", "a216", "a217", "a218", "a219", "a220", "a221", "a222", "a223", "a224", "a225", "a226", "a227", "a228", "a229", "a230", "a231", "a232", "a233", "a234", "a235", "a236", "a237", "a238", "a239", "a240", "a241", "a242", "a243", "a244", "a245", "a246", "a247", "a248", "a249", "a250", "a251", "a252", "a253", "a254", "a255", "s60", "s61", "s62", "s63", "s64", "s65", "s66", "s67", "s68", "s69")
