// 8-bit matrices with a power-of-two scale for each block of 128 values of a row: the format, its conversions, and the launchers.
//
// A matrix of R rows and C columns is q [R, ld] (e4m3 or e5m2 bytes, ld >= the columns rounded up to 128, the columns behind C zero) and
// s [blocks, lds] (one byte E8M0, 2^(byte - 127), for row r and block b at s[b * lds + r]).  The scale of a block is the smallest power of
// two, not below 2^-126, for which the block's largest finite magnitude fits the type; 2^0 for a block without one.  Why powers of two:
//  * v_mfma_scale_f32_16x16x128_f8f6f4 takes one with every operand row of its 128 values of k, so that a product's scales cost no
//    vector instruction (with fp32 scales every accumulator would be added to by the vector ALU once per block);
//  * a value's position between the numbers of the type does not depend on the scale: rows quantized along their columns and along their
//    rows hold the same values, but for those below 2^-13 (e4m3; e5m2: 2^-28) of their block's largest, which lose bits or vanish;
//  * the values a block stands for are bf16 numbers where its scale is 2^-117 or more, or where it was made from bf16 (2^128, to which magnitudes
//    from 1.9375 2^127 on round, aside): restoring them rounds nothing.  The norm's output goes into 8 bits from fp32; e4m3's smallest number
//    at the smallest scale, 2^-135, lies below bf16's, 2^-133.
// Scales of the rows of a block lie side by side because a tile of a product reads them for many rows and one block at a time.
#pragma once
#include "common.h"

namespace elf {

enum Fp8Format { FP8_E4M3 = 0, FP8_E5M2 = 1 };
constexpr int FP8_BLOCK = 128;

// x [T, C] (bf16, rows ldx apart) -> its rows in 8 bits (q, s) and / or its columns (qt [C, ldqt], st); square: one scale for 128 x 128.
int quant_fp8(const void* x, int64_t ldx, int64_t T, int64_t C, int fmt, int square, void* q, int64_t ldq, void* s, int64_t lds, void* qt, int64_t ldqt, void* st,
              int64_t ldst, hipStream_t stream);
// The 8-bit rows of a [T, C] matrix -> those of its transpose.
int transpose_fp8(const void* q, int64_t ldq, const void* s, int64_t lds, int64_t T, int64_t C, int fmt, void* qt, int64_t ldqt, void* st, int64_t ldst, hipStream_t stream);
int dequant_fp8(const void* q, int64_t ldq, const void* s, int64_t lds, int64_t T, int64_t C, int fmt, void* x, int64_t ldx, hipStream_t stream);
int rms_norm_fp8(const void* x, const void* residual, const void* gamma, void* h, void* q, int64_t ldq, void* s, int64_t lds, void* stats, int64_t T, int d, float eps,
                 int fmt, hipStream_t stream);
// C [M, N] (+)= A B^T, both of K columns; B is e4m3.  epi: an EPI_ of kernels.h, 0 to 3.
int gemm_fp8(int64_t M, int64_t N, int64_t K, int fmt_a, const void* A, int64_t lda, const void* sa, int64_t ldsa, const void* B, int64_t ldb, const void* sb, int64_t ldsb,
             void* C, int64_t ldc, int epi, const void* R, int64_t ldr, float* workspace, int64_t workspace_floats, hipStream_t stream);
// The workspace with which K is shared among workgroups where that is faster (0: it is not), and the way that a product takes: {rows and columns
// of a workgroup's tile, K ranges}.
int64_t gemm_fp8_workspace_floats(int64_t M, int64_t N, int64_t K);
int gemm_fp8_way(int64_t M, int64_t N, int64_t K, int64_t workspace_floats, int* way);

#ifdef __HIPCC__
// The scale's byte for a block whose largest finite magnitude times 2^-UP has these fp32 bits: top = 1.m 2^p fits up to 1.75 2^8 (e5m2:
// 1.75 2^15); the sum carries into the exponent where m > 0.75.
template <int FMT, int UP = 0>
__device__ __forceinline__ uint32_t fp8_scale_byte(uint32_t top_bits) {
	const int e = (int)((top_bits + 0x1fffffu) >> 23) - (FMT == FP8_E4M3 ? 8 : 15) + UP;
	return top_bits == 0 ? 127u : (uint32_t)(e < 1 ? 1 : e);
}
// 2^(127 - byte) (bytes 1 .. 253)
__device__ __forceinline__ float fp8_inverse(uint32_t byte) { return __builtin_bit_cast(float, (254u - byte) << 23); }
// What a block holds whose scale is not a number (byte 255): NaN in either type.
__device__ __forceinline__ uint32_t fp8_or_nan(uint32_t w, uint32_t scale_byte) { return scale_byte == 255u ? 0x7f7f7f7fu : w; }
// The scale itself, of any byte: 2^-127 is a subnormal number, 255 is not a number.
__device__ __forceinline__ float fp8_scale(uint32_t byte) { return __builtin_bit_cast(float, byte << 23 | (((byte + 1u) & 0xffu) < 2u ? 0x400000u : 0u)); }
// |v| as fp32 bits, 0 where v is no finite number
__device__ __forceinline__ uint32_t fp8_magnitude(float v) {
	const uint32_t a = __builtin_bit_cast(uint32_t, v) & 0x7fffffffu;
	return a < 0x7f800000u ? a : 0u;
}
// Four values as bytes, rounded to nearest even (the scale leaves none too large).  Not a number stays that; an infinity becomes it in
// e4m3, which has none.
template <int FMT>
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
	int w = 0;
	if constexpr (FMT == FP8_E4M3) {
		w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, false);
		w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
	} else {
		w = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, w, false);
		w = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, w, true);
	}
	return (uint32_t)w;
}
template <int FMT>
__device__ __forceinline__ void fp8_unpack4(uint32_t w, float (&v)[4]) {
	if constexpr (FMT == FP8_E4M3) {
		const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
		v[0] = lo[0], v[1] = lo[1], v[2] = hi[0], v[3] = hi[1];
	} else {
		const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_bf8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_bf8((int)w, true);
		v[0] = lo[0], v[1] = lo[1], v[2] = hi[0], v[3] = hi[1];
	}
}
// rows that start at any element: the memory system takes 16-byte accesses at any address
typedef bf16x8 bf16x8_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));

// Rows of bf16 that start between dwords (an odd number of columns).  A 16-byte store there costs much more than one that starts with a dword, so
// such lanes store one element later: the first element of the next lane's run is the last of theirs.  us, before -> after, and with rows on
// dwords: a product 2111 x 4287 x 1599 30.1 -> 25.0 (24.3), 8192 x 14335 out of 8 bits 107 -> 96 (85).  (Loads gain nothing by it.)
__device__ __forceinline__ bool between_dwords(const void* p) { return ((uintptr_t)p & 2) != 0; }
typedef u32x4 u32x4_any __attribute__((aligned(4)));
// 8 neighbouring elements w at p, where lanes between dwords leave their first to the lane before them (unless `first`) and take `next`, the
// first element of the lane behind them (unless `last`)
__device__ __forceinline__ void store_shifted(bf16_t* p, const u32x4& w, uint32_t next, bool first, bool last) {
	const bool sh = between_dwords(p);
	u32x4 v;
#pragma unroll
	for (int i = 0; i < 4; i++) v[i] = sh ? __builtin_amdgcn_alignbit(i < 3 ? w[i + 1] : next, w[i], 16) : w[i];
	if (sh && first) *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
	uint32_t* d = reinterpret_cast<uint32_t*>(p + (sh ? 1 : 0));
	if (sh && last) {
		d[0] = v[0], d[1] = v[1], d[2] = v[2];
		*reinterpret_cast<uint16_t*>(d + 3) = (uint16_t)v[3];
	} else {
		*reinterpret_cast<u32x4_any*>(d) = v;
	}
}

template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
	const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
	return v > o ? v : o;
}
// the largest of 8 and of 16 neighbouring lanes, in all of them
__device__ __forceinline__ uint32_t max_of_8(uint32_t v) {
	v = max_dpp<0xB1>(v);   // quad_perm 1 0 3 2
	v = max_dpp<0x4E>(v);   // quad_perm 2 3 0 1
	return max_dpp<0x141>(v);  // row_half_mirror
}
__device__ __forceinline__ uint32_t max_of_16(uint32_t v) { return max_dpp<0x140>(max_of_8(v)); }  // row_mirror
#endif

}  // namespace elf
