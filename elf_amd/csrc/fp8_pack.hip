// Into 8 bits and out of them: activations, gradients and weights, the transpose of an 8-bit matrix, and the root-mean-square norm that adds
// the residual and leaves in 8 bits.  The format is fp8.h's.  All of these are bound by memory; every input is read once.
#include "fp8.h"
#include "kernels.h"

namespace elf {

struct PackArgs {
	const void* x;
	int64_t ldx;
	const uint8_t* sx;  // 8-bit sources: their scales
	int64_t ldsx;
	uint8_t* q;
	int64_t ldq;
	uint8_t* s;
	int64_t lds;
	uint8_t* qt;
	int64_t ldqt;
	uint8_t* st;
	int64_t ldst;
	int64_t T, C;
	uint32_t col_blocks;
	bool between;  // rows of the bf16 output start between dwords
};

constexpr int SRC_BF16 = 2;  // (FP8_E4M3 and FP8_E5M2 are the other sources)
// 8-bit sources are held as a quarter of their values where they go into 8 bits again: the largest magnitudes of bf16 round to 2^128, which
// fp32 has not, and a quarter of the smallest is still exact.
constexpr int quartered(int src) { return src == SRC_BF16 ? 0 : 2; }

// 16 neighbouring values of row `row` from column `col` on, times 2^-UP; zeros outside the matrix
template <int SRC, int UP = 0>
__device__ __forceinline__ void load16(const PackArgs& g, int64_t row, int64_t col, float (&v)[16]) {
#pragma unroll
	for (int j = 0; j < 16; j++) v[j] = 0.f;
	if (row >= g.T || col >= g.C) return;
	if constexpr (SRC == SRC_BF16) {
		const bf16_t* p = reinterpret_cast<const bf16_t*>(g.x) + row * g.ldx + col;
		if (col + 16 <= g.C) {
			const bf16x8 a = *reinterpret_cast<const bf16x8_any*>(p), b = *reinterpret_cast<const bf16x8_any*>(p + 8);
#pragma unroll
			for (int j = 0; j < 8; j++) v[j] = (float)a[j], v[8 + j] = (float)b[j];
		} else {
#pragma unroll
			for (int j = 0; j < 15; j++)
				if (col + j < g.C) v[j] = (float)p[j];
		}
	} else {
		const u32x4 w = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint8_t*>(g.x) + row * g.ldx + col);
		const uint32_t byte = g.sx[(col >> 7) * g.ldsx + row];
		const int e = (int)byte - 127 - UP;
#pragma unroll
		for (int i = 0; i < 4; i++) {
			float u[4];
			fp8_unpack4<SRC>(fp8_or_nan(w[i], byte), u);
#pragma unroll
			for (int j = 0; j < 4; j++) v[i * 4 + j] = col + i * 4 + j < g.C ? __builtin_ldexpf(u[j], e) : 0.f;
		}
	}
}

// One workgroup: a square of 128 x 128 values, read once and held in registers: thread t has 16 columns of 4 rows.  Rows: the eight threads of
// a row find its largest magnitude among themselves and store its 128 bytes together.  Columns: largest magnitudes over the square's rows
// through LDS, then the bytes (a thread has 4 consecutive ones of each of its 16 columns) cross the square through LDS and leave as 128-byte
// runs along the rows' index, zeros behind the last row.  The square is the unit because a block's 128 scales, and 128 bytes of either
// layout, are then one whole cache line that one workgroup writes.
template <int SRC, int DST, bool ROWS, bool COLS, bool SQUARE>
__global__ __launch_bounds__(256) void pack_kernel(PackArgs g) {
	__shared__ uint32_t part[COLS ? 16 : 1][COLS ? 128 : 4];
	__shared__ __attribute__((aligned(16))) uint8_t row_byte[128];
	__shared__ __attribute__((aligned(16))) uint8_t col_byte[COLS ? 128 : 16];
	__shared__ __attribute__((aligned(16))) uint8_t tile[COLS ? 128 * 128 : 16];
	constexpr int UP = quartered(SRC);
	static_assert(UP == 0 || (COLS && !ROWS && !SQUARE), "8-bit sources are transposed");
	const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
	const int c = tid & 7, rq = tid >> 3;
	const int64_t cb = blockIdx.x % g.col_blocks, rb = blockIdx.x / g.col_blocks;
	const int64_t row0 = rb * 128 + rq * 4, col0 = cb * 128 + c * 16;
	float v[4][16];
#pragma unroll
	for (int p = 0; p < 4; p++) load16<SRC, UP>(g, row0 + p, col0, v[p]);

	uint32_t rmax[4], cmax[16];
#pragma unroll
	for (int p = 0; p < 4; p++) {
		rmax[p] = 0;
#pragma unroll
		for (int j = 0; j < 16; j++) {
			const uint32_t a = fp8_magnitude(v[p][j]);
			rmax[p] = max(rmax[p], a);
			if constexpr (COLS && !SQUARE) cmax[j] = p == 0 ? a : max(cmax[j], a);
		}
	}
	uint32_t square_byte = 127;
	if constexpr (SQUARE) {
		uint32_t m = max(max(rmax[0], rmax[1]), max(rmax[2], rmax[3]));
		m = max_of_16(m);
		m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
		m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
		if (lane == 0) part[0][wave] = m;
		__syncthreads();
		square_byte = fp8_scale_byte<DST>(max(max(part[0][0], part[0][1]), max(part[0][2], part[0][3])));
	}
	if constexpr (ROWS) {
#pragma unroll
		for (int p = 0; p < 4; p++) {
			const uint32_t byte = SQUARE ? square_byte : fp8_scale_byte<DST>(max_of_8(rmax[p]));
			const float inv = fp8_inverse(byte);
			u32x4 w;
#pragma unroll
			for (int i = 0; i < 4; i++) w[i] = fp8_pack4<DST>(v[p][i * 4] * inv, v[p][i * 4 + 1] * inv, v[p][i * 4 + 2] * inv, v[p][i * 4 + 3] * inv);
			if (row0 + p < g.T) *reinterpret_cast<u32x4*>(g.q + (row0 + p) * g.ldq + col0) = w;
			if (c == 0) row_byte[rq * 4 + p] = (uint8_t)byte;
		}
	}
	if constexpr (COLS) {
		if constexpr (!SQUARE) {
#pragma unroll
			for (int j = 0; j < 16; j++) cmax[j] = max_dpp<0x128>(cmax[j]);  // row_ror 8: the other half of 16 lanes has four rows more
			if ((lane & 8) == 0) {
#pragma unroll
				for (int i = 0; i < 4; i++) *reinterpret_cast<u32x4*>(&part[wave * 4 + (lane >> 4)][c * 16 + i * 4]) = u32x4{cmax[i * 4], cmax[i * 4 + 1], cmax[i * 4 + 2], cmax[i * 4 + 3]};
			}
			__syncthreads();
			if (tid < 128) {
				uint32_t m = 0;
#pragma unroll
				for (int i = 0; i < 16; i++) m = max(m, part[i][tid]);
				col_byte[tid] = (uint8_t)fp8_scale_byte<DST, UP>(m);
			}
		} else if (tid < 128) {
			col_byte[tid] = (uint8_t)square_byte;
		}
		__syncthreads();
		const u32x4 bytes = *reinterpret_cast<const u32x4*>(col_byte + c * 16);
		// dword t / 4 of column j lies in 16-byte chunk (t / 16) ^ (j / 16): without the swizzle the eight threads of a row would meet in one bank
#pragma unroll
		for (int j = 0; j < 16; j++) {
			const uint32_t byte = (bytes[j >> 2] >> (8 * (j & 3))) & 0xffu;
			float u[4];
#pragma unroll
			for (int p = 0; p < 4; p++) u[p] = UP ? __builtin_ldexpf(v[p][j], 127 - (int)byte + UP) : v[p][j] * fp8_inverse(byte);
			*reinterpret_cast<uint32_t*>(tile + (c * 16 + j) * 128 + (((rq >> 2) ^ c) << 4) + (rq & 3) * 4) = fp8_pack4<DST>(u[0], u[1], u[2], u[3]);
		}
	}
	__syncthreads();
	if constexpr (ROWS) {
		if (tid < 128 && rb * 128 + tid < g.T) g.s[cb * g.lds + rb * 128 + tid] = row_byte[tid];
	}
	if constexpr (COLS) {
#pragma unroll
		for (int i = 0; i < 4; i++) {
			const int col = i * 32 + (tid >> 3), chunk = tid & 7;
			if (cb * 128 + col < g.C)
				*reinterpret_cast<u32x4*>(g.qt + (cb * 128 + col) * g.ldqt + rb * 128 + chunk * 16) = *reinterpret_cast<const u32x4*>(tile + col * 128 + ((chunk ^ (col >> 4)) << 4));
		}
		if (tid < 128 && cb * 128 + tid < g.C) g.st[rb * g.ldst + cb * 128 + tid] = col_byte[tid];
	}
}

// Out of 8 bits: 16 lanes a row of a square, 8 values each, so that a row leaves as 256 contiguous bytes.  The factor rounds nothing (fp32 has
// 2^-127 times either type's smallest number, 2^-143); bf16 rounds what its subnormal numbers do not hold, where a scale is below 2^-117.
template <int FMT>
__global__ __launch_bounds__(256) void dequant_kernel(PackArgs g, bf16_t* out, int64_t ldo) {
	const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
	const int64_t cb = blockIdx.x % g.col_blocks, rb = blockIdx.x / g.col_blocks;
	const int64_t col = cb * 128 + c * 8;
	u32x2 raw[8];
	uint32_t byte[8];
#pragma unroll
	for (int p = 0; p < 8; p++) {
		const int64_t row = min(rb * 128 + p * 16 + r, g.T - 1);
		raw[p] = *reinterpret_cast<const u32x2*>(reinterpret_cast<const uint8_t*>(g.x) + row * g.ldx + col);
		byte[p] = g.sx[cb * g.ldsx + row];
	}
#pragma unroll
	for (int p = 0; p < 8; p++) {
		const int64_t row = rb * 128 + p * 16 + r;
		float u[2][4];
		fp8_unpack4<FMT>(raw[p][0], u[0]);
		fp8_unpack4<FMT>(raw[p][1], u[1]);
		const float scale = fp8_scale(byte[p]);
		bf16x8 o;
#pragma unroll
		for (int j = 0; j < 8; j++) o[j] = (bf16_t)(u[j >> 2][j & 3] * scale);  // (2^128 becomes an infinity)
		const u32x4 v = __builtin_bit_cast(u32x4, o);
		uint32_t next = 0;
		if (g.between) next = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v[0], 0x101, 0xf, 0xf, false);  // row_shl 1: the lane behind
		if (row >= g.T) continue;
		bf16_t* d = out + row * ldo + col;
		if (col + 8 <= g.C) {
			if (g.between) store_shifted(d, v, next, c == 0, c == 15 || col + 8 == g.C);
			else *reinterpret_cast<u32x4_any*>(d) = v;
		} else {
#pragma unroll
			for (int j = 0; j < 7; j++)
				if (col + j < g.C) d[j] = o[j];
		}
	}
}

// h = x + residual (rounded to bf16: what the residual stream keeps is what is normalized), y = h * rsqrt(mean(h^2) + eps) * gamma, and y goes
// into 8 bits straight from fp32: it is rounded once.  One wave a row, or four where the row is longer than 2048; a thread holds chunks of 8
// values, a block of 128 is 16 neighbouring lanes.  h may be x's or the residual's memory: a thread reads all of its chunks before it writes one.
template <int NCH, int WPR, int FMT>
__global__ __launch_bounds__(256) void rms_norm_fp8_kernel(const bf16_t* x, const bf16_t* residual, const bf16_t* __restrict__ gamma, bf16_t* h,
                                                           uint8_t* __restrict__ q, int64_t ldq, uint8_t* __restrict__ s, int64_t lds, float2* __restrict__ stats,
                                                           int64_t T, int d, float eps) {
	__shared__ float red[4];
	const int wave = threadIdx.x >> 6;
	const int tr = WPR == 1 ? (threadIdx.x & 63) : threadIdx.x;
	constexpr int TPR = 64 * WPR;
	const int64_t row = WPR == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
	if (row >= T) return;  // whole waves (WPR 1) or whole workgroups
	const int nchunks = d >> 3, padded = (d + 127) / 128 * 16;
	bf16x8 o[NCH], r[NCH];
#pragma unroll
	for (int i = 0; i < NCH; i++) {
		const int ch = tr + i * TPR;
		if (ch < nchunks) {
			o[i] = *reinterpret_cast<const bf16x8*>(x + row * d + ch * 8);
			if (residual) r[i] = *reinterpret_cast<const bf16x8*>(residual + row * d + ch * 8);
		}
	}
	float v[NCH][8];
	float ss = 0.f;
#pragma unroll
	for (int i = 0; i < NCH; i++) {
		const int ch = tr + i * TPR;
#pragma unroll
		for (int j = 0; j < 8; j++) v[i][j] = 0.f;
		if (ch < nchunks) {
			if (residual) {
#pragma unroll
				for (int j = 0; j < 8; j++) o[i][j] = (bf16_t)((float)o[i][j] + (float)r[i][j]);
				*reinterpret_cast<bf16x8*>(h + row * d + ch * 8) = o[i];
			}
#pragma unroll
			for (int j = 0; j < 8; j++) {
				v[i][j] = (float)o[i][j];
				ss += v[i][j] * v[i][j];
			}
		}
	}
	ss = wave_sum(ss);
	if constexpr (WPR > 1) {
		if ((threadIdx.x & 63) == 0) red[wave] = ss;
		__syncthreads();
		ss = red[0] + red[1] + red[2] + red[3];
	}
	const float rstd = rsqrtf(ss / d + eps);
	if (tr == 0) stats[row] = make_float2(0.f, rstd);
#pragma unroll
	for (int i = 0; i < NCH; i++) {
		const int ch = tr + i * TPR;
		uint32_t top = 0;
		if (ch < nchunks) {
			const bf16x8 g = *reinterpret_cast<const bf16x8*>(gamma + ch * 8);
#pragma unroll
			for (int j = 0; j < 8; j++) {
				v[i][j] = v[i][j] * rstd * (float)g[j];
				top = max(top, fp8_magnitude(v[i][j]));
			}
		}
		const uint32_t byte = fp8_scale_byte<FMT>(max_of_16(top));
		const float inv = fp8_inverse(byte);
		if (ch < padded) {
			u32x2 w;
#pragma unroll
			for (int k = 0; k < 2; k++) w[k] = fp8_pack4<FMT>(v[i][k * 4] * inv, v[i][k * 4 + 1] * inv, v[i][k * 4 + 2] * inv, v[i][k * 4 + 3] * inv);
			*reinterpret_cast<u32x2*>(q + row * ldq + ch * 8) = w;
			if ((ch & 15) == 0) s[(int64_t)(ch >> 4) * lds + row] = (uint8_t)byte;
		}
	}
}

// ------------------------------------------------------------------------------------------------ launchers
static bool rows_fit(const void* q, int64_t ld, const void* s, int64_t lds, int64_t rows, int64_t cols) {
	return q && s && ld >= (cols + 127) / 128 * 128 && ld % 16 == 0 && ((uintptr_t)q % 16) == 0 && lds >= rows && lds % 16 == 0 && ((uintptr_t)s % 16) == 0;
}
#define FP8_ROWS_RULE "rows of at least the columns rounded up to 128, scales of at least the rows, both a multiple of 16 bytes apart and 16-byte aligned"

static int pack_grid(int64_t T, int64_t C, uint32_t& col_blocks, uint32_t& tiles) {
	const int64_t cb = (C + 127) / 128, rb = (T + 127) / 128;
	constexpr int64_t MOST = (int64_t(1) << 24) - 1;  // workgroups of 256 threads: a grid has less than 2^32
	ELF_REQUIRE(cb <= MOST && rb <= MOST && cb * rb <= MOST, "fp8: %lld x %lld is too large for one launch", (long long)T, (long long)C);
	col_blocks = (uint32_t)cb, tiles = (uint32_t)(cb * rb);
	return 0;
}

template <int SRC, int DST>
static int launch_pack(const PackArgs& g, uint32_t tiles, bool rows, bool cols, bool square, hipStream_t stream) {
	const dim3 grid(tiles), block(256);
	if constexpr (SRC == SRC_BF16 && DST == FP8_E4M3) {
		if (square) {
			if (rows && cols) ELF_LAUNCH((pack_kernel<SRC, DST, true, true, true>), grid, block, 0, stream, g);
			else if (rows) ELF_LAUNCH((pack_kernel<SRC, DST, true, false, true>), grid, block, 0, stream, g);
			else ELF_LAUNCH((pack_kernel<SRC, DST, false, true, true>), grid, block, 0, stream, g);
			ELF_CHECK_HIP(hipGetLastError());
			return 0;
		}
	}
	if constexpr (SRC == SRC_BF16) {
		if (rows && cols) ELF_LAUNCH((pack_kernel<SRC, DST, true, true, false>), grid, block, 0, stream, g);
		else if (rows) ELF_LAUNCH((pack_kernel<SRC, DST, true, false, false>), grid, block, 0, stream, g);
		else ELF_LAUNCH((pack_kernel<SRC, DST, false, true, false>), grid, block, 0, stream, g);
	} else {
		ELF_LAUNCH((pack_kernel<SRC, DST, false, true, false>), grid, block, 0, stream, g);
	}
	ELF_CHECK_HIP(hipGetLastError());
	return 0;
}

int quant_fp8(const void* x, int64_t ldx, int64_t T, int64_t C, int fmt, int square, void* q, int64_t ldq, void* s, int64_t lds, void* qt, int64_t ldqt, void* st,
              int64_t ldst, hipStream_t stream) {
	ELF_REQUIRE(T > 0 && C > 0 && x, "quant_fp8: empty matrix or null pointer");
	ELF_REQUIRE(ldx >= C && ((uintptr_t)x % 2) == 0, "quant_fp8: rows of x overlap or x is not 2-byte aligned");
	ELF_REQUIRE(fmt == FP8_E4M3 || fmt == FP8_E5M2, "quant_fp8: unknown format %d", fmt);
	ELF_REQUIRE(!square || fmt == FP8_E4M3, "quant_fp8: squares of 128 x 128 (weights) are e4m3");
	ELF_REQUIRE(q || qt, "quant_fp8: neither rows nor columns are asked for");
	ELF_REQUIRE(!q || rows_fit(q, ldq, s, lds, T, C), "quant_fp8: bad row output: " FP8_ROWS_RULE);
	ELF_REQUIRE(!qt || rows_fit(qt, ldqt, st, ldst, C, T), "quant_fp8: bad column output: " FP8_ROWS_RULE);
	PackArgs g{x, ldx, nullptr, 0, (uint8_t*)q, ldq, (uint8_t*)s, lds, (uint8_t*)qt, ldqt, (uint8_t*)st, ldst, T, C, 0, false};
	uint32_t tiles;
	if (int rc = pack_grid(T, C, g.col_blocks, tiles)) return rc;
	if (fmt == FP8_E4M3) return launch_pack<SRC_BF16, FP8_E4M3>(g, tiles, q, qt, square != 0, stream);
	return launch_pack<SRC_BF16, FP8_E5M2>(g, tiles, q, qt, false, stream);
}

int transpose_fp8(const void* q, int64_t ldq, const void* s, int64_t lds, int64_t T, int64_t C, int fmt, void* qt, int64_t ldqt, void* st, int64_t ldst, hipStream_t stream) {
	ELF_REQUIRE(T > 0 && C > 0, "transpose_fp8: empty matrix");
	ELF_REQUIRE(fmt == FP8_E4M3 || fmt == FP8_E5M2, "transpose_fp8: unknown format %d", fmt);
	ELF_REQUIRE(rows_fit(q, ldq, s, lds, T, C), "transpose_fp8: bad input: " FP8_ROWS_RULE);
	ELF_REQUIRE(rows_fit(qt, ldqt, st, ldst, C, T), "transpose_fp8: bad output: " FP8_ROWS_RULE);
	PackArgs g{q, ldq, (const uint8_t*)s, lds, nullptr, 0, nullptr, 0, (uint8_t*)qt, ldqt, (uint8_t*)st, ldst, T, C, 0, false};
	uint32_t tiles;
	if (int rc = pack_grid(T, C, g.col_blocks, tiles)) return rc;
	if (fmt == FP8_E4M3) return launch_pack<FP8_E4M3, FP8_E4M3>(g, tiles, false, true, false, stream);
	return launch_pack<FP8_E5M2, FP8_E5M2>(g, tiles, false, true, false, stream);
}

int dequant_fp8(const void* q, int64_t ldq, const void* s, int64_t lds, int64_t T, int64_t C, int fmt, void* x, int64_t ldx, hipStream_t stream) {
	ELF_REQUIRE(T > 0 && C > 0 && x, "dequant_fp8: empty matrix or null pointer");
	ELF_REQUIRE(fmt == FP8_E4M3 || fmt == FP8_E5M2, "dequant_fp8: unknown format %d", fmt);
	ELF_REQUIRE(rows_fit(q, ldq, s, lds, T, C), "dequant_fp8: bad input: " FP8_ROWS_RULE);
	ELF_REQUIRE(ldx >= C && ((uintptr_t)x % 2) == 0, "dequant_fp8: rows of the output overlap or it is not 2-byte aligned");
	PackArgs g{q, ldq, (const uint8_t*)s, lds, nullptr, 0, nullptr, 0, nullptr, 0, nullptr, 0, T, C, 0, ldx % 2 != 0 || (uintptr_t)x % 4 != 0};
	uint32_t tiles;
	if (int rc = pack_grid(T, C, g.col_blocks, tiles)) return rc;
	if (fmt == FP8_E4M3) ELF_LAUNCH(dequant_kernel<FP8_E4M3>, dim3(tiles), dim3(256), 0, stream, g, (bf16_t*)x, ldx);
	else ELF_LAUNCH(dequant_kernel<FP8_E5M2>, dim3(tiles), dim3(256), 0, stream, g, (bf16_t*)x, ldx);
	ELF_CHECK_HIP(hipGetLastError());
	return 0;
}

template <int NCH, int WPR>
static int launch_norm(const void* x, const void* residual, const void* gamma, void* h, void* q, int64_t ldq, void* s, int64_t lds, void* stats, int64_t T, int d, float eps,
                       int fmt, hipStream_t stream) {
	const dim3 grid((uint32_t)(WPR == 1 ? (T + 3) / 4 : T)), block(256);
	if (fmt == FP8_E4M3)
		ELF_LAUNCH((rms_norm_fp8_kernel<NCH, WPR, FP8_E4M3>), grid, block, 0, stream, (const bf16_t*)x, (const bf16_t*)residual, (const bf16_t*)gamma, (bf16_t*)h, (uint8_t*)q, ldq,
		           (uint8_t*)s, lds, (float2*)stats, T, d, eps);
	else
		ELF_LAUNCH((rms_norm_fp8_kernel<NCH, WPR, FP8_E5M2>), grid, block, 0, stream, (const bf16_t*)x, (const bf16_t*)residual, (const bf16_t*)gamma, (bf16_t*)h, (uint8_t*)q, ldq,
		           (uint8_t*)s, lds, (float2*)stats, T, d, eps);
	ELF_CHECK_HIP(hipGetLastError());
	return 0;
}

int rms_norm_fp8(const void* x, const void* residual, const void* gamma, void* h, void* q, int64_t ldq, void* s, int64_t lds, void* stats, int64_t T, int d, float eps,
                 int fmt, hipStream_t stream) {
	ELF_REQUIRE(T > 0 && d > 0 && d % 8 == 0 && d <= 8192, "rms_norm_fp8: rows must be a multiple of 8 wide and at most 8192 (T=%lld d=%d)", (long long)T, d);
	ELF_REQUIRE(T < (int64_t(1) << 24), "rms_norm_fp8: %lld rows are too many for one launch", (long long)T);  // (a workgroup of 256 threads a row)
	ELF_REQUIRE(x && gamma && stats && (!residual || h), "rms_norm_fp8: null pointer");
	ELF_REQUIRE(((uintptr_t)x % 16) == 0 && ((uintptr_t)gamma % 16) == 0 && ((uintptr_t)residual % 16) == 0 && ((uintptr_t)h % 16) == 0 && ((uintptr_t)stats % 8) == 0,
	            "rms_norm_fp8: operands must be 16-byte aligned");
	ELF_REQUIRE(fmt == FP8_E4M3 || fmt == FP8_E5M2, "rms_norm_fp8: unknown format %d", fmt);
	ELF_REQUIRE(rows_fit(q, ldq, s, lds, T, d), "rms_norm_fp8: bad output: " FP8_ROWS_RULE);
	ProfScope prof(PROF_NORM_FWD, (residual ? 7.0 : 3.0) * T * d, stream);
#define ELF_NORM8(N, W) return launch_norm<N, W>(x, residual, gamma, h, q, ldq, s, lds, stats, T, d, eps, fmt, stream)
	const int chunks = (d + 127) / 128 * 16;
	if (chunks <= 64) ELF_NORM8(1, 1);
	if (chunks <= 128) ELF_NORM8(2, 1);
	if (chunks <= 256) ELF_NORM8(4, 1);
	if (chunks <= 512) ELF_NORM8(2, 4);
	ELF_NORM8(4, 4);
#undef ELF_NORM8
}

}  // namespace elf
