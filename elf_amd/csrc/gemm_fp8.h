// What the block-scaled 8-bit GEMM kernels share: their arguments, the layout of a K slice in LDS, operand fragments, and the epilogue.
#pragma once
#include <atomic>
#include <type_traits>

#include "fp8.h"
#include "gemm_tile.h"
#include "kernels.h"

namespace elf {
namespace fp8 {

using dma::static_for;

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int BK = FP8_BLOCK;  // K slice: one block, 128 bytes of a row

struct Args {
	const uint8_t* A;
	const uint8_t* B;
	const uint8_t* sa;
	const uint8_t* sb;
	int64_t lda, ldb, ldsa, ldsb;
	void* C;
	const bf16_t* R;
	int64_t ldc, ldr;
	int M, N, nk;  // nk: K slices
	int epi;
	int tiles_m, tiles_n;
	bool c_between;  // rows of C (bf16) start between dwords
	int splits, split_nk;  // K in `splits` ranges of split_nk slices (the last one of what is left): their parts go to C [splits][M][N], fp32
};

// D = W-rows x token-rows + C: the weight's rows go to the m side, so that a lane's four accumulators are four columns of one row of the
// output.  FMT: the tokens' type (the weight's is e4m3).  The low byte of either scale register counts; all four 32-wide parts of the block
// are given the same one.  What the instruction does with its 128 products was measured (one large product and one small one, at every
// distance): the products of 8 neighbouring k are added as far as 13 binary places below the largest sum of two operands' exponents (a subnormal
// number has the smallest normal one's) and cut off there, the sixteen sums and C in fp32.  1.5e-5 off in the 2-norm for normal data, 3.5e-5
// where magnitudes spread over e^4: a thousandth of the rounding to e4m3.
template <int FMT>
__device__ __forceinline__ f32x4 mfma8(const i32x8& w, const i32x8& x, const f32x4& c, int scale_w, int scale_x) {
	return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 0, FMT, 0, scale_w, 0, scale_x);
}

// Tile `pid`: XCD w % 8 takes a contiguous run of tiles, and a run goes down 8 tile rows before it moves on by a column.
__device__ __forceinline__ void tile_at(const Args& g, int pid, int& tm, int& tn) {
	const int ntiles = g.tiles_m * g.tiles_n;
	pid = (pid & 7) * (ntiles >> 3) + min(pid & 7, ntiles & 7) + (pid >> 3);
	constexpr int GROUP = 8;
	const int per_group = GROUP * g.tiles_n, first = (pid / per_group) * GROUP, rows = min(g.tiles_m - first, GROUP);
	tm = first + (pid % per_group) % rows;
	tn = (pid % per_group) / rows;
}

// 8 neighbouring accumulators of one row of C from column `col` on
__device__ __forceinline__ void store8(const Args& g, void* C, int64_t row, int col, const float (&acc)[8]) {
	if (row >= g.M || col >= g.N) return;
	if (g.epi <= EPI_BF16_RESID) {
		bf16_t* c = reinterpret_cast<bf16_t*>(C) + row * g.ldc + col;
		const bf16_t* r = g.R + row * g.ldr + col;
		if (col + 8 <= g.N) {
			float v[8];
#pragma unroll
			for (int j = 0; j < 8; j++) v[j] = acc[j];
			if (g.epi == EPI_BF16_RESID) {
				const bf16x8 rv = *reinterpret_cast<const bf16x8_any*>(r);
#pragma unroll
				for (int j = 0; j < 8; j++) v[j] += (float)rv[j];
			}
			bf16x8 o;
#pragma unroll
			for (int j = 0; j < 8; j++) o[j] = (bf16_t)v[j];
			*reinterpret_cast<bf16x8_any*>(c) = o;
		} else {
#pragma unroll
			for (int j = 0; j < 7; j++)
				if (col + j < g.N) c[j] = (bf16_t)(g.epi == EPI_BF16_RESID ? acc[j] + (float)r[j] : acc[j]);
		}
	} else {
		float* c = reinterpret_cast<float*>(C) + row * g.ldc + col;
		if (col + 8 <= g.N) {
			f32x4 lo = {acc[0], acc[1], acc[2], acc[3]}, hi = {acc[4], acc[5], acc[6], acc[7]};
			if (g.epi == EPI_F32_ACC) {
				lo += *reinterpret_cast<const f32x4_any*>(c);
				hi += *reinterpret_cast<const f32x4_any*>(c + 4);
			}
			*reinterpret_cast<f32x4_any*>(c) = lo;
			*reinterpret_cast<f32x4_any*>(c + 4) = hi;
		} else {
#pragma unroll
			for (int j = 0; j < 7; j++)
				if (col + j < g.N) c[j] = g.epi == EPI_F32_ACC ? c[j] + acc[j] : acc[j];
		}
	}
}

// A lane's accumulators of one row of a wave tile 32 CF wide: runs of 8 columns from col0 + 32 t on.  WHOLE: all of the tile's columns are the
// matrix's; its rows may not be (every lane of a wave calls this: a run's end may belong to another lane's).
template <bool WHOLE, int CF>
__device__ __forceinline__ void store_row(const Args& g, void* C, int64_t row, int col0, const f32x4 (&acc)[2 * CF]) {
	auto run = [&](int t, float (&v)[8]) {
#pragma unroll
		for (int e = 0; e < 8; e++) v[e] = acc[2 * t + (e >> 2)][e & 3];
	};
	const bool inside = row < g.M;
	if constexpr (!WHOLE) {
#pragma unroll
		for (int t = 0; t < CF; t++) {
			float v[8];
			run(t, v);
			store8(g, C, row, col0 + 32 * t, v);
		}
	} else if (g.epi <= EPI_BF16_RESID) {
		bf16_t* c = reinterpret_cast<bf16_t*>(C) + row * g.ldc + col0;
		bf16x8 rs[CF];
		if (g.epi == EPI_BF16_RESID) {
			const bf16_t* r = g.R + (inside ? row : 0) * g.ldr + col0;
#pragma unroll
			for (int t = 0; t < CF; t++) rs[t] = *reinterpret_cast<const bf16x8_any*>(r + 32 * t);
		}
		auto rounded = [&](int t) {
			float v[8];
			run(t, v);
			bf16x8 o;
#pragma unroll
			for (int e = 0; e < 8; e++) o[e] = (bf16_t)(g.epi == EPI_BF16_RESID ? v[e] + (float)rs[t][e] : v[e]);
			return o;
		};
		if (!g.c_between) {
			if (!inside) return;
#pragma unroll
			for (int t = 0; t < CF; t++) *reinterpret_cast<bf16x8_any*>(c + 32 * t) = rounded(t);
			return;
		}
		// the run behind that of lane group q is group q + 1's, behind group 3's group 0's next
		const int lane = threadIdx.x & 63;
		u32x4 w[CF];
		uint32_t next[CF];
#pragma unroll
		for (int t = 0; t < CF; t++) w[t] = __builtin_bit_cast(u32x4, rounded(t));
#pragma unroll
		for (int t = 0; t < CF; t++) next[t] = (uint32_t)__shfl((int)(lane < 16 ? w[t + 1 < CF ? t + 1 : t][0] : w[t][0]), (lane + 16) & 63, 64);
		if (!inside) return;
#pragma unroll
		for (int t = 0; t < CF; t++) store_shifted(c + 32 * t, w[t], next[t], lane < 16 && t == 0, lane >= 48 && t == CF - 1);
	} else {
		if (!inside) return;
		float* c = reinterpret_cast<float*>(C) + row * g.ldc + col0;
		f32x4 old[2 * CF];
		if (g.epi == EPI_F32_ACC) {
#pragma unroll
			for (int t = 0; t < 2 * CF; t++) old[t] = *reinterpret_cast<const f32x4_any*>(c + 32 * (t >> 1) + 4 * (t & 1));
		}
#pragma unroll
		for (int t = 0; t < 2 * CF; t++) *reinterpret_cast<f32x4_any*>(c + 32 * (t >> 1) + 4 * (t & 1)) = g.epi == EPI_F32_ACC ? old[t] + acc[t] : acc[t];
	}
}

// Direct-to-LDS loads through a buffer descriptor: lane l's 16 or 4 bytes from base + off[l] to lds + 16 l or 4 l.  An offset that is not
// below the descriptor's size reads zeros: rows behind a matrix need no address of their own.  (The scalar write of M0 and the load need a
// wait state between them.)
__device__ __forceinline__ u32x4 buffer_of(const uint8_t* base, uint32_t bytes) {
	const uint64_t p = (uint64_t)base;
	return u32x4{(uint32_t)p, (uint32_t)(p >> 32), bytes, 0x00027000u};
}
// the size of a descriptor over a block's scales from a tile's first row on: up to the last row, in whole dwords (the rest of a row of scales may
// be another matrix's, or nobody's)
__device__ __forceinline__ uint32_t scale_bytes(int rows) { return (uint32_t)min(256, (rows + 3) & ~3); }
template <int IMM>
__device__ __forceinline__ void load_lds16(const u32x4& buf, uint32_t off, uint32_t lds) {
	asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(buf), "n"(IMM) : "memory", "m0", "scc");
}
__device__ __forceinline__ void load_lds4(const u32x4& buf, uint32_t off, uint32_t lds) {
	asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(buf) : "memory", "m0");
}

// Places of the 16-byte chunks of a row's 128 bytes in LDS, as a function of the row: chunk c lies at c ^ swz(row).  Token rows are read 16
// neighbouring ones at a time, weight rows as fragments of rows 8 g + r (see w_row).
__device__ __forceinline__ int swz_x(int row) { return (row >> 1) & 7; }
__device__ __forceinline__ int swz_w(int row) { return (((row >> 3) & 3) << 1) | ((row >> 1) & 1); }
// The weight row (column of C) in slot `slot` of 16-row fragment j: a lane's accumulators of fragments 2 i and 2 i + 1 are then 8 neighbouring
// columns, 32 i + 8 (lane / 16) .. + 7.
__device__ __forceinline__ int w_row(int j, int slot) { return 32 * (j >> 1) + 4 * (j & 1) + 8 * (slot >> 2) + (slot & 3); }

// Lets a kernel have `bytes` of LDS, once a device (`devices`: those that have been asked).
inline int allow_lds(const void* kern, int bytes, std::atomic<uint64_t>& devices) {
	int device = 0;
	ELF_CHECK_HIP(hipGetDevice(&device));
	const uint64_t bit = uint64_t(1) << (device & 63);
	if (devices.load(std::memory_order_relaxed) & bit) return 0;
	ELF_CHECK_HIP(hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
	devices.fetch_or(bit, std::memory_order_relaxed);
	return 0;
}
constexpr int64_t GRID_256 = (int64_t(1) << 24) - 1;  // workgroups of 256 threads in a launch: a grid has less than 2^32 threads

template <int FMT>
int launch_tile(const Args& g, int tile, hipStream_t stream);
template <int FMT>
int launch_few(const Args& g, int waves, hipStream_t stream);
constexpr int FEW_ROWS = 64;

}  // namespace fp8
}  // namespace elf
