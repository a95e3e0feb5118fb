// Block-scaled 8-bit GEMM (format: fp8.h): C [M, N] (+)= sum over the blocks b of 128 columns of 2^(ea[m, b] + eb[n, b]) A_b[m] . B_b[n].
// Tiles for products that do not fill the chip with 256 x 256 ones, and the choice among all.
#include "gemm_fp8.h"

namespace elf {
namespace fp8 {

constexpr int64_t MOST = (int64_t(1) << 31) - 512;  // M, N and K

// 64 x 64 tiles: four waves, 2 x 2, each 32 x 32; a ring of four K slices in LDS, filled by direct-to-LDS loads three slices ahead.
// Bound: alone on a compute unit by the chain barrier -> fragment reads -> MFMAs of a slice, 0.32 us (two slices in LDS 0.53, eight 0.38); two workgroups
// take 0.45, 73 KB/us into LDS (two slices 0.54).
// A slice of an operand is its rows' 128 bytes of one block, 16-byte chunk c of row r in place c ^ f(r) so that the 16 lanes of a
// fragment read meet 16 different bank groups, and one scale byte a row.  Rows behind the matrix are zeros.
// A lane's share of a fragment is the chunks q and q + 4 of its row, q = lane / 16: the order of k within a block is free, as long as both
// operands have the same.
struct Ring {
	static constexpr int BM = 64, BN = 64, NS = 4;
	static constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK;
	static constexpr int SCALES = 4 * 256;  // a dword per thread
	static constexpr int STAGE = A_BYTES + B_BYTES + SCALES;
	static constexpr int BYTES = NS * STAGE;
};

template <int FMT>
__global__ __launch_bounds__(256) void gemm_kernel(Args g) {
	constexpr int BM = Ring::BM, BN = Ring::BN, NS = Ring::NS;
	constexpr int RA = BM / 32, RB = BN / 32;  // 16-row fragments of a wave
	constexpr int LA = Ring::A_BYTES / 4096, LB = Ring::B_BYTES / 4096;
	extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
	const int tid = threadIdx.x, lane = tid & 63;
	const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
	const int wm = wave >> 1, wn = wave & 1;
	const int ntiles = g.tiles_m * g.tiles_n, split = (int)blockIdx.x / ntiles;
	int tm, tn;
	tile_at(g, (int)blockIdx.x - split * ntiles, tm, tn);
	const int64_t kt0 = (int64_t)split * g.split_nk;
	const int nk = min(g.split_nk, g.nk - (int)kt0);
	const int m0 = __builtin_amdgcn_readfirstlane(tm * BM), n0 = __builtin_amdgcn_readfirstlane(tn * BN);

	uint32_t aoff[LA], boff[LB];
#pragma unroll
	for (int i = 0; i < LA; i++) {
		const int row = (wave * LA + i) * 8 + (lane >> 3);
		aoff[i] = (uint32_t)(row * g.lda) + (((lane & 7) ^ swz_x(row)) << 4);
	}
#pragma unroll
	for (int i = 0; i < LB; i++) {
		const int row = (wave * LB + i) * 8 + (lane >> 3);
		boff[i] = (uint32_t)(row * g.ldb) + (((lane & 7) ^ swz_w(row)) << 4);
	}
	// the descriptors' sizes end with the matrix: rows behind it read zeros
	const uint8_t *ap = g.A + m0 * g.lda + kt0 * BK, *bp = g.B + n0 * g.ldb + kt0 * BK;
	const uint32_t a_bytes = (uint32_t)((min(BM, g.M - m0) - 1) * g.lda) + BK, b_bytes = (uint32_t)((min(BN, g.N - n0) - 1) * g.ldb) + BK;
	// even waves fetch the scales of A's rows, odd ones of B's (two waves do what one could)
	const bool s_of_a = (wave & 1) == 0;
	const int64_t s_step = s_of_a ? g.ldsa : g.ldsb;
	const uint8_t* sp = (s_of_a ? g.sa + m0 : g.sb + n0) + kt0 * s_step;
	const uint32_t s_bytes = scale_bytes(s_of_a ? g.M - m0 : g.N - n0);
	const uint32_t lds = lds_addr(smem);

	// slice kt into a stage; one behind the last is fetched from the last: the count of loads in flight stays the same, and nobody reads it
	auto fetch = [&](int kt, int stage) {
		kt = min(kt, nk - 1);
		const uint32_t at = lds + (uint32_t)stage * Ring::STAGE;
		const u32x4 ab = buffer_of(ap + (int64_t)kt * BK, a_bytes), bb = buffer_of(bp + (int64_t)kt * BK, b_bytes);
		static_for<LA>([&](auto ic) { load_lds16<decltype(ic)::value * 1024>(ab, aoff[decltype(ic)::value], at + wave * (LA * 1024)); });
		static_for<LB>([&](auto ic) { load_lds16<decltype(ic)::value * 1024>(bb, boff[decltype(ic)::value], at + Ring::A_BYTES + wave * (LB * 1024)); });
		load_lds4(buffer_of(sp + kt * s_step, s_bytes), lane * 4, at + Ring::A_BYTES + Ring::B_BYTES + wave * 256);
	};

	f32x4 acc[RA][RB];
#pragma unroll
	for (int i = 0; i < RA; i++)
#pragma unroll
		for (int j = 0; j < RB; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

	const int l15 = lane & 15, q4 = lane >> 4;
#pragma unroll
	for (int i = 0; i < NS - 1; i++) fetch(i, i);
	int stage = 0;
	for (int kt = 0; kt < nk; kt++) {
		wait_counters<(NS - 2) * (LA + LB + 1), 0>();  // this wave's part of slice kt has landed, its reads of slice kt - 1 are done
		__syncthreads();
		fetch(kt + NS - 1, stage == 0 ? NS - 1 : stage - 1);
		const unsigned char* sl = smem + stage * Ring::STAGE;
		const unsigned char* sc = sl + Ring::A_BYTES + Ring::B_BYTES;
		i32x8 fw[RB];
		int ew[RB];
#pragma unroll
		for (int j = 0; j < RB; j++) {
			const int row = wn * (BN / 2) + w_row(j, l15);
			const unsigned char* p = sl + Ring::A_BYTES + row * BK;
			const i32x4 lo = *reinterpret_cast<const i32x4*>(p + ((q4 ^ swz_w(row)) << 4)), hi = *reinterpret_cast<const i32x4*>(p + (((q4 + 4) ^ swz_w(row)) << 4));
			fw[j] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
			ew[j] = sc[256 + row];
		}
#pragma unroll
		for (int i = 0; i < RA; i++) {
			const int row = wm * (BM / 2) + i * 16 + l15;
			const unsigned char* p = sl + row * BK;
			const i32x4 lo = *reinterpret_cast<const i32x4*>(p + ((q4 ^ swz_x(row)) << 4)), hi = *reinterpret_cast<const i32x4*>(p + (((q4 + 4) ^ swz_x(row)) << 4));
			const i32x8 fx = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
			const int ex = sc[row];
#pragma unroll
			for (int j = 0; j < RB; j++) acc[i][j] = mfma8<FMT>(fw[j], fx, acc[i][j], ew[j], ex);
		}
		stage = stage + 1 == NS ? 0 : stage + 1;
	}
	void* const C = reinterpret_cast<float*>(g.C) + (g.splits > 1 ? (int64_t)split * g.M * g.N : 0);
#pragma unroll
	for (int i = 0; i < RA; i++) {
		const int64_t row = m0 + wm * (BM / 2) + i * 16 + l15;
#pragma unroll
		for (int j = 0; j < RB; j += 2) {
			const float v[8] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3], acc[i][j + 1][0], acc[i][j + 1][1], acc[i][j + 1][2], acc[i][j + 1][3]};
			store8(g, C, row, n0 + wn * (BN / 2) + 16 * j + 8 * q4, v);
		}
	}
	wait_vmcnt<0>();  // the loads behind the last slice land in LDS too
}

template <int FMT>
static int launch_64(Args g, hipStream_t stream) {
	g.tiles_m = (g.M + Ring::BM - 1) / Ring::BM, g.tiles_n = (g.N + Ring::BN - 1) / Ring::BN;
	const int64_t nwork = (int64_t)g.tiles_m * g.tiles_n * g.splits;
	ELF_REQUIRE(nwork <= GRID_256, "gemm_fp8: too many tiles for one launch");
	auto kern = gemm_kernel<FMT>;
	constexpr int smem = Ring::BYTES;
	static std::atomic<uint64_t> devices{0};
	if (int rc = allow_lds(reinterpret_cast<const void*>(kern), smem, devices)) return rc;
	ELF_LAUNCH(kern, dim3((uint32_t)nwork), dim3(256), smem, stream, g);
	ELF_CHECK_HIP(hipGetLastError());
	return 0;
}

// C from the parts of a split K, added in the order of the K ranges.  Bound by the trip of its loads: four ranges' go out together.
__global__ __launch_bounds__(256) void join_kernel(Args g, const float* __restrict__ part) {
	const int chunks = (g.N + 7) / 8;
	const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
	const int64_t row = i / chunks;
	if (row >= g.M) return;
	const int col = (int)(i - row * chunks) * 8;
	float v[8] = {};
	constexpr int U = 4;
	for (int s0 = 0; s0 < g.splits; s0 += U) {
		f32x4 lo[U], hi[U];
#pragma unroll
		for (int u = 0; u < U; u++) {
			const float* p = part + ((int64_t)min(s0 + u, g.splits - 1) * g.M + row) * g.N + col;
			if (col + 8 <= g.N) {
				lo[u] = *reinterpret_cast<const f32x4_any*>(p), hi[u] = *reinterpret_cast<const f32x4_any*>(p + 4);
			} else {
#pragma unroll
				for (int j = 0; j < 4; j++) lo[u][j] = col + j < g.N ? p[j] : 0.f, hi[u][j] = col + 4 + j < g.N ? p[4 + j] : 0.f;
			}
		}
#pragma unroll
		for (int u = 0; u < U; u++)
			if (s0 + u < g.splits) {
#pragma unroll
				for (int j = 0; j < 4; j++) v[j] += lo[u][j], v[4 + j] += hi[u][j];
			}
	}
	store8(g, g.C, row, col, v);
}

// The way of a product: the fastest by estimate.  Times (us) that the estimates were taken from, on operands out of memory:
//   few rows, gemm_few_kernel / 64 x 64 / 64 x 64 and the better of 3 to 8 K ranges: 1 x 6144 x 4096 7.9 / 11.9, 1 x 4096 x 14336 13.0 / 35 / 15.7,
//     2 x 1455 x 7385 7.5 / - / 13.6, 21 x 379 x 6996 10.2 / - / 11.5, 32 x 4096 x 4096 7.9 / 12.1, 32 x 4096 x 14336 23.5 / 35.5 / 17.0,
//     48 x 4096 x 14336 33 / 36 / 17.7, 48 x 28672 x 4096 60 / 28.7, 64 x 1024 x 8192 - / 23 / 10.9
//   64 x 64 / 128 x 128 / 256 x 256: 79 x 26244 x 228 8.0 / 6.8 / 10.4, 5827 x 2080 x 162 19.5 / 12.5 / 12.6, 256 x 4096 x 4096 12.5 / 17.3 / 40,
//     512 x 4096 x 4096 16.1 / 17.5 / 40.7, 1024 x 4096 x 4096 29 / 19.3 / 41, 2111 x 4288 x 1600 32 / 21.0 / 24.9, 1625 x 14312 x 3520 157 / 96 / 85,
//     2048 x 6144 x 4096 99 / 53 / 44.8, 4096 x 6144 x 4096 189 / 106 / 92, 8192 x 28672 x 4096 1678 / 955 / 689
// Over 638 drawn sizes of 1 to 8192 rows, 64 to 28672 columns and K up to 14336 the way taken was 1.1 % slower than the fastest (geometric mean; 20 % at most), in a build
// of its own that could be told the way.  All of it is of bf16 outputs without a residual, and so is the memory that `out` counts: a
// residual or fp32 outputs move twice as much, fp32 sums four times.
// (128 x 256 tiles lay within 5 % of the better of their neighbours, 64 x 128 within 10 %; K ranges of 128 x 128 and 256 x 256 tiles never paid.)
struct Plan {
	int way, waves, splits, split_nk;
	float us;
};
enum Way { FEW, TILE64, TILE128, TILE256 };

static Plan plan(int64_t M, int64_t N, int nk, bool split) {
	constexpr float MEMORY = 4.8e6f;  // bytes a microsecond
	const float read = ((float)M + N) * nk * BK / MEMORY, out = 2.f * M * N / MEMORY, floor = read + out;
	Plan best{TILE64, 0, 1, nk, 0.f};
	auto tiles = [&](int t) { return ((M + t - 1) / t) * ((N + t - 1) / t); };
	auto longer = [](float a, float b) { return a > b ? a : b; };
	// rounds of 512 workgroups, two a compute unit, `pair` us each; a last one of at most 256, each with a compute unit to itself, `lone`
	auto rounds = [&](int64_t work, float pair, float lone) {
		const int64_t full = work / 512, rest = work - full * 512;
		return full * pair + (rest == 0 ? 0.f : rest <= 256 ? lone : pair);
	};
	best.us = 2.5f + longer(rounds(tiles(64), nk * 0.45f + 1.7f, nk * 0.32f + 0.7f), floor);
	if (split) {  // up to two workgroups a compute unit (93 x 4320 x 10866, 136 tiles, whole and in 2 and 3 ranges 29.1, 25.2 and 21.0 us; 48 x 4096 x 14336, 64 tiles, in
	              // 3, 4, 6 and 8 19.4, 17.0, 20.8 and 19.4); the join costs a launch and a write and a read of each range's sums, 8 MiB
	              // in all at most
		for (int s = 2; s <= 8 && tiles(64) * s <= 512; s++) {
			const int per = (nk + s - 1) / s, n = (nk + per - 1) / per;
			if (n != s || per < 4) continue;
			const float us = 4.7f + 0.5f * s + 8.f * s * M * N / MEMORY + longer(rounds(tiles(64) * s, per * 0.45f + 1.7f, per * 0.32f + 0.7f), read * 0.85f + out);  // (a read of several places a row: 5.7 TB/s)
			if (us < best.us) best = Plan{TILE64, 0, s, per, us};
		}
	}
	if (M <= FEW_ROWS && N <= (int64_t(1) << 25)) {  // (a grid's threads)
		// a block of K takes a workgroup as long as its reads; the last workgroups of a large N leave some compute units idle
		const int rows = M <= 16 ? 16 : M <= 32 ? 32 : 64;
		const float block = N < 2048 ? (16 + rows) * BK / 46e3f : rows == 16 ? 0.085f + 0.0028f * M : (16 + rows) * BK / 33e3f;
		const float turns = N <= 4096 ? 1.f : (N / 4096.f + (N + 4095) / 4096) / 2;
		const float us = 2.f + longer((nk * block + 0.3f) * turns, floor);
		// 16 waves where a compute unit has one workgroup (us with 16 and 8: 16 x 4096 x 14336 16.4 and 16.9, 2 x 24433 x 13421 62.6 and 55.5)
		if (us < best.us) best = Plan{FEW, nk >= 64 && N <= 4096 ? 16 : 8, 1, nk, us};
	}
	if (nk >= 2) {  // (both run two slices ahead)
		float us = 3.5f + 0.6f * out + longer(rounds(tiles(128), nk + 0.5f, nk * 0.45f + 0.5f), floor);
		if (us < best.us) best = Plan{TILE128, 0, 1, nk, us};
		const int64_t t = tiles(256), full = t / 256, rest = t - full * 256;
		us = 7.f + longer(full * (6.f + nk * 1.3f) + (rest ? 6.f + nk * 1.02f : 0.f), floor) + (N % 2 ? 5.f : 0.f);  // (odd rows leave slowly, behind the last slice)
		if (us < best.us) best = Plan{TILE256, 0, 1, nk, us};
	}
	return best;
}

template <int FMT>
static int launch(const Args& g, const Plan& p, hipStream_t stream) {
	switch (p.way) {
		case FEW: return launch_few<FMT>(g, p.waves, stream);
		case TILE128: return launch_tile<FMT>(g, 128, stream);
		case TILE256: return launch_tile<FMT>(g, 256, stream);
		default: return launch_64<FMT>(g, stream);
	}
}

}  // namespace fp8

int64_t gemm_fp8_workspace_floats(int64_t M, int64_t N, int64_t K) {
	if (M <= 0 || N <= 0 || K <= 0 || M > fp8::MOST || N > fp8::MOST || K > fp8::MOST) return 0;
	const fp8::Plan p = fp8::plan(M, N, (int)((K + 127) / 128), true);
	return p.splits > 1 ? p.splits * M * N : 0;
}

int gemm_fp8_way(int64_t M, int64_t N, int64_t K, int64_t workspace_floats, int* way) {
	ELF_REQUIRE(way && M > 0 && N > 0 && K > 0 && M <= fp8::MOST && N <= fp8::MOST && K <= fp8::MOST, "gemm_fp8_way: a size that the product refuses");
	const fp8::Plan p = fp8::plan(M, N, (int)((K + 127) / 128), workspace_floats >= gemm_fp8_workspace_floats(M, N, K));
	way[0] = p.way == fp8::FEW ? (M <= 16 ? 16 : M <= 32 ? 32 : 64) : p.way == fp8::TILE64 ? 64 : p.way == fp8::TILE128 ? 128 : 256;
	way[1] = p.way == fp8::FEW ? 16 : way[0];
	way[2] = p.splits;
	return 0;
}

int gemm_fp8(int64_t M, int64_t N, int64_t K, int fmt_a, const void* A, int64_t lda, const void* sa, int64_t ldsa, const void* B, int64_t ldb, const void* sb, int64_t ldsb,
             void* C, int64_t ldc, int epi, const void* R, int64_t ldr, float* workspace, int64_t workspace_floats, hipStream_t stream) {
	ELF_REQUIRE(M > 0 && N > 0 && K > 0 && A && sa && B && sb && C, "gemm_fp8: empty problem or null operand");
	ELF_REQUIRE(M <= fp8::MOST && N <= fp8::MOST && K <= fp8::MOST, "gemm_fp8: sizes go up to %lld", (long long)fp8::MOST);
	ELF_REQUIRE(fmt_a == FP8_E4M3 || fmt_a == FP8_E5M2, "gemm_fp8: unknown format %d", fmt_a);
	ELF_REQUIRE(epi >= EPI_BF16 && epi <= EPI_F32_STORE, "gemm_fp8: unknown epilogue %d", epi);
	const int64_t row = (K + 127) / 128 * 128;
	ELF_REQUIRE(lda >= row && ldb >= row && lda % 16 == 0 && ldb % 16 == 0 && ((uintptr_t)A % 16) == 0 && ((uintptr_t)B % 16) == 0,
	            "gemm_fp8: rows must hold K rounded up to 128 bytes, lie a multiple of 16 bytes apart and be 16-byte aligned");
	ELF_REQUIRE(lda < (int64_t(1) << 24) && ldb < (int64_t(1) << 24), "gemm_fp8: rows too far apart for the tile's 32-bit offsets (lda=%lld ldb=%lld)", (long long)lda, (long long)ldb);
	ELF_REQUIRE(ldsa >= M && ldsb >= N && ldsa % 16 == 0 && ldsb % 16 == 0 && ((uintptr_t)sa % 16) == 0 && ((uintptr_t)sb % 16) == 0,
	            "gemm_fp8: the scales of a block must cover the rows, lie a multiple of 16 bytes apart and be 16-byte aligned");
	const bool f32 = epi == EPI_F32_ACC || epi == EPI_F32_STORE;
	ELF_REQUIRE(ldc >= N && ((uintptr_t)C % (f32 ? 4 : 2)) == 0, "gemm_fp8: rows of C overlap or C is not aligned to its elements");
	ELF_REQUIRE(epi != EPI_BF16_RESID || (R && (ldr == 0 || ldr >= N) && ((uintptr_t)R % 2) == 0), "gemm_fp8: epilogue 1 needs a residual with rows of N values (ldr 0: one row for all)");
	ProfScope prof(PROF_GEMM, 2.0 * M * N * K, stream);
	ELF_REQUIRE(!workspace || ((uintptr_t)workspace % 16) == 0, "gemm_fp8: the workspace must be 16-byte aligned");
	const int nk = (int)(row / 128);
	const fp8::Plan p = fp8::plan(M, N, nk, workspace && workspace_floats >= gemm_fp8_workspace_floats(M, N, K));
	const fp8::Args g{(const uint8_t*)A, (const uint8_t*)B, (const uint8_t*)sa, (const uint8_t*)sb, lda, ldb, ldsa, ldsb, C, (const bf16_t*)R, ldc, ldr, (int)M, (int)N, nk, epi, 0, 0, !f32 && (ldc % 2 != 0 || (uintptr_t)C % 4 != 0), p.splits, p.split_nk};
	auto launch = [&](const fp8::Args& a) { return fmt_a == FP8_E4M3 ? fp8::launch<FP8_E4M3>(a, p, stream) : fp8::launch<FP8_E5M2>(a, p, stream); };
	if (p.splits == 1) return launch(g);
	fp8::Args part = g;
	part.C = workspace, part.ldc = N, part.epi = EPI_F32_STORE;
	if (int rc = launch(part)) return rc;
	ELF_LAUNCH(fp8::join_kernel, dim3((uint32_t)(((N + 7) / 8 * M + 255) / 256)), dim3(256), 0, stream, g, (const float*)workspace);
	ELF_CHECK_HIP(hipGetLastError());
	return 0;
}

}  // namespace elf
