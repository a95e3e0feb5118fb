// The block-scaled 8-bit GEMM on tiles of 256 x 256 and 128 x 128.
#include "gemm_fp8.h"

namespace elf {
namespace fp8 {

// Four waves, 2 x 2, of 16 RF rows x 32 CF columns each.  A K slice is one block; a wave multiplies it in two half-steps of RF x CF MFMAs of 32
// cycles: the first and the second 16 CF of its columns.  The loop keeps the matrix pipe fed:
//  * NS slices of either operand in LDS, and a part's stage is loaded again as soon as it has been read: token rows and the weight rows of the
//    first half-step in one piece, those of the second half-step in another.  One barrier a half-step, a quarter of the way in, where the reads
//    before it are long done: with two slices, loads have one and a half to land.
//  * the loads and the fragment reads of what comes next go out between the MFMAs one at a time.  A row slab's fragment is read again for the
//    next slice as soon as its last MFMA of this one is issued, so there is one copy of them; those of the weight rows take turns.
//  * workgroups are persistent: the slices of their tiles follow each other without a gap (the last NS of a tile load the first NS of the next),
//    and C leaves from registers.
// Measured: 8192 x 28672 x 4096 on 256 x 256 tiles 669 to 730 us from part to part, 2.9 to 2.6 PFLOP/s (8192^3 2.9; the vendor's product of
// matrices with one scale each 2.75): bound by power, the matrix pipe busy 71 % of the cycles at 1.57 GHz, no LDS bank conflict.  64 tiles alone
// take 1.25 us a slice at full clock, 0.97 with operands in L2, for 0.85 of MFMAs.  128 x 128 tiles: 0.6 us a slice, 1.0 for two workgroups of a
// compute unit (0.26 us of MFMAs a slice each): bound by the rate at which a compute unit is served, 50 to 73 KB/us on tiles of every size, for more
// slices in LDS gain nothing.  2111 x 4287 x 1599, 26 us: matrix pipe busy 29 % of the cycles, the path of returning loads 67 % (half of that it waits), L1 waits for
// L2 30 %, L2 hits 82 %.  Not faster, at the same 128 x 128 and on 128 x 256: three and four slices in LDS, one
// barrier a slice with both operands' fragments a slice ahead, eight waves; on 256 x 256: barriers earlier and later, weight fragments read earlier.
template <int RF, int CF, int NS>
struct Tile {
	static constexpr int M = 32 * RF, N = 64 * CF;
	static constexpr int X_BYTES = M * BK, W_BYTES = N * BK, SCALES = 4 * 256;  // of a slice (scales: a dword per thread)
	static constexpr int FIRST = RF + CF + 1, SECOND = CF;  // loads of a wave: 1 KiB pieces of token rows, weight rows and a row of scales; weight rows
	static constexpr int X_AT = 0, W_AT = NS * X_BYTES, S_AT = W_AT + NS * W_BYTES, BYTES = S_AT + (NS + 1) * SCALES;
	static constexpr int PER_CU = 2 * BYTES <= 160 * 1024 ? 2 : 1;  // workgroups of a compute unit
	static constexpr int TAIL = RF == 8 ? 2 : 0;  // row slabs whose reads are left for the next slice's first MFMAs
	static constexpr int MFMAS = RF * CF, BARRIER = MFMAS / 4 - 1, SLOTS = MFMAS - 1 - BARRIER;
	static_assert(CF % 2 == 0 && RF + 2 * CF <= 16 && BYTES <= 160 * 1024 && (NS - 1) * (FIRST + SECOND) < 64, "");
};

template <int FMT, bool FIRST>
__device__ __forceinline__ void mfma_at(f32x4& acc, const i32x8& w, const i32x8& x, int scale_w, int scale_x) {
	if constexpr (FIRST) {
		if constexpr (FMT == FP8_E4M3) asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, 0, %3, %4 op_sel_hi:[0,0,0]" : "=a"(acc) : "v"(w), "v"(x), "v"(scale_w), "v"(scale_x));
		else asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, 0, %3, %4 op_sel_hi:[0,0,0] blgp:1" : "=a"(acc) : "v"(w), "v"(x), "v"(scale_w), "v"(scale_x));
	} else {
		if constexpr (FMT == FP8_E4M3) asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]" : "+a"(acc) : "v"(w), "v"(x), "v"(scale_w), "v"(scale_x));
		else asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0] blgp:1" : "+a"(acc) : "v"(w), "v"(x), "v"(scale_w), "v"(scale_x));
	}
}

template <int RF, int CF, int NS, int FMT>
__global__ __launch_bounds__(256, (Tile<RF, CF, NS>::PER_CU)) void gemm_tile_kernel(Args g) {
	using T = Tile<RF, CF, NS>;
	extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
	const int tid = threadIdx.x, lane = tid & 63;
	const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
	const int wm = wave >> 1, wn = wave & 1;
	const int l15 = lane & 15, q4 = lane >> 4;
	const uint32_t lds = lds_addr(smem);

	// Byte offsets, from the tile's first row, of the chunks this lane fetches.  A piece is 8 rows; the 4 CF pieces of weight rows of a half-step
	// are the first (second) 2 CF of either column half's 4 CF.
	uint32_t xoff[RF], woff[2 * CF];
#pragma unroll
	for (int i = 0; i < RF; i++) {
		const int row = (wave * RF + i) * 8 + (lane >> 3);
		xoff[i] = (uint32_t)(row * g.lda) + (((lane & 7) ^ swz_x(row)) << 4);
	}
#pragma unroll
	for (int i = 0; i < 2 * CF; i++) {
		const int row = ((wave >> 1) * 4 * CF + (i / CF) * 2 * CF + (wave & 1) * CF + i % CF) * 8 + (lane >> 3);
		woff[i] = (uint32_t)(row * g.ldb) + (((lane & 7) ^ swz_w(row)) << 4);
	}
	const uint32_t x_lds = lds + T::X_AT + wave * (RF * 1024), w_lds = lds + T::W_AT + ((wave >> 1) * 4 * CF + (wave & 1) * CF) * 1024, s_lds = lds + T::S_AT + wave * 256;

	// What the slices of a tile are loaded from: the operands at its rows (the descriptors' sizes end with the matrix) and the
	// scales of the operand that this wave fetches (even waves: token rows, odd: weight rows; two waves do what one could)
	struct Source {
		const uint8_t *x, *w, *s;
		uint32_t x_bytes, w_bytes, s_bytes;
		int m0, n0;
	};
	const bool s_of_x = (wave & 1) == 0;
	const int64_t s_step = s_of_x ? g.ldsa : g.ldsb;
	const int ntiles = g.tiles_m * g.tiles_n, nk = g.nk;  // nk: at least NS
	auto source = [&](int pid) {
		Source t;
		int tm, tn;
		tile_at(g, pid, tm, tn);
		t.m0 = __builtin_amdgcn_readfirstlane(tm * T::M);
		t.n0 = __builtin_amdgcn_readfirstlane(tn * T::N);
		t.x = g.A + t.m0 * g.lda;
		t.w = g.B + t.n0 * g.ldb;
		t.x_bytes = (uint32_t)((min(T::M, g.M - t.m0) - 1) * g.lda) + BK;
		t.w_bytes = (uint32_t)((min(T::N, g.N - t.n0) - 1) * g.ldb) + BK;
		t.s = s_of_x ? g.sa + t.m0 : g.sb + t.n0;
		t.s_bytes = scale_bytes(s_of_x ? g.M - t.m0 : g.N - t.n0);
		return t;
	};
	int pid = blockIdx.x;
	Source cur = source(pid), nxt = cur;

	// slices nk .. nk + NS - 1 are the next tile's first ones or, behind the workgroup's last tile, its own, which nobody reads
	auto x_buf = [&](int step) { return step < nk ? buffer_of(cur.x + (int64_t)step * BK, cur.x_bytes) : buffer_of(nxt.x + (int64_t)(step - nk) * BK, nxt.x_bytes); };
	auto w_buf = [&](int step) { return step < nk ? buffer_of(cur.w + (int64_t)step * BK, cur.w_bytes) : buffer_of(nxt.w + (int64_t)(step - nk) * BK, nxt.w_bytes); };
	auto s_buf = [&](int step) { return step < nk ? buffer_of(cur.s + step * s_step, cur.s_bytes) : buffer_of(nxt.s + (step - nk) * s_step, nxt.s_bytes); };

	int stage = 0, s_stage = 0;  // of the slice that is multiplied; the loads go into stage `stage` and, of scales, into the one before s_stage
	auto before = [](int s) { return s == 0 ? NS : s - 1; };
	auto after = [](int s, int n) { return s + 1 == n ? 0 : s + 1; };
	auto first_load = [&](auto pc, int st, int s_st, const u32x4& xb, const u32x4& wb, const u32x4& sb) {
		constexpr int P = decltype(pc)::value;
		if constexpr (P < RF) load_lds16<P * 1024>(xb, xoff[P], x_lds + st * T::X_BYTES);
		else if constexpr (P < RF + CF) load_lds16<(P - RF) * 1024>(wb, woff[P - RF], w_lds + st * T::W_BYTES);
		else load_lds4(sb, lane * 4, s_lds + s_st * T::SCALES);
	};
	auto second_load = [&](auto pc, int st, const u32x4& wb) {
		constexpr int P = decltype(pc)::value;
		load_lds16<(2 * CF + P) * 1024>(wb, woff[CF + P], w_lds + st * T::W_BYTES);
	};
	static_for<NS>([&](auto sc) {
		constexpr int S = decltype(sc)::value;
		const u32x4 xb = x_buf(S), wb = w_buf(S), sb = s_buf(S);
		static_for<T::FIRST>([&](auto pc) { first_load(pc, S, S, xb, wb, sb); });
		static_for<T::SECOND>([&](auto pc) { second_load(pc, S, wb); });
	});
	constexpr int IN_FLIGHT = (NS - 1) * (T::FIRST + T::SECOND);  // younger than what has to have landed, at every barrier
	wait_vmcnt<IN_FLIGHT>();
	__syncthreads();

	// LDS addresses of this lane's fragment reads (chunk q4, and q4 + 4 at ^ 64) and scales in stage 0
	const uint32_t x_at = lds + T::X_AT + (wm * 16 * RF + l15) * BK + ((q4 ^ swz_x(l15)) << 4);
	const uint32_t w_at = lds + T::W_AT + (wn * 32 * CF + w_row(0, l15)) * BK + ((q4 ^ swz_w(w_row(0, l15))) << 4);
	const uint32_t sx_at = lds + T::S_AT + wm * 16 * RF + l15, sw_at = lds + T::S_AT + 256 + wn * 32 * CF + w_row(0, l15);

	i32x8 fx[RF], fw[2][CF];
	int ex[RF], ew[2][CF];
	f32x4 acc[RF][2 * CF];
	auto chunk = [&](uint32_t at) { return *reinterpret_cast<const i32x4 ELF_LDS*>((uintptr_t)at); };
	auto byte = [&](uint32_t at) { return (int)*reinterpret_cast<const uint8_t ELF_LDS*>((uintptr_t)at); };
	// read 3 i + p of the token rows: part p of slab i's fragment (its halves, its scale), of the slice in stage st; so of the weight rows
	auto read_x = [&](auto rc, int st, int s_st) {
		constexpr int I = decltype(rc)::value / 3, P = decltype(rc)::value % 3;
		if constexpr (P < 2) {
			const i32x4 v = chunk(((x_at + st * T::X_BYTES) ^ (P * 64)) + I * (16 * BK));
#pragma unroll
			for (int e = 0; e < 4; e++) fx[I][P * 4 + e] = v[e];
		} else ex[I] = byte(sx_at + s_st * T::SCALES + I * 16);
	};
	auto read_w = [&](auto hc, auto rc, int st, int s_st) {
		constexpr int H = decltype(hc)::value, J = decltype(rc)::value / 3, P = decltype(rc)::value % 3;
		constexpr int ROW = H * 16 * CF + 32 * (J >> 1) + 4 * (J & 1);
		if constexpr (P < 2) {
			const i32x4 v = chunk(((w_at + st * T::W_BYTES) ^ (P * 64)) + ROW * BK);
#pragma unroll
			for (int e = 0; e < 4; e++) fw[H][J][P * 4 + e] = v[e];
		} else ew[H][J] = byte(sw_at + s_st * T::SCALES + ROW);
	};
	constexpr std::integral_constant<int, 0> C0{};
	constexpr std::integral_constant<int, 1> C1{};
	constexpr int X_READS = 3 * (RF - T::TAIL), W_READS = 3 * CF;
	static_for<X_READS>([&](auto rc) { read_x(rc, 0, 0); });
	static_for<W_READS>([&](auto rc) { read_w(C0, rc, 0, 0); });

	// One slice.  First half-step: the reads that the slice before left, then the barrier (the wave's reads of this slice's token rows and first
	// weight rows are done, the second weight rows have landed), then the loads that go where those were, and the reads of the second weight
	// rows.  Second half-step: the barrier (the second weight rows are read, the next slice's first part has landed), then the loads of the
	// second weight rows, and the next slice's reads.  Operation o of a list of m goes behind MFMA BARRIER + 1 + o SLOTS / m; a token slab's reads
	// not before its last MFMA.
	auto slice = [&](auto first, int kt) {
		constexpr bool FIRST = decltype(first)::value;
		const u32x4 xb = x_buf(kt + NS), wb = w_buf(kt + NS), sb = s_buf(kt + NS);
		const int next = after(stage, NS), s_next = after(s_stage, NS + 1);
		static_for<T::MFMAS>([&](auto nc) {
			constexpr int n = decltype(nc)::value, i = n / CF, j = n % CF, k = n - T::BARRIER - 1;
			mfma_at<FMT, FIRST>(acc[i][j], fw[0][j], fx[i], ew[0][j], ex[i]);
			if constexpr (n < 3 * T::TAIL) read_x(std::integral_constant<int, X_READS + n>{}, stage, s_stage);
			if constexpr (n == T::BARRIER) {
				wait_counters<IN_FLIGHT, 0>();
				__syncthreads();
			}
			static_for<W_READS>([&](auto rc) {
				if constexpr (decltype(rc)::value * T::SLOTS / W_READS == k) read_w(C1, rc, stage, s_stage);
			});
			static_for<T::FIRST>([&](auto pc) {
				if constexpr (decltype(pc)::value * T::SLOTS / T::FIRST == k) first_load(pc, stage, before(s_stage), xb, wb, sb);
			});
			__builtin_amdgcn_sched_barrier(0);
		});
		static_for<T::MFMAS>([&](auto nc) {
			constexpr int n = decltype(nc)::value, i = n / CF, j = n % CF, k = n - T::BARRIER - 1;
			mfma_at<FMT, FIRST>(acc[i][CF + j], fw[1][j], fx[i], ew[1][j], ex[i]);
			if constexpr (n == T::BARRIER) {
				wait_counters<IN_FLIGHT, 0>();
				__syncthreads();
			}
			static_for<W_READS>([&](auto rc) {
				if constexpr (decltype(rc)::value * T::SLOTS / W_READS == k) read_w(C0, rc, next, s_next);
			});
			static_for<X_READS>([&](auto rc) {
				constexpr int r = decltype(rc)::value, even = r * T::SLOTS / X_READS, ready = (r / 3 + 1) * CF - 1 - T::BARRIER - 1;
				if constexpr ((even > ready ? even : ready) == k) read_x(rc, next, s_next);
			});
			static_for<T::SECOND>([&](auto pc) {
				if constexpr (decltype(pc)::value * T::SLOTS / T::SECOND == k) second_load(pc, stage, wb);
			});
			__builtin_amdgcn_sched_barrier(0);
		});
		stage = next, s_stage = s_next;
	};

	for (;;) {
		const int pid_n = pid + (int)gridDim.x;
		const bool more = pid_n < ntiles;
		if (more) nxt = source(pid_n);
		slice(std::true_type{}, 0);
		for (int kt = 1; kt < nk; kt++) slice(std::false_type{}, kt);

		// (the compiler knows nothing of the MFMAs' latency: the last one's result is there after 32 wait states, it needs fewer)
		asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
		const int64_t row0 = cur.m0 + wm * 16 * RF + l15;
		const int col0 = cur.n0 + wn * 32 * CF + 8 * q4;
		const bool whole = cur.n0 + T::N <= g.N;
#pragma unroll
		for (int i = 0; i < RF; i++) {
			__builtin_amdgcn_sched_barrier(0);
#pragma unroll
			for (int j = 0; j < 2 * CF; j++) asm volatile("" : "+a"(acc[i][j]));  // (a row slab's accumulators are not read before its turn)
			if (whole) store_row<true, CF>(g, g.C, row0 + i * 16, col0, acc[i]);
			else store_row<false, CF>(g, g.C, row0 + i * 16, col0, acc[i]);
		}
		if (!more) break;
		pid = pid_n, cur = nxt;
		asm volatile("s_nop 7" ::: "memory");  // accumulator reads above, accumulator writes by the next tile's first MFMAs
	}
	wait_vmcnt<0>();  // the loads behind the last tile land in LDS too
}

template <int RF, int CF, int NS, int FMT>
static int launch_sized(Args g, hipStream_t stream) {
	using T = Tile<RF, CF, NS>;
	g.tiles_m = (g.M + T::M - 1) / T::M, g.tiles_n = (g.N + T::N - 1) / T::N;
	// (the loads run NS slices ahead, into the next tile's: a K that had fewer would be read past its end)
	ELF_REQUIRE(g.nk >= NS && g.splits == 1, "gemm_fp8: these tiles need %d blocks of K in one range", NS);
	const int64_t ntiles = (int64_t)g.tiles_m * g.tiles_n;
	ELF_REQUIRE(ntiles < (int64_t(1) << 30), "gemm_fp8: too many tiles for one launch");  // (their numbers are ints)
	auto kern = gemm_tile_kernel<RF, CF, NS, FMT>;
	static std::atomic<uint64_t> devices{0};
	if (int rc = allow_lds(reinterpret_cast<const void*>(kern), T::BYTES, devices)) return rc;
	constexpr int64_t MOST = 256 * T::PER_CU;
	ELF_LAUNCH(kern, dim3((uint32_t)(ntiles < MOST ? ntiles : MOST)), dim3(256), T::BYTES, stream, g);
	ELF_CHECK_HIP(hipGetLastError());
	return 0;
}

template <int FMT>
int launch_tile(const Args& g, int tile, hipStream_t stream) {
	return tile == 256 ? launch_sized<8, 4, 2, FMT>(g, stream) : launch_sized<4, 2, 2, FMT>(g, stream);
}
template int launch_tile<FP8_E4M3>(const Args& g, int tile, hipStream_t stream);
template int launch_tile<FP8_E5M2>(const Args& g, int tile, hipStream_t stream);

}  // namespace fp8
}  // namespace elf
