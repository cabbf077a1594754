// matmul_mfma.cuh — tiled matrix products C[m][n] = sum_k M[m][k] N[n][k] on v_mfma_f32_16x16x32_{f16,bf16}, the core of the gated feed-forward block (gated_ffn.hip)
// and of the Muon step (muon.hip).
//
// Scheme.  A workgroup owns a BN x BM tile and walks k in steps of 32.  Both operands of a step go from memory into LDS by DMA (buffer_load ... lds, 16 bytes a lane: no
// registers, no ds_write), three steps ahead of the matrix instructions (a ring of four LDS buffers).  The buffer descriptor of a step ends where the operand ends, and the hardware returns
// zero behind it, so the last rows and the last k of any size need no branch; a chunk behind k in the middle of a row asks for an offset behind the descriptor.
// Operands come in two layouts:
//   KC   [rows][k], k contiguous:     LDS [row][k], a fragment (lane: one row, 8 k) is one ds_read_b128;
//   RC   [k][rows], rows contiguous:  LDS [k][row], a fragment is two ds_read_b64_tr_b16 (the LDS unit transposes 4 x 16 blocks on the way out).
// Bank conflicts: the DMA writes LDS linearly, so the 16-byte chunks of a row are permuted by which chunk each lane ASKS for, chunk ^ swizzle(row): for KC such that 16 rows of
// one chunk column cover every bank once, for RC such that the four k rows of a transposed block and its neighbour fall on different 32-byte units.  Measured: no conflicts for rows of
// 128 bytes (the Muon step's), a tenth of the LDS cycles for RC; but half of them for KC rows of 64 bytes (28 % of the CU's cycles at 8192 x 4096 - 8192, behind the MFMAs).
// What bounds it.  The matrix pipes and, below them, power: at 8192 x 4096 x 8192 the clock falls to 1.4 GHz (1.6 to 1.8 in the Muon step's products), the pipes are busy for three
// quarters of it and a product of that size runs at 1.3 PFLOP/s (y of the gated block, 0.42 ms), where the library's runs at 1.25 to 1.55 by layout and type.  Three things keep the pipes fed: fragments are read half a step
// ahead of the MFMAs that take them; the DMA instructions stand between MFMAs, two to a half step (eight in a row block the wave's issue, and with it its MFMAs, until the memory
// pipe has taken them); and the only waits are for data that was asked for two steps ago.
// The N side is the A operand of the MFMA: a lane then holds four consecutive n of one m per register quad, which is the contiguous direction of the output.
#pragma once

#include "ngp_device.cuh"

#pragma clang fp contract(fast)

namespace ngp {
namespace mm {

typedef _Float16 f16;
typedef __bf16 b16;
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef b16 b16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

enum { KC = 0, RC = 1 };

struct Mat {             // rows x k, see above; ld in elements, a multiple of 8; p 16-byte aligned; KC: k a multiple of 8
	const void* p;
	uint64_t ld;
	uint32_t rows, k;
};

template <class T> __device__ __forceinline__ f32x4 mfma16(i32x4 a, i32x4 b, f32x4 c);
template <> __device__ __forceinline__ f32x4 mfma16<f16>(i32x4 a, i32x4 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0); }
template <> __device__ __forceinline__ f32x4 mfma16<b16>(i32x4 a, i32x4 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0); }
template <class T> __device__ __forceinline__ f32x16 mfma(i32x4 a, i32x4 b, f32x16 c);
template <> __device__ __forceinline__ f32x16 mfma<f16>(i32x4 a, i32x4 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0); }
template <> __device__ __forceinline__ f32x16 mfma<b16>(i32x4 a, i32x4 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0); }

__device__ __forceinline__ lds_char* lds_of(void* p) { return (lds_char*)(__attribute__((address_space(3))) void*)p; }

// 16 bytes of every lane straight into LDS at `lds` + 16 lane.  The instruction returns nothing to a register, and the compiler, told of it as a builtin, would wait for ALL
// DMA in flight before each LDS read; written here, the waits are the two below and stand where the buffers change hands.  m0 is the compiler's too (its own LDS DMA, messages):
// without the clobber it keeps a value there across this one.  Its warning that m0 is not preserved is what the clobber says.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma16(i32x4 rsrc, lds_char* lds, int voff) {
	asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"((uint32_t)(uintptr_t)lds), "v"(voff), "s"(rsrc) : "m0", "memory");
}
#pragma clang diagnostic pop
// every DMA of this wave but the last PENDING has landed, every LDS read of it has returned; then all waves
template <int PENDING = 0> __device__ __forceinline__ void wait_and_sync() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(PENDING) : "memory"); }

// One operand's tile of BR rows x BK k: who loads what, and how a fragment is read back.
template <int LAY, int BR, int THREADS, int BK>
struct Tile {
	static constexpr int BYTES = BR * BK * 2;
	static constexpr int CHUNKS = LAY == KC ? BK / 8 : BR / 8;       // 16-byte chunks per LDS row
	static constexpr int LOADS = BYTES / 16 / THREADS;
	static_assert(BYTES % (16 * THREADS) == 0, "every thread issues the same number of loads");
	static __device__ __forceinline__ int swizzle(int r) {
		if (LAY == KC) return BK == 64 ? (r >> 1) & 7 : (r >> 2) & 3;
		return CHUNKS >= 16 ? (r & 3) << 1 | (r & 8) : (r & 2) | (r & 8) >> 1;
	}

	// All but k_here, k_past and voff are uniform and 32 bits where the loop touches them: the next descriptor is five scalar instructions (worked out in 64 bits, with a compare on the
	// vector unit, it was a quarter of a small tile's step).
	const char* base;        // of this step
	int64_t step_bytes;
	int row_bytes, end_bytes;   // KC: bytes to the last row of the tile, 0.  RC: bytes from row to row (of k), bytes of the operand in a row from here on
	int k_left;
	int k_here;              // KC: k of this thread's chunk in the step; beyond `k_left` it reads zero
	bool k_past;
	int voff[LOADS];

	// steps of BK from k0 on (a multiple of BK)
	__device__ __forceinline__ void init(const Mat& m, uint32_t row0, uint32_t k0, int tid) {
		const int ld2 = (int)((uint32_t)m.ld * 2u);
		const bool any = row0 < m.rows;   // a tile without rows reads nothing
		if (LAY == KC) {
			base = (const char*)m.p + ((uint64_t)row0 * m.ld + k0) * 2;
			step_bytes = BK * 2;
			const uint32_t rows = any ? m.rows - row0 : 0;
			row_bytes = any ? (int)((rows < BR ? rows : BR) - 1) * ld2 : -0x40000000;
			end_bytes = 0;
		} else {
			base = (const char*)m.p + ((uint64_t)k0 * m.ld + row0) * 2;
			step_bytes = (int64_t)m.ld * BK * 2;
			row_bytes = any ? ld2 : 0;
			end_bytes = any ? (int)((m.rows - row0) * 2u) : -0x40000000;
		}
		k_left = (int)(m.k - k0);
#pragma unroll
		for (int i = 0; i < LOADS; ++i) {
			const int slot = i * THREADS + tid, r = slot / CHUNKS, c = (slot % CHUNKS) ^ swizzle(r);
			voff[i] = (int)((uint32_t)r * (uint32_t)m.ld * 2u) + c * 16;
			if (LAY == KC && i == 0) k_here = c * 8;   // the same for every i: a thread's rows differ by a multiple of 16
		}
		asm volatile("s_nop 4");   // a word of the descriptors below that came from the vector unit must be five wait states old when a memory instruction reads it
	}
	// descriptor of the current step (it ends where the operand does: what lies behind reads as zero), then on to the next
	__device__ __forceinline__ i32x4 next() {
		const uint64_t b = (uint64_t)base;
		const int here = k_left < BK ? k_left : BK, end = LAY == KC ? row_bytes + 2 * k_left : (here - 1) * row_bytes + end_bytes;
		const i32x4 r = {(int)(uint32_t)b, (int)((uint32_t)(b >> 32) & 0xffffu), end > 0 ? end : 0, 0x00020000};
		k_past = LAY == KC && k_here >= k_left;
		base += step_bytes;
		k_left -= BK;
		return r;
	}
	// the i-th DMA of the step that next() gave into `lds` (wave-uniform)
	__device__ __forceinline__ void issue(const i32x4& r, int i, lds_char* lds, int wave) const {
		dma16(r, lds + (i * THREADS + wave * 64) * 16, k_past ? (int)0x80000000 : voff[i]);
	}
	// fragment of rows row0 .. row0 + 15, all 32 k: lane l has row l & 15 and k = 8 (l >> 4) .. + 7
	static __device__ __forceinline__ i32x4 frag(const lds_char* lds, int row0, int lane) {
		static_assert(BK == 32, "one k-block a step");
		if (LAY == KC) {
			const int r = row0 + (lane & 15), c = (lane >> 4) ^ swizzle(lane & 15);
			return *(const __attribute__((address_space(3))) i32x4*)(lds + r * 64 + c * 16);
		}
		const int k = 8 * (lane >> 4) + ((lane & 15) >> 2), c = row0 / 8 + ((lane & 3) >> 1);   // the four lanes of a k bring 16 rows; k + 4 has the same swizzle
		const lds_char* p = lds + k * (CHUNKS * 16) + (c ^ swizzle(k)) * 16 + (lane & 1) * 8;
		const i32x2 lo = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
		const i32x2 hi = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + 4 * CHUNKS * 16)));
		return i32x4{lo.x, lo.y, hi.x, hi.y};
	}
};

// The product's main loop.  NM N-side matrices of BN rows each share one M-side tile of BM rows (gate and up projection: NM = 2).  WN x WM waves; a wave owns BN / WN rows of every
// N-side matrix and BM / WM rows of the M side.
template <class T, int NLAY, int MLAY, int NM, int BN, int BM, int WN, int WM>
struct Product {
	static constexpr int BK = 32, STAGES = 4;   // a power of two: with a counted ring position instead of the step's low bits the kernels lost 2.5 %
	static constexpr int THREADS = 64 * WN * WM, NB = BN / WN / 16, MB = BM / WM / 16, HALF = NM * NB / 2;
	using NT = Tile<NLAY, BN, THREADS, BK>;
	using MT = Tile<MLAY, BM, THREADS, BK>;
	static constexpr int STAGE_BYTES = NM * NT::BYTES + MT::BYTES, LDS_BYTES = STAGES * STAGE_BYTES;
	static constexpr int LOADS = NM * NT::LOADS + MT::LOADS, EARLY = LOADS / 2;   // a step's DMA: the first EARLY beside its first half of MFMAs, the others beside its second

	// acc[j][nb][mb] += the product over k0 .. k1 of rows n0.. of n[j] and m0.. of m.  Every thread of the workgroup calls it; LDS is
	// free again on return.
	static __device__ __forceinline__ void run(f32x4 (&acc)[NM][NB][MB], const Mat* n, const Mat& m, uint32_t n0, uint32_t m0, uint32_t k0, uint32_t k1, lds_char* lds) {
		const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wave % WN, wm = wave / WN;
		NT nt[NM];
		MT mt;
#pragma unroll
		for (int j = 0; j < NM; ++j) nt[j].init(n[j], n0, k0, tid);
		mt.init(m, m0, k0, tid);
		const int steps = (int)((k1 - k0 + BK - 1) / BK);
		// Steps are issued without end (those behind the last one would bring the next split's or, behind the operand, zeros: nothing reads them), so that the count of DMA in flight is
		// the same in every step and the waits can be counted.
		i32x4 rn[NM], rm;
		int ahead = 0;
		lds_char* to = lds;
		auto next_step = [&]() {
#pragma unroll
			for (int j = 0; j < NM; ++j) rn[j] = nt[j].next();
			rm = mt.next();
			to = lds + (ahead & (STAGES - 1)) * STAGE_BYTES;
			++ahead;
		};
		auto issue = [&](int i) {   // i is a constant where it is called
			if (i < NM * NT::LOADS) nt[i / NT::LOADS].issue(rn[i / NT::LOADS], i % NT::LOADS, to + (i / NT::LOADS) * NT::BYTES, wave);
			else mt.issue(rm, i - NM * NT::LOADS, to + NM * NT::BYTES, wave);
		};
		i32x4 fm[2][MB], fn[2][HALF];   // M side of this step and the next; N side of this half and the next
		auto read_m = [&](int set, int b, const lds_char* p) { fm[set][b] = MT::frag(p + NM * NT::BYTES, wm * (BM / WM) + b * 16, lane); };
		auto read_n = [&](int half, int i, const lds_char* p) {
			const int u = half * HALF + i;
			fn[half][i] = NT::frag(p + u / NB * NT::BYTES, wn * (BN / WN) + u % NB * 16, lane);
		};
		// half a step's MFMAs, with `count` other instructions (DMA, LDS reads) spread between them: other(0) .. other(count - 1)
		auto multiply = [&](int half, int set, int count, auto other) {
			constexpr int COUNT = HALF * MB;
			__builtin_amdgcn_sched_barrier(0);
#pragma unroll
			for (int i = 0; i < COUNT; ++i) {
				const int u = half * HALF + i / MB, c = i % MB;
				acc[u / NB][u % NB][c] = mfma16<T>(fn[half][i / MB], fm[set][c], acc[u / NB][u % NB][c]);
#pragma unroll
				for (int d = 0; d < count; ++d)
					if (d * COUNT / count == i) {
						__builtin_amdgcn_sched_barrier(0);
						other(d);
						__builtin_amdgcn_sched_barrier(0);
					}
			}
			__builtin_amdgcn_sched_barrier(0);
		};
#pragma unroll
		for (int s = 0; s < STAGES - 1; ++s) {
			next_step();
#pragma unroll
			for (int i = 0; i < LOADS; ++i) issue(i);
		}
		wait_and_sync<(STAGES - 2) * LOADS>();
#pragma unroll
		for (int b = 0; b < MB; ++b) read_m(0, b, lds);
#pragma unroll
		for (int i = 0; i < HALF; ++i) read_n(0, i, lds);
		auto step = [&](int s, int set) {   // set: s & 1, a constant
			next_step();
			const lds_char* p = lds + (s & (STAGES - 1)) * STAGE_BYTES;
			multiply(0, set, HALF + EARLY, [&](int d) { if (d < HALF) read_n(1, d, p); else issue(d - HALF); });
			wait_and_sync<(STAGES - 3) * LOADS + EARLY>();   // the next step has landed, this one has been read: its buffer is the next to be filled
			const lds_char* q = lds + ((s + 1) & (STAGES - 1)) * STAGE_BYTES;   // behind the last step: not used
			multiply(1, set, MB + HALF + LOADS - EARLY, [&](int d) { if (d < MB) read_m(set ^ 1, d, q); else if (d < MB + HALF) read_n(0, d - MB, q); else issue(EARLY + d - MB - HALF); });
		};
		int s = 0;
		for (; s + 1 < steps; s += 2) {
			step(s, 0);
			step(s + 1, 1);
		}
		if (s < steps) step(s, 0);
		wait_and_sync();   // the DMA behind the last step too: LDS may belong to another workgroup next
	}
};

// ---- which tile a workgroup takes --------------------------------------------------------------------------------------------------------
// Workgroups go to the 8 XCDs in turn, each with its own L2: give an XCD one contiguous run of the tile order, and walk that order eight tile rows at a time, so that the
// tiles in flight on one XCD share both operands' panels.
__device__ __forceinline__ uint32_t xcd_order(uint32_t pid, uint32_t total) {
	const uint32_t xcd = pid & 7, per = total >> 3, rem = total & 7;
	return xcd * per + (xcd < rem ? xcd : rem) + (pid >> 3);
}
__device__ __forceinline__ void tile_of(uint32_t pid, uint32_t total, uint32_t tiles_n, uint32_t tiles_m, uint32_t& tn, uint32_t& tm, uint32_t& split) {
	uint32_t t = xcd_order(pid, total);
	const uint32_t tiles = tiles_n * tiles_m;
	split = t / tiles;
	t -= split * tiles;
	constexpr uint32_t G = 8;
	const uint32_t group = t / (G * tiles_n), first = group * G, size = tiles_m - first < G ? tiles_m - first : G;
	t -= group * G * tiles_n;
	tm = first + t % size;
	tn = t / size;
}

// ---- epilogue ----------------------------------------------------------------------------------------------------------------------------
template <class T> struct Out { T* p; uint64_t ld; uint32_t rows, cols; };   // row-major; columns are the N side

// A wave brings 32 rows x NBLK * 16 columns of results into row order through LDS of its own (Rows<NBLK>::BYTES), so that a row's columns leave in 16-byte pieces: put_block rounds a
// 16 x 16 block (once, to nearest even) into it, store_rows writes the rows.  Register layout of a block: lane l holds row m = l & 15 and columns n = 4 (l >> 4) .. + 3.
// The wave's own LDS operations are in order: no barrier between the two.
template <int NBLK> struct Rows { static constexpr int PITCH = NBLK * 32 + 16, BYTES = 32 * PITCH; };

template <class T, int NBLK>
__device__ __forceinline__ void put_block(const f32x4& v, int b, int upper, lds_char* lds, int lane) {   // block b of the row; upper: rows 16 .. 31
	typedef T t4 __attribute__((ext_vector_type(4)));
	*(__attribute__((address_space(3))) t4*)(lds + (upper * 16 + (lane & 15)) * Rows<NBLK>::PITCH + (b * 16 + 4 * (lane >> 4)) * 2) = t4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
}

template <class T, int NBLK>
__device__ __forceinline__ void store_rows(const Out<T>& o, uint32_t n0, uint32_t m0, const lds_char* lds, int lane) {
	typedef T t8 __attribute__((ext_vector_type(8)));
	constexpr int PIECES = NBLK * 2, ROWS = 64 / PIECES;
	const bool wide = (((uint64_t)o.p | (o.ld * 2)) & 15) == 0;
	const int piece = lane % PIECES;
	const uint32_t n = n0 + piece * 8;
#pragma unroll
	for (int r = 0; r < 32; r += ROWS) {
		const int row = r + lane / PIECES;
		const t8 h = *(const __attribute__((address_space(3))) t8*)(lds + row * Rows<NBLK>::PITCH + piece * 16);
		const uint32_t m = m0 + row;
		if (m >= o.rows) continue;
		T* p = o.p + (uint64_t)m * o.ld + n;
		if (wide && n + 8 <= o.cols) *(t8*)p = h;
		else
#pragma unroll
			for (int e = 0; e < 8; ++e)
				if (n + e < o.cols) p[e] = h[e];
	}
}

} // namespace mm
} // namespace ngp
