// gated_ffn_narrow.cuh — the gated block where its weights fit into LDS: many rows of few columns (the samples of a batch of rays or pixels), one pass over memory.
//
// A wave owns 32 rows.  Their products are formed transposed (features x rows), as in the framework's own MLP kernels: a lane holds one row, the rows of x ARE the B operand as they
// lie in memory, and the result of one product is, rounded and packed, the B operand of the next — a product does not care in which order k is summed, so the down projection's
// weights are staged in the order the registers have.  Nothing between x and y (or dy and dx) touches memory.  Included by gated_ffn.hip (activate).
// Bound by memory, of which 262144 x 32 - 64 - 16 in f16 needs 25 MB (forward) and 42 MB (backward): 8.7 us, of which 5 are the bytes and the rest a launch and the weights' staging,
// and 27 us + 4 for the sum.  There the backward pass is bound by the latency of its two phases: a wave waits half of its time, the LDS is busy for two fifths of it.
#pragma once

namespace ngp {
namespace ffn {

// 8 elements of a row from k on, zeros behind the width.  VEC: the row is 16-byte aligned and its width a multiple of 8.
template <class T, bool VEC>
__device__ __forceinline__ i32x4 load8(const T* row, uint32_t k, uint32_t width) {
	if (VEC) return k < width ? *(const i32x4*)(row + k) : i32x4{0, 0, 0, 0};
	typedef T t8 __attribute__((ext_vector_type(8)));
	t8 v;
#pragma unroll
	for (int e = 0; e < 8; ++e) {   // a load that is always allowed and a choice: no branch between the loads
		const T r = row[min(k + e, width ? width - 1 : 0)];
		v[e] = k + e < width ? r : (T)0.0f;
	}
	return __builtin_bit_cast(i32x4, v);
}
template <class T> __device__ __forceinline__ int pack2(float a, float b) {
	typedef T t2 __attribute__((ext_vector_type(2)));
	return __builtin_bit_cast(int, t2{(T)a, (T)b});
}
// registers 8 t .. 8 t + 7 of a 32 x 32 result as a B operand: slot (lane group g, j) is row 16 t + 8 (j >> 2) + 4 g + (j & 3) of the block
template <class T> __device__ __forceinline__ i32x4 as_operand(const f32x16& v, int t) {
	return i32x4{pack2<T>(v[8 * t], v[8 * t + 1]), pack2<T>(v[8 * t + 2], v[8 * t + 3]), pack2<T>(v[8 * t + 4], v[8 * t + 5]), pack2<T>(v[8 * t + 6], v[8 * t + 7])};
}
__device__ __forceinline__ f32x16 zero16() { return f32x16{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0}; }

// 32 x 32 results (lane: one row, block rows: columns of the output) -> row-major memory.  The two lane groups hold alternate quads of a row; one swap of half-waves makes 16 bytes of it.
template <class T>
__device__ __forceinline__ void store_transposed(const f32x16& v, T* row, uint32_t n0, uint32_t width, bool wide, int lane) {
	typedef T t8 __attribute__((ext_vector_type(8)));
#pragma unroll
	for (int p = 0; p < 2; ++p) {
		int a0 = pack2<T>(v[8 * p], v[8 * p + 1]), a1 = pack2<T>(v[8 * p + 2], v[8 * p + 3]), b0 = pack2<T>(v[8 * p + 4], v[8 * p + 5]), b1 = pack2<T>(v[8 * p + 6], v[8 * p + 7]);
		auto s0 = __builtin_amdgcn_permlane32_swap(a0, b0, false, false);
		auto s1 = __builtin_amdgcn_permlane32_swap(a1, b1, false, false);
		const i32x4 q = {(int)s0[0], (int)s1[0], (int)s0[1], (int)s1[1]};
		const uint32_t n = n0 + 16 * p + 8 * (lane >> 5);
		if (!row) continue;
		if (wide && n + 8 <= width) *(i32x4*)(row + n) = q;
		else {
			const t8 h = __builtin_bit_cast(t8, q);
#pragma unroll
			for (int e = 0; e < 8; ++e)
				if (n + e < width) row[n + e] = h[e];
		}
	}
}

// Fragment `rows r0 .., k k0 ..` of a row-major weight matrix in A-operand order, once per workgroup; perm: k in the order of as_operand.  By 16 (perm: 8) bytes where no piece ends
// inside a row's last one, else by elements: these are eight times the requests, and all workgroups make them of the same lines at once.
template <class T>
__device__ __forceinline__ void stage_fragment(lds_char* dst, const T* w, uint32_t rows, uint32_t cols, uint32_t r0, uint32_t k0, bool turned, bool perm, int lane) {
	typedef T t8 __attribute__((ext_vector_type(8)));
	t8 v;
	const uint32_t r = r0 + (lane & 31);
	if (!turned && cols % 8 == 0) {
		typedef i32x4 i32x4_any __attribute__((aligned(2)));
		typedef i32x2 i32x2_any __attribute__((aligned(2)));
		const T* row = w + (uint64_t)min(r, rows - 1) * cols;
		const uint32_t k = k0 + (perm ? 4 : 8) * (lane >> 5);
		i32x4 q = {0, 0, 0, 0};
		if (!perm) {
			if (r < rows && k < cols) q = *(const i32x4_any*)(row + k);
		} else {
			i32x2 lo = {0, 0}, hi = {0, 0};
			if (r < rows && k < cols) lo = *(const i32x2_any*)(row + k);
			if (r < rows && k + 8 < cols) hi = *(const i32x2_any*)(row + k + 8);
			q = i32x4{lo.x, lo.y, hi.x, hi.y};
		}
		*(__attribute__((address_space(3))) i32x4*)(dst + lane * 16) = q;
		return;
	}
#pragma unroll
	for (int j = 0; j < 8; ++j) {
		const uint32_t k = k0 + (perm ? 8 * (j >> 2) + 4 * (lane >> 5) + (j & 3) : 8 * (lane >> 5) + j);
		const uint32_t a = turned ? k : r, b = turned ? r : k;   // turned: the operand is w^T
		const T e = w[(uint64_t)min(a, rows - 1) * cols + min(b, cols - 1)];
		v[j] = a < rows && b < cols ? e : (T)0.0f;
	}
	*(__attribute__((address_space(3))) t8*)(dst + lane * 16) = v;
}

struct NarrowArgs {
	const void *x, *wg, *wu, *wd, *dy;
	void *y, *dx;
	uint64_t x_ld, y_ld, dy_ld, dx_ld;
	uint32_t rows, d, f, o;
	int act;
	float* partial;
};

// ---- forward: DB k-blocks of 16 input columns, OB blocks of 32 output columns, any number of blocks of 32 hidden columns ----
// workgroups a CU that the registers leave room for without spilling
constexpr int narrow_waves(int db, int ob, bool vec) { return ob == 4 ? (db <= 2 ? 3 : 2) : db <= 2 || (vec && db == 4) ? 4 : 2; }

template <class T, int DB, int OB, bool VEC>
__global__ void __launch_bounds__(256, narrow_waves(DB, OB, VEC)) narrow_forward_kernel(NarrowArgs a) {
	extern __shared__ __attribute__((aligned(1024))) char smem[];
	lds_char* const lds = lds_of(smem);
	constexpr int PER = 2 * DB + 2 * OB;   // fragments of 1 KiB per hidden block: gate, up (DB each), down (2 k-blocks x OB)
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const uint32_t tiles = (a.rows + 31) / 32, step = gridDim.x * 4;
	const bool wide = ((a.y_ld & 7) | ((uintptr_t)a.y & 15)) == 0;
	i32x4 x[DB], next[DB];
	auto load = [&](uint32_t tile, i32x4 (&v)[DB]) {
		const uint32_t m = min(tile * 32 + (lane & 31), a.rows - 1);   // rows behind the last are read as the last and not stored
		const T* row = (const T*)a.x + m * a.x_ld;
#pragma unroll
		for (int k = 0; k < DB; ++k) v[k] = load8<T, VEC>(row, k * 16 + 8 * (lane >> 5), a.d);
	};
	uint32_t tile = blockIdx.x * 4 + wave;
	if (tile < tiles) load(tile, next);
	const uint32_t fb_n = (a.f + 31) / 32;
	for (uint32_t i = wave; i < fb_n * PER; i += 4) {
		const uint32_t fb = i / PER, c = i % PER;
		if (c < 2 * DB) stage_fragment<T>(lds + i * 1024, (const T*)(c < DB ? a.wg : a.wu), a.f, a.d, fb * 32, (c % DB) * 16, false, false, lane);
		else stage_fragment<T>(lds + i * 1024, (const T*)a.wd, a.o, a.f, (c - 2 * DB) / 2 * 32, fb * 32 + (c & 1) * 16, false, true, lane);
	}
	__syncthreads();
	for (; tile < tiles; tile += step) {
#pragma unroll
		for (int k = 0; k < DB; ++k) x[k] = next[k];
		if (tile + step < tiles) load(tile + step, next);
		f32x16 y[OB];
#pragma unroll
		for (int b = 0; b < OB; ++b) y[b] = zero16();
		for (uint32_t fb = 0; fb < fb_n; ++fb) {
			const lds_char* w = lds + fb * (PER * 1024) + lane * 16;
			f32x16 g = zero16(), u = zero16();
#pragma unroll
			for (int k = 0; k < DB; ++k) {
				g = mfma<T>(*(const __attribute__((address_space(3))) i32x4*)(w + k * 1024), x[k], g);
				u = mfma<T>(*(const __attribute__((address_space(3))) i32x4*)(w + (DB + k) * 1024), x[k], u);
			}
			with_activation(a.act, [&](auto kind) {
#pragma unroll
				for (int i = 0; i < 16; ++i) g[i] = activate<decltype(kind)::value>(g[i]).x * u[i];
			});
#pragma unroll
			for (int t = 0; t < 2; ++t) {
				const i32x4 h = as_operand<T>(g, t);
#pragma unroll
				for (int b = 0; b < OB; ++b) y[b] = mfma<T>(*(const __attribute__((address_space(3))) i32x4*)(w + (2 * DB + 2 * b + t) * 1024), h, y[b]);
			}
		}
		const uint32_t m = tile * 32 + (lane & 31);
		T* row = m < a.rows ? (T*)a.y + m * a.y_ld : nullptr;
#pragma unroll
		for (int b = 0; b < OB; ++b) store_transposed<T>(y[b], row, b * 32, a.o, wide, lane);
	}
}

// ---- backward: DB, FB, OB blocks of 32 input, hidden and output columns; a workgroup of 4 waves takes 64 rows at a time ----
// Phase 1: a wave forms g, u and dh of 32 rows and half of the hidden blocks (all of one block: the waves of FB = 1 share the rows of x), and leaves dg, du, h beside x and dy in LDS.
// Phase 2: the 64 rows are the k of the weight gradients (both operands by transposed LDS reads) and the columns of dx; the gradients' 32 x 32 blocks are shared out over the waves
// and stay in registers over all rows of the workgroup.  At the end every workgroup leaves its sums in `partial`, and narrow_sum_kernel adds the workgroups in their order.
template <int DB, int FB, int OB> struct NarrowBackward {
	static constexpr int ROWS = 64, BLOCKS = 2 * FB * DB + FB * OB, OWN = (BLOCKS + 3) / 4;
	static constexpr int PX = DB * 64 + 16, PY = OB * 64 + 16, PF = FB * 64 + 16;                       // LDS row pitches in bytes
	static constexpr int OFF_X = 0, OFF_Y = OFF_X + ROWS * PX, OFF_G = OFF_Y + ROWS * PY, OFF_U = OFF_G + ROWS * PF, OFF_H = OFF_U + ROWS * PF, OFF_W = (OFF_H + ROWS * PF + 1023) / 1024 * 1024;
	static constexpr int W_GU = FB * 2 * DB, W_D = FB * 2 * OB;                                         // fragments: gate (the same again: up), down^T
	static constexpr int LDS_BYTES = OFF_W + (2 * W_GU + W_D) * 1024, RESIDENT = LDS_BYTES <= 80 * 1024 ? 2 : 1;
};
static_assert(NarrowBackward<2, 4, 2>::LDS_BYTES <= 160 * 1024, "the largest instance fits into a CU's LDS");

// rows `r0 ..` (contiguous direction), k (LDS rows) k0 .. k0 + 15 of a row-major LDS tile as an operand: two transposed reads
__device__ __forceinline__ i32x4 turned_fragment(const lds_char* tile, int pitch, int r0, int k0, int lane) {
	const lds_char* p = tile + (k0 + 8 * (lane >> 5) + ((lane & 15) >> 2)) * pitch + (r0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2;
	const i32x2 lo = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
	const i32x2 hi = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + 4 * pitch)));
	return i32x4{lo.x, lo.y, hi.x, hi.y};
}

template <class T, int DB, int FB, int OB, bool VEC>
__global__ void __launch_bounds__(256, (NarrowBackward<DB, FB, OB>::RESIDENT)) narrow_backward_kernel(NarrowArgs a) {
	using S = NarrowBackward<DB, FB, OB>;
	__shared__ __attribute__((aligned(1024))) char smem[S::LDS_BYTES];
	lds_char* const lds = lds_of(smem);
	lds_char* const w = lds + S::OFF_W;
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	auto weight = [&](int i) { return *(const __attribute__((address_space(3))) i32x4*)(w + i * 1024 + lane * 16); };
	f32x16 acc[S::OWN];
#pragma unroll
	for (int i = 0; i < S::OWN; ++i) acc[i] = zero16();
	const int tile_row = (wave & 1) * 32, half = wave >> 1, mine = tile_row + (lane & 31);   // this wave's rows and hidden blocks in phase 1
	constexpr int F1 = FB > 1 ? FB / 2 : 1;
	const uint32_t tiles = (a.rows + 63) / 64;
	const bool wide = ((a.dx_ld & 7) | ((uintptr_t)a.dx & 15)) == 0;
	i32x4 nx[2 * DB], ny[2 * OB];
	auto load = [&](uint32_t tile) {
		const uint64_t m = (uint64_t)tile * 64 + mine;
		const bool in = m < a.rows;                       // rows behind the last count as zeros: they are k of the weight gradients
		const T *rx = (const T*)a.x + (in ? m : 0) * a.x_ld, *ry = (const T*)a.dy + (in ? m : 0) * a.dy_ld;
#pragma unroll
		for (int k = 0; k < 2 * DB; ++k) nx[k] = load8<T, VEC>(rx, k * 16 + 8 * (lane >> 5), in ? a.d : 0);
#pragma unroll
		for (int k = 0; k < 2 * OB; ++k) ny[k] = load8<T, VEC>(ry, k * 16 + 8 * (lane >> 5), in ? a.o : 0);
	};
	uint32_t tile = blockIdx.x;
	if (tile < tiles) load(tile);
	for (int i = wave; i < 2 * S::W_GU + S::W_D; i += 4) {
		if (i < 2 * S::W_GU) {
			const int c = i % S::W_GU;
			stage_fragment<T>(w + i * 1024, (const T*)(i < S::W_GU ? a.wg : a.wu), a.f, a.d, c / (2 * DB) * 32, c % (2 * DB) * 16, false, false, lane);
		} else {
			const int c = i - 2 * S::W_GU;
			stage_fragment<T>(w + i * 1024, (const T*)a.wd, a.o, a.f, c / (2 * OB) * 32, c % (2 * OB) * 16, true, false, lane);
		}
	}
	// the 32 input columns of block db as rows, k hidden columns 16 c ..: the transpose of gate's (up's) fragments by transposed reads
	auto weight_turned = [&](int up, int db, int c) {
		const int f = c * 16 + 8 * (lane >> 5) + ((lane & 15) >> 2), d = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);   // of the block; four f by four d a lane's group
		const lds_char* p = w + (up * S::W_GU + (f >> 5) * 2 * DB + db * 2 + (d >> 4)) * 1024 + ((d >> 3) & 1) * 512 + (f & 31) * 16 + (d & 7) * 2;
		const i32x2 lo = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
		const i32x2 hi = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + 64)));   // f + 4
		return i32x4{lo.x, lo.y, hi.x, hi.y};
	};
	for (; tile < tiles; tile += gridDim.x) {
		__syncthreads();   // phase 2 of the rows before has been read (first time: the weights are there)
		i32x4 x[2 * DB], y[2 * OB];
#pragma unroll
		for (int k = 0; k < 2 * DB; ++k) x[k] = nx[k];
#pragma unroll
		for (int k = 0; k < 2 * OB; ++k) y[k] = ny[k];
		if (half == 0) {
#pragma unroll
			for (int k = 0; k < 2 * DB; ++k) *(__attribute__((address_space(3))) i32x4*)(lds + S::OFF_X + mine * S::PX + k * 32 + (lane >> 5) * 16) = x[k];
		}
		if (half == 1 || FB == 1) {
#pragma unroll
			for (int k = 0; k < 2 * OB; ++k) *(__attribute__((address_space(3))) i32x4*)(lds + S::OFF_Y + mine * S::PY + k * 32 + (lane >> 5) * 16) = y[k];
		}
		if (tile + gridDim.x < tiles) load(tile + gridDim.x);
		if (FB > 1 || half == 0) {
#pragma unroll
			for (int c = 0; c < F1; ++c) {
				const int fb = half * F1 + c;
				f32x16 g = zero16(), u = zero16(), dh = zero16();
#pragma unroll
				for (int k = 0; k < 2 * DB; ++k) {
					g = mfma<T>(weight(fb * 2 * DB + k), x[k], g);
					u = mfma<T>(weight(S::W_GU + fb * 2 * DB + k), x[k], u);
				}
#pragma unroll
				for (int k = 0; k < 2 * OB; ++k) dh = mfma<T>(weight(2 * S::W_GU + fb * 2 * OB + k), y[k], dh);
				with_activation(a.act, [&](auto kind) {
#pragma unroll
					for (int i = 0; i < 16; ++i) {
						const float2 r = activate<decltype(kind)::value>(g[i]);
						const float up = u[i];
						u[i] = dh[i] * r.x;
						g[i] = dh[i] * up * r.y;
						dh[i] = r.x * up;   // now du, dg, h
					}
				});
#pragma unroll
				for (int q = 0; q < 4; ++q) {
					const int at = mine * S::PF + (fb * 32 + 8 * q + 4 * (lane >> 5)) * 2;
					*(__attribute__((address_space(3))) i32x2*)(lds + S::OFF_G + at) = i32x2{pack2<T>(g[4 * q], g[4 * q + 1]), pack2<T>(g[4 * q + 2], g[4 * q + 3])};
					*(__attribute__((address_space(3))) i32x2*)(lds + S::OFF_U + at) = i32x2{pack2<T>(u[4 * q], u[4 * q + 1]), pack2<T>(u[4 * q + 2], u[4 * q + 3])};
					*(__attribute__((address_space(3))) i32x2*)(lds + S::OFF_H + at) = i32x2{pack2<T>(dh[4 * q], dh[4 * q + 1]), pack2<T>(dh[4 * q + 2], dh[4 * q + 3])};
				}
			}
		}
		__syncthreads();
#pragma unroll
		for (int i = 0; i < S::OWN; ++i) {
			const int b = wave + 4 * i;   // gate blocks, up blocks (fb, db), down blocks (fb, ob)
			if (S::BLOCKS % 4 && b >= S::BLOCKS) break;
			const bool down = b >= 2 * FB * DB;
			const int c = down ? b - 2 * FB * DB : b % (FB * DB), fb = c / (down ? OB : DB), r = c % (down ? OB : DB);
			const lds_char* ta = lds + (down ? S::OFF_Y : b < FB * DB ? S::OFF_G : S::OFF_U);
			const lds_char* tb = lds + (down ? S::OFF_H : S::OFF_X);
			const int pa = down ? S::PY : S::PF, pb = down ? S::PF : S::PX, ra = (down ? r : fb) * 32, rb = (down ? fb : r) * 32;
#pragma unroll
			for (int k = 0; k < S::ROWS / 16; ++k) acc[i] = mfma<T>(turned_fragment(ta, pa, ra, k * 16, lane), turned_fragment(tb, pb, rb, k * 16, lane), acc[i]);
		}
		if (a.dx) {
#pragma unroll
			for (int i = 0; i < (2 * DB + 3) / 4; ++i) {
				const int c = 3 - wave + 4 * i, rt = c & 1, db = c >> 1;   // rows rt * 32 .., input block db; first to the waves with fewer blocks of the gradients
				if (db >= DB) break;
				f32x16 v = zero16();
#pragma unroll
				for (int k = 0; k < 2 * FB; ++k) {
					const int at = (rt * 32 + (lane & 31)) * S::PF + k * 32 + (lane >> 5) * 16;
					v = mfma<T>(weight_turned(0, db, k), *(const __attribute__((address_space(3))) i32x4*)(lds + S::OFF_G + at), v);
					v = mfma<T>(weight_turned(1, db, k), *(const __attribute__((address_space(3))) i32x4*)(lds + S::OFF_U + at), v);
				}
				const uint64_t m = (uint64_t)tile * 64 + rt * 32 + (lane & 31);
				store_transposed<T>(v, m < a.rows ? (T*)a.dx + m * a.dx_ld : nullptr, db * 32, a.d, wide, lane);
			}
		}
	}
	if (!a.partial) return;
#pragma unroll
	for (int i = 0; i < S::OWN; ++i) {
		const int b = wave + 4 * i;
		if (S::BLOCKS % 4 && b >= S::BLOCKS) break;
		float* p = a.partial + ((uint64_t)blockIdx.x * S::BLOCKS + b) * 1024 + lane;
#pragma unroll
		for (int e = 0; e < 16; ++e) p[e * 64] = acc[i][e];
	}
}

// gradients = the workgroups' sums, added in their order: 16 waves take a sixteenth each of 64 elements of a block
template <class T>
__global__ void __launch_bounds__(1024) narrow_sum_kernel(const float* partial, uint32_t groups, uint32_t blocks, uint32_t db_n, uint32_t fb_n, uint32_t ob_n, uint32_t d, uint32_t f, uint32_t o, T* dwg, T* dwu, T* dwd) {
	__shared__ float sums[16][64];
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
	const uint32_t b = blockIdx.x >> 4, e = blockIdx.x & 15;   // block of 32 x 32, register of it
	float s = 0.0f;
	const float* p = partial + (uint64_t)b * 1024 + e * 64 + lane;
#pragma unroll 8
	for (uint32_t g = wave; g < groups; g += 16) s += p[(uint64_t)g * blocks * 1024];
	sums[wave][lane] = s;
	__syncthreads();
	if (wave) return;
	for (int i = 1; i < 16; ++i) s += sums[i][lane];
	const bool down = b >= 2 * fb_n * db_n;
	const uint32_t c = down ? b - 2 * fb_n * db_n : b % (fb_n * db_n), fb = c / (down ? ob_n : db_n), r = c % (down ? ob_n : db_n);
	const uint32_t row = (down ? r : fb) * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3), col = (down ? fb : r) * 32 + (lane & 31);
	if (down) { if (row < o && col < f) dwd[(uint64_t)row * f + col] = (T)s; }
	else if (row < f && col < d) (b < fb_n * db_n ? dwg : dwu)[(uint64_t)row * d + col] = (T)s;
}

} // namespace ffn
} // namespace ngp
