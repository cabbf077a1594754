// gated_ffn.hip — the gated feed-forward block y = (act(x Wg^T) * (x Wu^T)) Wd^T, forward and backward (include/ngp_hip.h: ngp_hip_gated_ffn_*).
//
//   forward    h = act(g) * u with g = x Wg^T, u = x Wu^T;  y = h Wd^T
//   backward   dh = dy Wd;  dg = dh * u * act'(g);  du = dh * act(g);  dx = dg Wg + du Wu;  dWg = dg^T x;  dWu = du^T x;  dWd = dy^T h
//
// Rounding: every product is accumulated in fp32.  What goes through memory between two products (h forward; dg, du, h backward) is rounded once to the tensors' type: the next
// product's operands are of that type, and one rounding of the operand beside one of the result is sqrt(2) of the error of rounding the result alone.  g and u are never stored:
// the backward pass computes them again, next to dh, in the registers where all three meet (a stored, rounded g would add a third rounding to every gradient).
#include <algorithm>
#include <stdio.h>
#include "ngp_device.cuh"
#include "matmul_mfma.cuh"

#pragma clang fp contract(fast)

namespace ngp {
namespace ffn {

using namespace mm;

// act(g) and act'(g)
template <int ACT>
__device__ __forceinline__ float2 activate(float g) {
	if (ACT == NGP_ACT_NONE) return make_float2(g, 1.0f);
	if (ACT == NGP_ACT_RELU) return g <= 0.0f ? make_float2(0.0f, 0.0f) : make_float2(g, 1.0f);   // a NaN stays one
	if (ACT == NGP_ACT_GELU) {   // g Phi(g); erfc keeps the small tail's digits
		const float phi = 0.5f * erfcf(g * -0.70710678f);
		return make_float2(g * phi, phi + g * 0.39894228f * __expf(-0.5f * g * g));
	}
	const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-g));   // both within 2 ulp
	if (ACT == NGP_ACT_LOGISTIC) return make_float2(s, s * (1.0f - s));
	return make_float2(g * s, s * (1.0f + g * (1.0f - s)));     // NGP_ACT_SILU
}
template <int V> struct Constant { static constexpr int value = V; };
// f(Constant<act>): the choice is made once, outside the loops over a tile
template <class F>
__device__ __forceinline__ void with_activation(int act, F f) {
	switch (act) {
		case NGP_ACT_NONE: f(Constant<NGP_ACT_NONE>()); break;
		case NGP_ACT_RELU: f(Constant<NGP_ACT_RELU>()); break;
		case NGP_ACT_LOGISTIC: f(Constant<NGP_ACT_LOGISTIC>()); break;
		case NGP_ACT_SILU: f(Constant<NGP_ACT_SILU>()); break;
		default: f(Constant<NGP_ACT_GELU>());
	}
}

} // namespace ffn
} // namespace ngp

#include "gated_ffn_narrow.cuh"
#include "gated_ffn_few.cuh"

namespace ngp {
namespace ffn {

template <bool BIG> struct Shape;   // BIG: 256 x 256 in 8 waves, one workgroup a CU; else 128 x 128 in 4 waves, two a CU
template <> struct Shape<true> { static constexpr int N = 256, M = 256, WN = 2, WM = 4, THREADS = 512, RESIDENT = 2; };
template <> struct Shape<false> { static constexpr int N = 128, M = 128, WN = 2, WM = 2, THREADS = 256, RESIDENT = 2; };

template <int NM, int NB, int MB> __device__ __forceinline__ void clear(f32x4 (&acc)[NM][NB][MB]) {
#pragma unroll
	for (int j = 0; j < NM; ++j)
#pragma unroll
		for (int a = 0; a < NB; ++a)
#pragma unroll
			for (int b = 0; b < MB; ++b) acc[j][a][b] = f32x4{0, 0, 0, 0};
}

// h = act(x Wg^T) * (x Wu^T): one tile of rows of x against N / 2 gate rows and the same N / 2 up rows, so that both factors of an h meet in one lane
template <class T, bool BIG>
__global__ void __launch_bounds__(Shape<BIG>::THREADS, Shape<BIG>::RESIDENT) gate_up_kernel(Mat x, Mat wg, Mat wu, Out<T> h, int act, uint32_t tiles_n, uint32_t tiles_m) {
	using S = Shape<BIG>;
	using P = Product<T, KC, KC, 2, S::N / 2, S::M, S::WN, S::WM>;
	__shared__ __attribute__((aligned(1024))) char lds[P::LDS_BYTES];
	uint32_t tn, tm, split;
	tile_of(blockIdx.x, gridDim.x, tiles_n, tiles_m, tn, tm, split);
	f32x4 acc[2][P::NB][P::MB];
	clear(acc);
	const Mat w[2] = {wg, wu};
	const uint32_t n0 = tn * (S::N / 2), m0 = tm * S::M;
	P::run(acc, w, x, n0, m0, 0, x.k, lds_of(lds));
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % S::WN, wm = wave / S::WN;
	lds_char* mine = lds_of(lds) + wave * Rows<P::NB>::BYTES;
#pragma unroll
	for (int c = 0; c < P::MB; ++c) {
		with_activation(act, [&](auto a) {
#pragma unroll
			for (int b = 0; b < P::NB; ++b) {
				f32x4 v;
#pragma unroll
				for (int i = 0; i < 4; ++i) v[i] = activate<decltype(a)::value>(acc[0][b][c][i]).x * acc[1][b][c][i];
				put_block<T, P::NB>(v, b, c & 1, mine, lane);
			}
		});
		if (c & 1) store_rows<T, P::NB>(h, n0 + wn * (P::NB * 16), m0 + wm * (P::MB * 16) + (c - 1) * 16, mine, lane);
	}
}

struct Pair { Mat n, m; };                        // one product's operands
template <class T> struct Rows2 { Out<T> a, b; uint32_t a_rows; };   // rows 0 .. a_rows - 1 of the result go to a, the rest to b (b starts at row a_rows)

template <class T, int NB, int MB>
__device__ __forceinline__ void store_tile(f32x4 (&acc)[1][NB][MB], const Rows2<T>& o, uint32_t n0, uint32_t m0, lds_char* lds, int lane) {
#pragma unroll
	for (int c = 0; c < MB; ++c) {
#pragma unroll
		for (int b = 0; b < NB; ++b) put_block<T, NB>(acc[0][b][c], b, c & 1, lds, lane);
		if (!(c & 1)) continue;
		const uint32_t m = m0 + (c - 1) * 16;   // a_rows is a multiple of 32 wherever b is used: 32 rows never lie on both sides
		if (m < o.a_rows) store_rows<T, NB>(o.a, n0, m, lds, lane);
		else store_rows<T, NB>(o.b, n0, m - o.a_rows, lds, lane);
	}
}

// C = sum of up to two products of the same k (dx = dg Wg + du Wu), all of it or one split.  With splits, a workgroup leaves its accumulators in `partial` as they lie in the registers,
// and split_sum_kernel adds the splits in their order: the result does not depend on which workgroup ends first.
template <class T, int NLAY, int MLAY, bool BIG>
__global__ void __launch_bounds__(Shape<BIG>::THREADS, Shape<BIG>::RESIDENT) product_kernel(Pair p0, Pair p1, int n_products, Rows2<T> out, uint32_t tiles_n, uint32_t tiles_m, uint32_t splits, uint32_t k_split, float* partial) {
	using S = Shape<BIG>;
	using P = Product<T, NLAY, MLAY, 1, S::N, S::M, S::WN, S::WM>;
	__shared__ __attribute__((aligned(1024))) char lds[P::LDS_BYTES];
	uint32_t tn, tm, split;
	tile_of(blockIdx.x, gridDim.x, tiles_n, tiles_m, tn, tm, split);
	f32x4 acc[1][P::NB][P::MB];
	clear(acc);
	const uint32_t n0 = tn * S::N, m0 = tm * S::M;
	if (partial) {   // split s of product s / splits
		const bool second = split >= splits;
		const Pair& p = second ? p1 : p0;
		const uint32_t k0 = (second ? split - splits : split) * k_split;
		P::run(acc, &p.n, p.m, n0, m0, k0, p.n.k - k0 < k_split ? p.n.k : k0 + k_split, lds_of(lds));
	} else {
		P::run(acc, &p0.n, p0.m, n0, m0, 0, p0.n.k, lds_of(lds));
		if (n_products == 2) P::run(acc, &p1.n, p1.m, n0, m0, 0, p1.n.k, lds_of(lds));
	}
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % S::WN, wm = wave / S::WN;
	if (partial) {
		float* q = partial + ((uint64_t)split * tiles_n * tiles_m + (uint64_t)tm * tiles_n + tn) * (S::N * S::M) + threadIdx.x * 4;
#pragma unroll
		for (int b = 0; b < P::NB; ++b)
#pragma unroll
			for (int c = 0; c < P::MB; ++c) *(f32x4*)(q + (b * P::MB + c) * (S::THREADS * 4)) = acc[0][b][c];
		return;
	}
	store_tile<T, P::NB, P::MB>(acc, out, n0 + wn * (P::NB * 16), m0 + wm * (P::MB * 16), lds_of(lds) + wave * Rows<P::NB>::BYTES, lane);
}

// `splits` partials -> ceil(splits / SUM_FAN) in the first of them, sixteen neighbours in their order: a long list of splits would otherwise be one workgroup's serial work
constexpr uint32_t SUM_FAN = 16;
__global__ void __launch_bounds__(256) split_fold_kernel(float* partial, uint32_t splits, uint64_t floats) {   // floats: of one split, a multiple of 1024
	const uint64_t blocks = floats / 1024, at = (blockIdx.x % blocks) * 1024 + threadIdx.x * 4;
	const uint32_t first = (uint32_t)(blockIdx.x / blocks) * SUM_FAN, end = min(first + SUM_FAN, splits);
	f32x4 v = *(const f32x4*)(partial + first * floats + at);
#pragma unroll 4
	for (uint32_t s = first + 1; s < end; ++s) v += *(const f32x4*)(partial + s * floats + at);
	*(f32x4*)(partial + first * floats + at) = v;
}

// the splits of a tile (every `every`-th of them), added in order, rounded once
template <class T, bool BIG>
__global__ void __launch_bounds__(Shape<BIG>::THREADS) split_sum_kernel(const float* partial, uint32_t splits, uint32_t every, Rows2<T> out, uint32_t tiles_n, uint32_t tiles_m) {
	using S = Shape<BIG>;
	constexpr int NB = S::N / S::WN / 16, MB = S::M / S::WM / 16;
	__shared__ __attribute__((aligned(16))) char lds[S::WN * S::WM * Rows<NB>::BYTES];
	const uint32_t tn = blockIdx.x % tiles_n, tm = blockIdx.x / tiles_n;
	const float* q = partial + (uint64_t)blockIdx.x * (S::N * S::M) + threadIdx.x * 4;
	const uint64_t stride = (uint64_t)every * tiles_n * tiles_m * (S::N * S::M);
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % S::WN, wm = wave / S::WN;
	f32x4 acc[1][NB][MB];
	clear(acc);
	for (uint32_t s = 0; s < splits; ++s, q += stride)
#pragma unroll
		for (int b = 0; b < NB; ++b)
#pragma unroll
			for (int c = 0; c < MB; ++c) acc[0][b][c] += *(const f32x4*)(q + (b * MB + c) * (S::THREADS * 4));
	store_tile<T, NB, MB>(acc, out, tn * S::N + wn * (NB * 16), tm * S::M + wm * (MB * 16), lds_of(lds) + wave * Rows<NB>::BYTES, lane);
}

// g, u and dh of a tile in one set of registers; from them dg, du (next to each other: d[m][0 .. f8) and d[m][f8 .. 2 f8)) and h
template <class T, bool BIG>
__global__ void __launch_bounds__(Shape<BIG>::THREADS, Shape<BIG>::RESIDENT) hidden_backward_kernel(Mat x, Mat wg, Mat wu, Mat dy, Mat wd, Out<T> dg, Out<T> du, Out<T> h, int act, uint32_t tiles_n, uint32_t tiles_m) {
	using S = Shape<BIG>;
	using P = Product<T, KC, KC, 2, S::N / 2, S::M, S::WN, S::WM>;
	using Q = Product<T, RC, KC, 1, S::N / 2, S::M, S::WN, S::WM>;
	__shared__ __attribute__((aligned(1024))) char lds[P::LDS_BYTES];
	static_assert(Q::LDS_BYTES <= P::LDS_BYTES, "one buffer for both");
	uint32_t tn, tm, split;
	tile_of(blockIdx.x, gridDim.x, tiles_n, tiles_m, tn, tm, split);
	f32x4 gu[2][P::NB][P::MB], dh[1][P::NB][P::MB];
	clear(gu);
	const Mat w[2] = {wg, wu};
	const uint32_t n0 = tn * (S::N / 2), m0 = tm * S::M;
	P::run(gu, w, x, n0, m0, 0, x.k, lds_of(lds));
	clear(dh);
	Q::run(dh, &wd, dy, n0, m0, 0, dy.k, lds_of(lds));
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % S::WN, wm = wave / S::WN;
	lds_char* mine = lds_of(lds) + wave * (3 * Rows<P::NB>::BYTES);
	static_assert(S::WN * S::WM * 3 * Rows<P::NB>::BYTES <= P::LDS_BYTES, "three results of every wave at once");
	const uint32_t n = n0 + wn * (P::NB * 16);
#pragma unroll
	for (int c = 0; c < P::MB; ++c) {
		with_activation(act, [&](auto kind) {
#pragma unroll
			for (int b = 0; b < P::NB; ++b) {
				f32x4 g, u, v;
#pragma unroll
				for (int i = 0; i < 4; ++i) {
					const float2 a = activate<decltype(kind)::value>(gu[0][b][c][i]);
					const float up = gu[1][b][c][i], d = dh[0][b][c][i];
					v[i] = a.x * up;
					g[i] = d * up * a.y;
					u[i] = d * a.x;
				}
				put_block<T, P::NB>(v, b, c & 1, mine, lane);
				put_block<T, P::NB>(g, b, c & 1, mine + Rows<P::NB>::BYTES, lane);
				put_block<T, P::NB>(u, b, c & 1, mine + 2 * Rows<P::NB>::BYTES, lane);
			}
		});
		if (!(c & 1)) continue;
		const uint32_t m = m0 + wm * (P::MB * 16) + (c - 1) * 16;
		store_rows<T, P::NB>(h, n, m, mine, lane);
		store_rows<T, P::NB>(dg, n, m, mine + Rows<P::NB>::BYTES, lane);
		store_rows<T, P::NB>(du, n, m, mine + 2 * Rows<P::NB>::BYTES, lane);
	}
}

// rows of any width, stride and alignment -> rows of a multiple of 8 elements, 16-byte aligned, zeros behind the width
__global__ void __launch_bounds__(256) pad_rows_kernel(const uint16_t* __restrict__ src, uint64_t src_ld, uint64_t rows, uint32_t cols, uint16_t* __restrict__ dst, uint32_t dst_ld) {
	const uint64_t n = rows * (dst_ld / 8);
	for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (uint64_t)gridDim.x * 256) {
		const uint64_t r = i / (dst_ld / 8);
		const uint32_t c = (uint32_t)(i % (dst_ld / 8)) * 8;
		uint32_t w[4];
#pragma unroll
		for (int e = 0; e < 4; ++e) {
			const uint32_t a = c + 2 * e < cols ? src[r * src_ld + c + 2 * e] : 0, b = c + 2 * e + 1 < cols ? src[r * src_ld + c + 2 * e + 1] : 0;
			w[e] = a | b << 16;
		}
		*(uint4*)(dst + r * dst_ld + c) = make_uint4(w[0], w[1], w[2], w[3]);
	}
}

__global__ void __launch_bounds__(256) zero_kernel(uint16_t* p, uint64_t n) {
	for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (uint64_t)gridDim.x * 256) p[i] = 0;
}

// ---- host ------------------------------------------------------------------------------------------------------------------------------

constexpr uint32_t MAX_WIDTH = 1u << 20;
constexpr uint64_t MAX_ROWS = 1ull << 31, MAX_DMA_LD = 1u << 21;   // a tile's 256 rows stay within the 2 GiB of a buffer descriptor

static inline uint64_t up8(uint64_t v) { return (v + 7) & ~7ull; }
static inline uint64_t up256(uint64_t v) { return (v + 255) & ~255ull; }
static inline uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

static int refuse(const char* what) { set_last_error(what, hipErrorInvalidValue); return -1; }

static int check_block(const NgpGatedFfn* b, const char* who) {
	char msg[256];
	const char* bad = nullptr;
	if (!b) bad = "no block description";
	else if (b->n_in < 1 || b->n_hidden < 1 || b->n_out < 1 || b->n_in > MAX_WIDTH || b->n_hidden > MAX_WIDTH || b->n_out > MAX_WIDTH) bad = "widths must be 1 .. 2^20";
	else if (b->dtype != NGP_DTYPE_F16 && b->dtype != NGP_DTYPE_BF16) bad = "dtype must be F16 or BF16";
	else if (b->activation != NGP_ACT_NONE && b->activation != NGP_ACT_RELU && b->activation != NGP_ACT_LOGISTIC && b->activation != NGP_ACT_SILU && b->activation != NGP_ACT_GELU) bad = "activation must be None, ReLU, Logistic, SiLU or GELU";
	if (!bad) return 0;
	snprintf(msg, sizeof(msg), "%s: %s", who, bad);
	return refuse(msg);
}

// The workspace in order; a null base gives the sizes alone.
struct Arena {
	char* base;
	uint64_t used = 0;
	void* take(uint64_t bytes) { void* p = base ? base + used : nullptr; used += up256(bytes); return p; }
};

struct Plan { bool big; uint32_t tiles_n, tiles_m, splits, k_split, partials; };

// Tile and splits of one product.  256 x 256 tiles need the least LDS and memory traffic per multiplication and win wherever they fill the 256 CUs; below that, 128 x 128 tiles
// (two workgroups a CU), and where even those are few and k is long, k is split until about 512 workgroups run, with at least 8 steps of 64 each.
static Plan plan_product(uint64_t n, uint64_t m, uint64_t k, uint32_t n_products) {
	Plan p;
	const uint64_t t256 = ceil_div(n, 256) * ceil_div(m, 256);
	p.big = t256 >= 192;
	const uint32_t t = p.big ? 256 : 128;
	p.tiles_n = (uint32_t)ceil_div(n, t); p.tiles_m = (uint32_t)ceil_div(m, t);
	const uint64_t tiles = (uint64_t)p.tiles_n * p.tiles_m;
	uint64_t splits = 1;
	if (!p.big && tiles < 256) splits = std::max<uint64_t>(1, std::min<uint64_t>(512 / (tiles * n_products), k / 512));
	p.k_split = (uint32_t)(ceil_div(ceil_div(k, 64), splits) * 64);
	p.splits = (uint32_t)std::max<uint64_t>(1, ceil_div(k, p.k_split));
	p.partials = p.splits > 1 ? p.splits * n_products : 0;
	return p;
}
// room for its splits, never less than any smaller batch of the same block takes: the splits' tiles are at most 512, and at most k / 512 for each tile and product
static uint64_t partial_room(uint64_t n, uint64_t m, uint64_t k, uint32_t n_products) {
	return k >= 1024 ? std::min<uint64_t>(512, ceil_div(n, 128) * ceil_div(m, 128) * n_products * (k / 512)) * (128 * 128 * 4) : 0;
}

struct Tensor { const void* p; uint64_t ld; uint64_t rows; uint32_t cols; };
static bool dma_ready(const Tensor& t) { return ((uintptr_t)t.p & 15) == 0 && t.ld % 8 == 0 && t.cols % 8 == 0 && t.ld <= MAX_DMA_LD; }

static uint32_t copy_grid(uint64_t n) { return (uint32_t)std::min<uint64_t>(ceil_div(n, 256), 4096); }

// ---- narrow blocks: which, and their launches

constexpr uint32_t NARROW_GROUPS = 512;   // of the backward pass: two to three workgroups a CU, and the fewer, the less there is to add at the end

static uint32_t narrow_forward_lds(const NgpGatedFfn& b) {   // 0: not narrow
	if (b.n_in > 128 || b.n_out > 128) return 0;
	const uint32_t kb = b.n_in <= 16 ? 1 : b.n_in <= 32 ? 2 : b.n_in <= 64 ? 4 : 8, ob = b.n_out <= 32 ? 1 : b.n_out <= 64 ? 2 : 4;
	const uint64_t bytes = ceil_div(b.n_hidden, 32) * (2 * kb + 2 * ob) * 1024;
	return bytes <= 128 * 1024 ? (uint32_t)bytes : 0;
}
static bool narrow_backward(const NgpGatedFfn& b) { return b.n_in <= 64 && b.n_out <= 64 && b.n_hidden <= 128; }
static uint64_t narrow_partial_bytes(const NgpGatedFfn& b, uint64_t rows) {
	const uint64_t db = ceil_div(b.n_in, 32), fb = b.n_hidden <= 32 ? 1 : b.n_hidden <= 64 ? 2 : 4, ob = ceil_div(b.n_out, 32);
	return std::min<uint64_t>(NARROW_GROUPS, ceil_div(rows, 64)) * (2 * fb * db + fb * ob) * 4096;
}

template <class T, int DB, int OB, bool VEC>
static void launch_narrow_forward(hipStream_t st, const NarrowArgs& a, uint32_t lds) {
	if (lds > 64 * 1024) (void)hipFuncSetAttribute((const void*)narrow_forward_kernel<T, DB, OB, VEC>, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
	const uint32_t per_cu = std::max(1u, std::min((uint32_t)narrow_waves(DB, OB, VEC), 160 * 1024 / lds));
	hipLaunchKernelGGL((narrow_forward_kernel<T, DB, OB, VEC>), dim3(std::min((a.rows + 127) / 128, 256 * per_cu)), dim3(256), lds, st, a);
}
template <class T, int DB, int OB> static void pick_narrow_forward(hipStream_t st, const NarrowArgs& a, uint32_t lds, bool vec) {
	if (vec) launch_narrow_forward<T, DB, OB, true>(st, a, lds);
	else launch_narrow_forward<T, DB, OB, false>(st, a, lds);
}
template <class T, int DB> static void pick_narrow_forward(hipStream_t st, const NarrowArgs& a, uint32_t lds, bool vec) {
	if (a.o <= 32) pick_narrow_forward<T, DB, 1>(st, a, lds, vec);
	else if (a.o <= 64) pick_narrow_forward<T, DB, 2>(st, a, lds, vec);
	else pick_narrow_forward<T, DB, 4>(st, a, lds, vec);
}
template <class T> static int run_narrow_forward(hipStream_t st, const NarrowArgs& a, uint32_t lds, bool vec) {
	if (a.d <= 16) pick_narrow_forward<T, 1>(st, a, lds, vec);
	else if (a.d <= 32) pick_narrow_forward<T, 2>(st, a, lds, vec);
	else if (a.d <= 64) pick_narrow_forward<T, 4>(st, a, lds, vec);
	else pick_narrow_forward<T, 8>(st, a, lds, vec);
	NGP_LAUNCH_CHECK("narrow_forward_kernel");
	return 0;
}

template <class T, int DB, int FB, int OB> static void launch_narrow_backward(hipStream_t st, const NarrowArgs& a, bool vec, void* dwg, void* dwu, void* dwd) {
	const uint32_t groups = std::min<uint32_t>(NARROW_GROUPS, (a.rows + 63) / 64);
	if (vec) hipLaunchKernelGGL((narrow_backward_kernel<T, DB, FB, OB, true>), dim3(groups), dim3(256), 0, st, a);
	else hipLaunchKernelGGL((narrow_backward_kernel<T, DB, FB, OB, false>), dim3(groups), dim3(256), 0, st, a);
	constexpr uint32_t blocks = NarrowBackward<DB, FB, OB>::BLOCKS;
	if (a.partial) hipLaunchKernelGGL((narrow_sum_kernel<T>), dim3(blocks * 16), dim3(1024), 0, st, (const float*)a.partial, groups, blocks, (uint32_t)DB, (uint32_t)FB, (uint32_t)OB, a.d, a.f, a.o, (T*)dwg, (T*)dwu, (T*)dwd);
}
template <class T, int DB, int OB> static void pick_narrow_backward(hipStream_t st, const NarrowArgs& a, bool vec, void* dwg, void* dwu, void* dwd) {
	if (a.f <= 32) launch_narrow_backward<T, DB, 1, OB>(st, a, vec, dwg, dwu, dwd);
	else if (a.f <= 64) launch_narrow_backward<T, DB, 2, OB>(st, a, vec, dwg, dwu, dwd);
	else launch_narrow_backward<T, DB, 4, OB>(st, a, vec, dwg, dwu, dwd);
}
template <class T> static int run_narrow_backward(hipStream_t st, const NarrowArgs& a, bool vec, void* dwg, void* dwu, void* dwd) {
	if (a.d <= 32) { if (a.o <= 32) pick_narrow_backward<T, 1, 1>(st, a, vec, dwg, dwu, dwd); else pick_narrow_backward<T, 1, 2>(st, a, vec, dwg, dwu, dwd); }
	else { if (a.o <= 32) pick_narrow_backward<T, 2, 1>(st, a, vec, dwg, dwu, dwd); else pick_narrow_backward<T, 2, 2>(st, a, vec, dwg, dwu, dwd); }
	NGP_LAUNCH_CHECK("narrow_backward_kernel");
	return 0;
}
// ---- few rows: a launch for h and one for y.  Workgroups of 4 to 16 waves (8 for the pair of matrices, whose sums take twice the LDS): about 2048 waves, 8 a CU.
template <class T, int NM, int MB> static void launch_few(hipStream_t st, const T* x, uint64_t x_ld, uint32_t rows, const T* w0, const T* w1, uint32_t n, uint32_t k, T* out, uint64_t out_ld, int act) {
	const uint32_t groups = (n + 15) / 16;
	uint32_t waves = 4;
	while (waves < (NM == 2 ? 8 : 16) && groups * waves < 2048 && waves * (FEW_CHUNK * 32) < k) waves *= 2;
	hipLaunchKernelGGL((few_rows_kernel<T, NM, MB>), dim3(groups), dim3(64 * waves), 0, st, x, x_ld, rows, w0, w1, n, k, out, out_ld, act);
}
template <class T, int NM> static void pick_few(hipStream_t st, const T* x, uint64_t x_ld, uint32_t rows, const T* w0, const T* w1, uint32_t n, uint32_t k, T* out, uint64_t out_ld, int act) {
	if (rows <= 16) launch_few<T, NM, 1>(st, x, x_ld, rows, w0, w1, n, k, out, out_ld, act);
	else if (rows <= 32) launch_few<T, NM, 2>(st, x, x_ld, rows, w0, w1, n, k, out, out_ld, act);
	else launch_few<T, NM, 4>(st, x, x_ld, rows, w0, w1, n, k, out, out_ld, act);
}
template <class T> static int run_few(hipStream_t st, const NgpGatedFfn& b, uint32_t rows, const void* x, uint64_t x_ld, const void* wg, const void* wu, const void* wd, void* y, uint64_t y_ld, void* h) {
	const uint32_t pitch = (b.n_hidden + 31) & ~31u;
	pick_few<T, 2>(st, (const T*)x, x_ld, rows, (const T*)wg, (const T*)wu, b.n_hidden, b.n_in, (T*)h, pitch, b.activation);
	pick_few<T, 1>(st, (const T*)h, pitch, rows, (const T*)wd, nullptr, b.n_out, b.n_hidden, (T*)y, y_ld, 0);
	NGP_LAUNCH_CHECK("few_rows_kernel");
	return 0;
}

static bool vector_rows(const void* p, uint64_t ld, uint32_t cols) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && cols % 8 == 0; }

// What a call keeps in its workspace.  `any`: room for padded copies of every input, else of those whose width is no multiple of 8.
struct Space {
	uint32_t d8, f8, o8, fp;                                   // widths as the copies have them; fp: row pitch of h, dg and du
	void *x = nullptr, *wg = nullptr, *wu = nullptr, *wd = nullptr, *dy = nullptr, *h = nullptr, *d = nullptr;
	float* partial = nullptr;
	Plan y, dx, dwgu, dwd;
	uint64_t bytes;
	bool has_copies(uint32_t width, bool any) const { return any || width % 8; }
	Space(char* base, const NgpGatedFfn& b, uint64_t rows, bool backward, bool any) {
		Arena a{base};
		bytes = 0;
		d8 = (uint32_t)up8(b.n_in); f8 = (uint32_t)up8(b.n_hidden); o8 = (uint32_t)up8(b.n_out); fp = (f8 + 31) & ~31u;
		if (backward ? narrow_backward(b) : narrow_forward_lds(b) != 0) {
			if (backward) partial = (float*)a.take(narrow_partial_bytes(b, rows));
			bytes = a.used;
			return;
		}
		if (!backward && rows <= FEW_ROWS) {
			h = a.take(rows * fp * 2);
			bytes = a.used;
			return;
		}
		if (has_copies(b.n_in, any)) { x = a.take(rows * d8 * 2); wg = a.take((uint64_t)b.n_hidden * d8 * 2); wu = a.take((uint64_t)b.n_hidden * d8 * 2); }
		if (has_copies(b.n_hidden, any)) wd = a.take((uint64_t)b.n_out * f8 * 2);
		if (backward && has_copies(b.n_out, any)) dy = a.take(rows * o8 * 2);
		h = a.take(rows * fp * 2);
		uint64_t part = 0;
		if (backward) {
			d = a.take(rows * fp * 4);
			dx = plan_product(b.n_in, rows, b.n_hidden, 2);
			dwgu = plan_product(b.n_in, 2 * (uint64_t)fp, rows, 1);
			dwd = plan_product(b.n_hidden, b.n_out, rows, 1);
			part = std::max(partial_room(b.n_in, rows, b.n_hidden, 2), std::max(partial_room(b.n_in, 2 * (uint64_t)fp, rows, 1), partial_room(b.n_hidden, b.n_out, rows, 1)));
		} else {
			y = plan_product(b.n_out, rows, f8, 1);
			part = partial_room(b.n_out, rows, f8, 1);
		}
		partial = (float*)a.take(part);   // one after the other on one stream: they share it
		bytes = a.used;
	}
};

struct Launch {
	hipStream_t st;
	int rc = 0;
	bool ok(const char* what) {
		if (rc) return false;
		const hipError_t e = hipGetLastError();
		if (e != hipSuccess) { set_last_error(what, e); rc = (int)e; }
		return rc == 0;
	}
	// `t` as the DMA takes it, through `copy` where it is not ready (copy null: not reserved)
	Tensor ready(const Tensor& t, void* copy, uint32_t width8) {
		if (rc || dma_ready(t)) return t;
		if (!copy) { rc = refuse("ngp_hip_gated_ffn: a row that is not 16-byte aligned needs the workspace of NGP_FFN_ANY_LAYOUT"); return t; }
		hipLaunchKernelGGL(pad_rows_kernel, dim3(copy_grid(t.rows * (width8 / 8))), dim3(256), 0, st, (const uint16_t*)t.p, t.ld, t.rows, t.cols, (uint16_t*)copy, width8);
		ok("pad_rows_kernel");
		return Tensor{copy, width8, t.rows, width8};
	}
	template <class T, int NLAY, int MLAY> void product(const Plan& p, const Pair& p0, const Pair* p1, const Rows2<T>& out, float* partial) {
		if (rc) return;
		const uint32_t tiles = p.tiles_n * p.tiles_m;
		float* part = p.partials ? partial : nullptr;
		const dim3 grid(tiles * std::max(1u, p.partials));
		if (p.big) hipLaunchKernelGGL((product_kernel<T, NLAY, MLAY, true>), grid, dim3(Shape<true>::THREADS), 0, st, p0, p1 ? *p1 : p0, p1 ? 2 : 1, out, p.tiles_n, p.tiles_m, p.splits, p.k_split, part);
		else hipLaunchKernelGGL((product_kernel<T, NLAY, MLAY, false>), grid, dim3(256), 0, st, p0, p1 ? *p1 : p0, p1 ? 2 : 1, out, p.tiles_n, p.tiles_m, p.splits, p.k_split, part);
		if (!ok("product_kernel") || !part) return;
		uint32_t splits = p.partials, every = 1;
		if (splits > SUM_FAN) {
			const uint64_t floats = (uint64_t)tiles * 128 * 128;
			hipLaunchKernelGGL(split_fold_kernel, dim3((uint32_t)(floats / 1024 * ceil_div(splits, SUM_FAN))), dim3(256), 0, st, part, splits, floats);
			splits = (uint32_t)ceil_div(splits, SUM_FAN);
			every = SUM_FAN;
		}
		hipLaunchKernelGGL((split_sum_kernel<T, false>), dim3(tiles), dim3(256), 0, st, (const float*)part, splits, every, out, p.tiles_n, p.tiles_m);
		ok("split_sum_kernel");
	}
};

static Mat kc(const Tensor& t) { return Mat{t.p, t.ld, (uint32_t)t.rows, t.cols}; }            // rows of the tensor = rows of the operand
static Mat rc(const Tensor& t) { return Mat{t.p, t.ld, t.cols, (uint32_t)t.rows}; }            // rows of the tensor = k
template <class T> static Rows2<T> whole(void* p, uint64_t ld, uint64_t rows, uint32_t cols) { const Out<T> o{(T*)p, ld, (uint32_t)rows, cols}; return Rows2<T>{o, o, 0xffffffffu}; }

template <class T>
static int forward(hipStream_t st, const NgpGatedFfn& b, const Space& s, Tensor x, Tensor wg, Tensor wu, Tensor wd, void* y, uint64_t y_ld) {
	Launch l{st};
	x = l.ready(x, s.x, s.d8); wg = l.ready(wg, s.wg, s.d8); wu = l.ready(wu, s.wu, s.d8); wd = l.ready(wd, s.wd, s.f8);
	if (l.rc) return l.rc;
	const Out<T> h{(T*)s.h, s.fp, (uint32_t)x.rows, s.fp};
	const bool big = ceil_div(s.fp, 128) * ceil_div(x.rows, 256) >= 192;
	const uint32_t tn = (uint32_t)ceil_div(s.fp, big ? 128 : 64), tm = (uint32_t)ceil_div(x.rows, big ? 256 : 128);
	if (big) hipLaunchKernelGGL((gate_up_kernel<T, true>), dim3(tn * tm), dim3(Shape<true>::THREADS), 0, st, kc(x), kc(wg), kc(wu), h, b.activation, tn, tm);
	else hipLaunchKernelGGL((gate_up_kernel<T, false>), dim3(tn * tm), dim3(256), 0, st, kc(x), kc(wg), kc(wu), h, b.activation, tn, tm);
	l.ok("gate_up_kernel");
	const Tensor th{s.h, s.fp, x.rows, s.f8};
	l.product<T, KC, KC>(s.y, Pair{kc(wd), kc(th)}, nullptr, whole<T>(y, y_ld, x.rows, b.n_out), s.partial);
	return l.rc;
}

template <class T>
static int backward(hipStream_t st, const NgpGatedFfn& b, const Space& s, Tensor x, Tensor wg, Tensor wu, Tensor wd, Tensor dy, void* dx, uint64_t dx_ld, void* dwg, void* dwu, void* dwd) {
	Launch l{st};
	x = l.ready(x, s.x, s.d8); wg = l.ready(wg, s.wg, s.d8); wu = l.ready(wu, s.wu, s.d8); wd = l.ready(wd, s.wd, s.f8); dy = l.ready(dy, s.dy, s.o8);
	if (l.rc) return l.rc;
	const uint32_t rows = (uint32_t)x.rows;
	T* const d = (T*)s.d;
	const Out<T> h{(T*)s.h, s.fp, rows, s.fp}, dg{d, 2ull * s.fp, rows, s.fp}, du{d + s.fp, 2ull * s.fp, rows, s.fp};
	const bool big = ceil_div(s.fp, 128) * ceil_div(rows, 256) >= 192;
	const uint32_t tn = (uint32_t)ceil_div(s.fp, big ? 128 : 64), tm = (uint32_t)ceil_div(rows, big ? 256 : 128);
	if (big) hipLaunchKernelGGL((hidden_backward_kernel<T, true>), dim3(tn * tm), dim3(Shape<true>::THREADS), 0, st, kc(x), kc(wg), kc(wu), kc(dy), rc(wd), dg, du, h, b.activation, tn, tm);
	else hipLaunchKernelGGL((hidden_backward_kernel<T, false>), dim3(tn * tm), dim3(256), 0, st, kc(x), kc(wg), kc(wu), kc(dy), rc(wd), dg, du, h, b.activation, tn, tm);
	l.ok("hidden_backward_kernel");
	const Tensor tdg{dg.p, dg.ld, rows, s.f8}, tdu{du.p, du.ld, rows, s.f8}, tboth{d, 2ull * s.fp, rows, 2 * s.fp}, th{s.h, s.fp, rows, s.fp};
	if (dx) {
		const Pair up{rc(wu), kc(tdu)};
		l.product<T, RC, KC>(s.dx, Pair{rc(wg), kc(tdg)}, &up, whole<T>(dx, dx_ld, rows, b.n_in), s.partial);
	}
	if (dwg) {
		const Rows2<T> out{Out<T>{(T*)dwg, b.n_in, b.n_hidden, b.n_in}, Out<T>{(T*)dwu, b.n_in, b.n_hidden, b.n_in}, s.fp};
		l.product<T, RC, RC>(s.dwgu, Pair{rc(x), rc(tboth)}, nullptr, out, s.partial);
		l.product<T, RC, RC>(s.dwd, Pair{rc(th), rc(dy)}, nullptr, whole<T>(dwd, b.n_hidden, b.n_out, b.n_hidden), s.partial);
	}
	return l.rc;
}

} // namespace ffn
} // namespace ngp

using namespace ngp;

extern "C" {

uint64_t ngp_hip_gated_ffn_workspace_bytes(const NgpGatedFfn* block_host, uint64_t n_rows, uint32_t flags) {
	if (ffn::check_block(block_host, "ngp_hip_gated_ffn_workspace_bytes")) return 0;
	return n_rows == 0 || n_rows > ffn::MAX_ROWS ? 0 : ffn::Space(nullptr, *block_host, n_rows, flags & NGP_FFN_BACKWARD, flags & NGP_FFN_ANY_LAYOUT).bytes;
}

int ngp_hip_gated_ffn_forward(void* stream, const NgpGatedFfn* b, uint64_t n_rows, const void* x, uint64_t x_stride, const void* w_gate, const void* w_up, const void* w_down,
                              void* y, uint64_t y_stride, void* workspace, uint64_t workspace_bytes) {
	using namespace ffn;
	if (check_block(b, "ngp_hip_gated_ffn_forward")) return -1;
	if (n_rows > MAX_ROWS) return refuse("ngp_hip_gated_ffn_forward: more than 2^31 rows");
	if (n_rows == 0) return 0;
	if (!x || !w_gate || !w_up || !w_down || !y) return refuse("ngp_hip_gated_ffn_forward: null tensor");
	if (x_stride < b->n_in || y_stride < b->n_out) return refuse("ngp_hip_gated_ffn_forward: a row stride is smaller than its row");
	if (((uintptr_t)x | (uintptr_t)w_gate | (uintptr_t)w_up | (uintptr_t)w_down | (uintptr_t)y) & 1) return refuse("ngp_hip_gated_ffn_forward: a tensor is not aligned to its elements");
	const Tensor tx{x, x_stride, n_rows, b->n_in}, tg{w_gate, b->n_in, b->n_hidden, b->n_in}, tu{w_up, b->n_in, b->n_hidden, b->n_in}, td{w_down, b->n_hidden, b->n_out, b->n_hidden};
	if (const uint32_t lds = narrow_forward_lds(*b)) {
		const NarrowArgs a{x, w_gate, w_up, w_down, nullptr, y, nullptr, x_stride, y_stride, 0, 0, (uint32_t)n_rows, b->n_in, b->n_hidden, b->n_out, b->activation, nullptr};
		const bool vec = vector_rows(x, x_stride, b->n_in);
		return b->dtype == NGP_DTYPE_F16 ? run_narrow_forward<f16>((hipStream_t)stream, a, lds, vec) : run_narrow_forward<b16>((hipStream_t)stream, a, lds, vec);
	}
	const bool plain = (b->n_in % 8 || (dma_ready(tx) && dma_ready(tg) && dma_ready(tu))) && (b->n_hidden % 8 || dma_ready(td));
	const Space s((char*)workspace, *b, n_rows, false, !plain);
	if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < s.bytes) return refuse("ngp_hip_gated_ffn_forward: workspace null, not 16-byte aligned or too small (ngp_hip_gated_ffn_workspace_bytes; rows that are not 16-byte aligned: NGP_FFN_ANY_LAYOUT)");
	if (n_rows <= FEW_ROWS) return b->dtype == NGP_DTYPE_F16 ? run_few<f16>((hipStream_t)stream, *b, (uint32_t)n_rows, x, x_stride, w_gate, w_up, w_down, y, y_stride, s.h)
	                                                         : run_few<b16>((hipStream_t)stream, *b, (uint32_t)n_rows, x, x_stride, w_gate, w_up, w_down, y, y_stride, s.h);
	if (b->dtype == NGP_DTYPE_F16) return forward<f16>((hipStream_t)stream, *b, s, tx, tg, tu, td, y, y_stride);
	return forward<b16>((hipStream_t)stream, *b, s, tx, tg, tu, td, y, y_stride);
}

int ngp_hip_gated_ffn_backward(void* stream, const NgpGatedFfn* b, uint64_t n_rows, const void* x, uint64_t x_stride, const void* w_gate, const void* w_up, const void* w_down,
                               const void* dy, uint64_t dy_stride, void* dx, uint64_t dx_stride, void* dw_gate, void* dw_up, void* dw_down, void* workspace, uint64_t workspace_bytes) {
	using namespace ffn;
	if (check_block(b, "ngp_hip_gated_ffn_backward")) return -1;
	if (n_rows > MAX_ROWS) return refuse("ngp_hip_gated_ffn_backward: more than 2^31 rows");
	if ((dw_gate == nullptr) != (dw_up == nullptr) || (dw_gate == nullptr) != (dw_down == nullptr)) return refuse("ngp_hip_gated_ffn_backward: the three weight gradients go together");
	if (!dx && !dw_gate) return refuse("ngp_hip_gated_ffn_backward: nothing to compute");
	if (((uintptr_t)dw_gate | (uintptr_t)dw_up | (uintptr_t)dw_down | (uintptr_t)dx) & 1) return refuse("ngp_hip_gated_ffn_backward: a tensor is not aligned to its elements");
	hipStream_t st = (hipStream_t)stream;
	if (n_rows == 0) {   // the gradient of an empty batch
		if (!dw_gate) return 0;
		const uint64_t n = (uint64_t)b->n_hidden * b->n_in, m = (uint64_t)b->n_out * b->n_hidden;
		hipLaunchKernelGGL(zero_kernel, dim3(copy_grid(n)), dim3(256), 0, st, (uint16_t*)dw_gate, n);
		hipLaunchKernelGGL(zero_kernel, dim3(copy_grid(n)), dim3(256), 0, st, (uint16_t*)dw_up, n);
		hipLaunchKernelGGL(zero_kernel, dim3(copy_grid(m)), dim3(256), 0, st, (uint16_t*)dw_down, m);
		NGP_LAUNCH_CHECK("zero_kernel");
		return 0;
	}
	if (!x || !w_gate || !w_up || !w_down || !dy) return refuse("ngp_hip_gated_ffn_backward: null tensor");
	if (x_stride < b->n_in || dy_stride < b->n_out || (dx && dx_stride < b->n_in)) return refuse("ngp_hip_gated_ffn_backward: a row stride is smaller than its row");
	if (((uintptr_t)x | (uintptr_t)w_gate | (uintptr_t)w_up | (uintptr_t)w_down | (uintptr_t)dy) & 1) return refuse("ngp_hip_gated_ffn_backward: a tensor is not aligned to its elements");
	const Tensor tx{x, x_stride, n_rows, b->n_in}, tg{w_gate, b->n_in, b->n_hidden, b->n_in}, tu{w_up, b->n_in, b->n_hidden, b->n_in}, td{w_down, b->n_hidden, b->n_out, b->n_hidden}, ty{dy, dy_stride, n_rows, b->n_out};
	if (narrow_backward(*b)) {
		const uint64_t need = dw_gate ? narrow_partial_bytes(*b, n_rows) : 0;
		if (need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)) return refuse("ngp_hip_gated_ffn_backward: workspace null, not 16-byte aligned or too small (ngp_hip_gated_ffn_workspace_bytes)");
		const NarrowArgs a{x, w_gate, w_up, w_down, dy, nullptr, dx, x_stride, 0, dy_stride, dx_stride, (uint32_t)n_rows, b->n_in, b->n_hidden, b->n_out, b->activation, need ? (float*)workspace : nullptr};
		const bool vec = vector_rows(x, x_stride, b->n_in) && vector_rows(dy, dy_stride, b->n_out);
		return b->dtype == NGP_DTYPE_F16 ? run_narrow_backward<f16>(st, a, vec, dw_gate, dw_up, dw_down) : run_narrow_backward<b16>(st, a, vec, dw_gate, dw_up, dw_down);
	}
	const bool plain = (b->n_in % 8 || (dma_ready(tx) && dma_ready(tg) && dma_ready(tu))) && (b->n_hidden % 8 || dma_ready(td)) && (b->n_out % 8 || dma_ready(ty));
	const Space s((char*)workspace, *b, n_rows, true, !plain);
	if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < s.bytes) return refuse("ngp_hip_gated_ffn_backward: workspace null, not 16-byte aligned or too small (ngp_hip_gated_ffn_workspace_bytes; rows that are not 16-byte aligned: NGP_FFN_ANY_LAYOUT)");
	if (b->dtype == NGP_DTYPE_F16) return backward<f16>(st, *b, s, tx, tg, tu, td, ty, dx, dx_stride, dw_gate, dw_up, dw_down);
	return backward<b16>(st, *b, s, tx, tg, tu, td, ty, dx, dx_stride, dw_gate, dw_up, dw_down);
}

} // extern "C"
