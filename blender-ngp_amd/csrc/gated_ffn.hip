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
	if (ACT == NGP_ACT_GELU) {
		// g Phi(g).  Phi(-a) = e^(-a^2/2) R(a) for a >= 0, R smooth: t P(t), t = 1 / (1 + 0.325 a), P the polynomial of degree 7 with the least relative error, 6.8e-7 (with the
		// roundings here Phi(-a) is within 2e-6 of itself up to a = 6: its small tail keeps its digits).  One exponential serves the value and the derivative; with erfcf the
		// backward pass of 4096 x 1024 - 2816 - 1024 took 222 us, SiLU's 202.
		const float e = __expf(-0.5f * g * g), t = __builtin_amdgcn_rcpf(1.0f + 0.325f * fabsf(g));
		float p = 0.0338170901f;
		p = fmaf(p, t, -0.113520846f); p = fmaf(p, t, 0.0853101463f); p = fmaf(p, t, 0.0260451920f); p = fmaf(p, t, 0.0935166031f);
		p = fmaf(p, t, 0.115503825f); p = fmaf(p, t, 0.129672095f); p = fmaf(p, t, 0.129656151f);
		const float tail = p * t * e, phi = g < 0.0f ? tail : 1.0f - tail;
		return make_float2(g * phi, fmaf(g * 0.39894228f, e, phi));
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

enum { SMALL, BIG, HALF };
template <int SHAPE> struct Shape;   // BIG: 256 x 256 in 8 waves, one workgroup a CU; HALF: 256 x 128 in 8 waves; SMALL: 128 x 128 in 4 waves, two a CU
template <> struct Shape<BIG> { static constexpr int N = 256, M = 256, WN = 2, WM = 4, THREADS = 512, RESIDENT = 2; };
template <> struct Shape<HALF> { static constexpr int N = 256, M = 128, WN = 4, WM = 2, THREADS = 512, RESIDENT = 2; };
template <> struct Shape<SMALL> { static constexpr int N = 128, M = 128, WN = 2, WM = 2, THREADS = 256, RESIDENT = 2; };

template <int NM, int NB, int MB> __device__ __forceinline__ void clear(f32x4 (&acc)[NM][NB][MB]) {
#pragma unroll
	for (int j = 0; j < NM; ++j)
#pragma unroll
		for (int a = 0; a < NB; ++a)
#pragma unroll
			for (int b = 0; b < MB; ++b) acc[j][a][b] = f32x4{0, 0, 0, 0};
}

// h = act(x Wg^T) * (x Wu^T): one tile of rows of x against N / 2 gate rows and the same N / 2 up rows, so that both factors of an h meet in one lane and one tile of x serves both.
// Bound by the matrix pipes: 8192 x 4096 - 8192 in bf16 0.86 ms, 1.28 PFLOP/s.
template <class T, int SHAPE> struct HiddenProducts {
	using S = Shape<SHAPE>;
	using P = Product<T, KC, KC, 2, S::N / 2, S::M, S::WN, S::WM>;
	using Q = Product<T, RC, KC, 1, S::N / 2, S::M, S::WN, S::WM>;
	static_assert(Q::LDS_BYTES <= P::LDS_BYTES, "one buffer for both");
};
template <class T, int SHAPE>
__device__ __forceinline__ void gate_up_tile(const Mat& x, const Mat& wg, const Mat& wu, const Out<T>& h, int act, uint32_t n0, uint32_t m0, lds_char* lds) {
	using S = Shape<SHAPE>;
	using P = typename HiddenProducts<T, SHAPE>::P;
	f32x4 acc[2][P::NB][P::MB];
	clear(acc);
	const Mat w[2] = {wg, wu};
	P::run(acc, w, x, n0, m0, 0, x.k, lds);
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % S::WN, wm = wave / S::WN;
	lds_char* mine = lds + wave * Rows<P::NB>::BYTES;
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

// The tiles of a launch over all of h: rows of BIG tiles and, behind them, rows of tiles half as high, where those spare most of a round of the chip (cover_of)
struct Cover { uint32_t tiles_n, tiles_m, half_first, half_tiles_m; };   // half_first: the first workgroup with a half tile, a multiple of 8
// f(Constant<shape>, n0, m0) for this workgroup's tile
template <int SHAPE, bool HALVES, class F>
__device__ __forceinline__ void with_tile(const Cover& c, F f) {
	uint32_t tn, tm, split;
	if (!HALVES || blockIdx.x < c.half_first) {
		if (HALVES && blockIdx.x >= c.tiles_n * c.tiles_m) return;
		tile_of(blockIdx.x, c.tiles_n * c.tiles_m, c.tiles_n, c.tiles_m, tn, tm, split);
		f(Constant<SHAPE>(), tn * (Shape<SHAPE>::N / 2), tm * Shape<SHAPE>::M);
	} else {
		tile_of(blockIdx.x - c.half_first, c.tiles_n * c.half_tiles_m, c.tiles_n, c.half_tiles_m, tn, tm, split);
		f(Constant<HALF>(), tn * (Shape<HALF>::N / 2), c.tiles_m * Shape<BIG>::M + tm * Shape<HALF>::M);
	}
}
template <class T, int SHAPE, bool HALVES>
__global__ void __launch_bounds__(Shape<SHAPE>::THREADS, Shape<SHAPE>::RESIDENT) gate_up_kernel(Mat x, Mat wg, Mat wu, Out<T> h, int act, Cover cover) {
	__shared__ __attribute__((aligned(1024))) char lds[HiddenProducts<T, SHAPE>::P::LDS_BYTES];
	with_tile<SHAPE, HALVES>(cover, [&](auto shape, uint32_t n0, uint32_t m0) { gate_up_tile<T, decltype(shape)::value>(x, wg, wu, h, act, n0, m0, lds_of(lds)); });
}

struct Pair { Mat n, m; };                        // one product's operands
template <class T> struct Rows2 { Out<T> a, b; uint32_t a_rows; };   // rows 0 .. a_rows - 1 of the result go to a, the rest to b (b starts at row a_rows)

// One result: the sum of up to two products of the same k (dx = dg Wg + du Wu), each in `splits` parts of k_split.  partials: splits over all products, 0: none, straight to `out`.
template <class T> struct Item {
	Pair p[2];
	Rows2<T> out;
	float* partial;
	uint32_t n_products, tiles_n, tiles_m, splits, k_split, partials, turned;   // turned: the M side has k as its rows too
	uint32_t first, count;   // workgroups; first is a multiple of 8, so that a workgroup's number within the item still says which XCD it runs on
};
template <class T> struct Group { Item<T> item[3]; uint32_t n; };

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

template <class T, int NLAY, int MLAY, int SHAPE>
__device__ __forceinline__ void one_tile(const Item<T>& it, uint32_t pid, lds_char* lds) {
	using S = Shape<SHAPE>;
	using P = Product<T, NLAY, MLAY, 1, S::N, S::M, S::WN, S::WM>;
	uint32_t tn, tm, split;
	tile_of(pid, it.count, it.tiles_n, it.tiles_m, tn, tm, split);
	f32x4 acc[1][P::NB][P::MB];
	clear(acc);
	const uint32_t n0 = tn * S::N, m0 = tm * S::M;
	const bool parts = it.partials != 0;   // part `split % splits` of product `split / splits`
	const uint32_t from = parts ? split / it.splits : 0, to = parts ? from + 1 : it.n_products;
	for (uint32_t q = from; q < to; ++q) {
		const Pair& p = it.p[q];
		const uint32_t k0 = parts ? split % it.splits * it.k_split : 0;
		P::run(acc, &p.n, p.m, n0, m0, k0, p.n.k - k0 < it.k_split ? p.n.k : k0 + it.k_split, lds);
	}
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % S::WN, wm = wave / S::WN;
	if (parts) {
		float* q = it.partial + ((uint64_t)split * it.tiles_n * it.tiles_m + (uint64_t)tm * it.tiles_n + tn) * (S::N * S::M) + threadIdx.x * 4;
#pragma unroll
		for (int b = 0; b < P::NB; ++b)
#pragma unroll
			for (int c = 0; c < P::MB; ++c) *(f32x4*)(q + (b * P::MB + c) * (S::THREADS * 4)) = acc[0][b][c];
		return;
	}
	store_tile<T, P::NB, P::MB>(acc, it.out, n0 + wn * (P::NB * 16), m0 + wm * (P::MB * 16), lds + wave * Rows<P::NB>::BYTES, lane);
}

// All results that are ready to be computed at one point in one launch: y (FORWARD), or dx and the three weight gradients, whose tiles fill the chip together where each alone would
// leave a part of it idle.  Bound by the matrix pipes: the five products behind 8192 x 4096 - 8192 - 4096 in f16 2.06 ms, 1.33 PFLOP/s; those of 4096 x 1024 - 2816 - 1024 125 us,
// 0.97 (196 tiles for 256 CUs, a third of them with 5632 of k to the others' 4096).  With splits, a workgroup leaves its accumulators in `partial` as they lie in the registers, and group_sum_kernel adds the splits in their order: the
// result does not depend on which workgroup ends first.
template <class T, int SHAPE, bool FORWARD>
__global__ void __launch_bounds__(Shape<SHAPE>::THREADS, Shape<SHAPE>::RESIDENT) group_kernel(Group<T> g) {
	using S = Shape<SHAPE>;
	__shared__ __attribute__((aligned(1024))) char lds[Product<T, KC, KC, 1, S::N, S::M, S::WN, S::WM>::LDS_BYTES];
	uint32_t i = 0;
	while (i + 1 < g.n && blockIdx.x >= g.item[i + 1].first) ++i;
	const Item<T>& it = g.item[i];
	const uint32_t pid = blockIdx.x - it.first;
	if (pid >= it.count) return;
	if (FORWARD) one_tile<T, KC, KC, SHAPE>(it, pid, lds_of(lds));
	else if (it.turned) one_tile<T, RC, RC, SHAPE>(it, pid, lds_of(lds));
	else one_tile<T, RC, KC, SHAPE>(it, pid, lds_of(lds));
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

// The splits of the tiles (every `every`-th of them, where they have been folded), added in order, rounded once; a workgroup takes two of a tile's MB block rows, the 32 rows that
// are stored together.  Items without splits have no tiles here.  Bound by memory and by starting up: 32 MB of sums 11 us, 5 MB 5 us.
template <class T>
__global__ void __launch_bounds__(256) group_sum_kernel(Group<T> g) {
	using S = Shape<SMALL>;
	constexpr int NB = S::N / S::WN / 16, MB = S::M / S::WM / 16;
	__shared__ __attribute__((aligned(16))) char lds[S::WN * S::WM * Rows<NB>::BYTES];
	const uint32_t pid = blockIdx.x / (MB / 2), c0 = blockIdx.x % (MB / 2) * 2;
	uint32_t i = 0;
	while (i + 1 < g.n && pid >= g.item[i + 1].first) ++i;
	const Item<T>& it = g.item[i];
	const uint32_t t = pid - it.first, tiles = it.tiles_n * it.tiles_m, tn = t % it.tiles_n, tm = t / it.tiles_n;
	const uint32_t every = it.partials > SUM_FAN ? SUM_FAN : 1, splits = (it.partials + every - 1) / every;
	const float* q = it.partial + (uint64_t)t * (S::N * S::M) + c0 * (S::THREADS * 4) + threadIdx.x * 4;
	const uint64_t stride = (uint64_t)every * tiles * (S::N * S::M);
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % S::WN, wm = wave / S::WN;
	f32x4 acc[1][NB][2];
	clear(acc);
#pragma unroll 4
	for (uint32_t s = 0; s < splits; ++s)
#pragma unroll
		for (int b = 0; b < NB; ++b)
#pragma unroll
			for (int c = 0; c < 2; ++c) acc[0][b][c] += *(const f32x4*)(q + s * stride + (b * MB + c) * (S::THREADS * 4));
	store_tile<T, NB, 2>(acc, it.out, tn * S::N + wn * (NB * 16), tm * S::M + wm * (MB * 16) + c0 * 16, lds_of(lds) + wave * Rows<NB>::BYTES, lane);
}
constexpr uint32_t SUM_GROUPS = Shape<SMALL>::M / Shape<SMALL>::WM / 16 / 2;   // workgroups to a tile

// g, u and dh of a tile in one set of registers; from them dg, du (next to each other: d[m][0 .. f8) and d[m][f8 .. 2 f8)) and h.  Three products for three results and nothing else
// read twice.  Bound by the matrix pipes: 8192 x 4096 - 8192 - 4096 in f16 1.48 ms, 1.11 PFLOP/s.
template <class T, int SHAPE>
__device__ __forceinline__ void hidden_backward_tile(const Mat& x, const Mat& wg, const Mat& wu, const Mat& dy, const Mat& wd, const Out<T>& dg, const Out<T>& du, const Out<T>& h, int act, uint32_t n0, uint32_t m0,
                                                     lds_char* lds) {
	using S = Shape<SHAPE>;
	using P = typename HiddenProducts<T, SHAPE>::P;
	using Q = typename HiddenProducts<T, SHAPE>::Q;
	f32x4 gu[2][P::NB][P::MB], dh[1][P::NB][P::MB];
	clear(gu);
	const Mat w[2] = {wg, wu};
	P::run(gu, w, x, n0, m0, 0, x.k, lds);
	clear(dh);
	Q::run(dh, &wd, dy, n0, m0, 0, dy.k, lds);
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % S::WN, wm = wave / S::WN;
	lds_char* mine = lds + wave * (3 * Rows<P::NB>::BYTES);
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

template <class T, int SHAPE, bool HALVES>
__global__ void __launch_bounds__(Shape<SHAPE>::THREADS, Shape<SHAPE>::RESIDENT) hidden_backward_kernel(Mat x, Mat wg, Mat wu, Mat dy, Mat wd, Out<T> dg, Out<T> du, Out<T> h, int act, Cover cover) {
	__shared__ __attribute__((aligned(1024))) char lds[HiddenProducts<T, SHAPE>::P::LDS_BYTES];
	with_tile<SHAPE, HALVES>(cover, [&](auto shape, uint32_t n0, uint32_t m0) { hidden_backward_tile<T, decltype(shape)::value>(x, wg, wu, dy, wd, dg, du, h, act, n0, m0, lds_of(lds)); });
}

// rows of any width, stride and alignment -> rows of a multiple of 8 elements, 16-byte aligned, zeros behind the width; all of a call's tensors in one launch.
// Bound by starting up: 1537 x 387 - 1061 - 259, 5 MB, 6 us.
struct PadJob { const uint16_t* src; uint16_t* dst; uint64_t src_ld, pieces; uint32_t cols, dst_ld, first; };   // pieces: rows x dst_ld / 8; first: of its workgroups
struct PadJobs { PadJob job[5]; uint32_t n; };
constexpr uint32_t PAD_BLOCK = 1024;   // pieces of a workgroup
__global__ void __launch_bounds__(256) pad_rows_kernel(PadJobs jobs) {
	uint32_t j = 0;
	while (j + 1 < jobs.n && blockIdx.x >= jobs.job[j + 1].first) ++j;
	const PadJob& p = jobs.job[j];
	const uint32_t per_row = p.dst_ld / 8;
#pragma unroll
	for (int q = 0; q < 4; ++q) {
		const uint64_t i = (uint64_t)(blockIdx.x - p.first) * PAD_BLOCK + q * 256 + threadIdx.x;
		if (i >= p.pieces) continue;
		const uint64_t r = i / per_row;
		const uint32_t c = (uint32_t)(i % per_row) * 8;
		const uint16_t* row = p.src + r * p.src_ld;
		uint32_t v[8];
#pragma unroll
		for (int e = 0; e < 8; ++e) v[e] = row[min(c + e, p.cols - 1)];
#pragma unroll
		for (int e = 0; e < 8; ++e) v[e] = c + e < p.cols ? v[e] : 0u;
		*(uint4*)(p.dst + r * p.dst_ld + c) = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
	}
}

__global__ void __launch_bounds__(256) zero_kernel(uint16_t* p, uint64_t n) {
	for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (uint64_t)gridDim.x * 256) p[i] = 0;
}

// ---- host ------------------------------------------------------------------------------------------------------------------------------

constexpr uint32_t MAX_WIDTH = 1u << 20;
constexpr uint64_t MAX_ROWS = 1ull << 30, MAX_DMA_LD = 1u << 21;   // a tile's 256 rows stay within the 2 GiB of a buffer descriptor

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

// The sizes of one result before it has pointers, and how a group of them is cut: 256 x 256 tiles, or 128 x 128 (two workgroups a CU) with k in parts of at least 512, 1024, ..
// The least estimate of the group's time wins: the longest workgroup, or the CUs' common work and half of the longest, and what split sums cost.  In microseconds, fitted to 17 backward
// and 13 forward passes from 1 to 30000 rows with every cut each: 1.2 % above the best on average, 8 % at worst (profiles/gated_ffn_cuts.txt).  The fixed rule before (256 x 256 from 192 tiles on, else the smallest parts that
// make at most 512 workgroups) left the long sums of dx to a few workgroups where the weights' gradients alone had more tiles: 1 row backward through 4096 - 10240 - 4096 441 us where
// this takes 180, 100 rows 2048 - 8192 - 2048 312 and 84, 3000 rows 512 - 1536 - 512 75 and 62.
struct Size { uint64_t n, m, k; uint32_t n_products; };
struct Plan { uint32_t tiles_n, tiles_m, splits, k_split, partials; };
static Plan cut(const Size& s, bool big, uint64_t part) {
	const uint32_t t = big ? 256 : 128;
	const uint64_t splits = big ? 1 : std::max<uint64_t>(1, std::min<uint64_t>(ceil_div(s.k, part), s.k / 512));
	Plan p;
	p.tiles_n = (uint32_t)ceil_div(s.n, t); p.tiles_m = (uint32_t)ceil_div(s.m, t);
	p.k_split = (uint32_t)(ceil_div(ceil_div(s.k, 64), splits) * 64);
	p.splits = (uint32_t)std::max<uint64_t>(1, ceil_div(s.k, p.k_split));
	p.partials = p.splits > 1 ? p.splits * s.n_products : 0;
	return p;
}
constexpr uint64_t MAX_PARTIAL_TILES = 512;
static bool plan_group(const Size* s, int count, Plan* plan) {
	double least = 0.0;
	bool best_big = false;
	auto consider = [&](bool big, uint64_t part) {
		const double step = big ? 1.07 : 0.84, alone = big ? 1.07 : 0.24, ends = big ? 20.0 : 11.0;   // a step of 32 k on a full CU and on a workgroup's own; start and end
		const uint32_t slots = big ? 256 : 512;
		Plan p[3];
		double longest = 0.0, work = 0.0;
		uint64_t groups = 0, partial_tiles = 0;
		for (int i = 0; i < count; ++i) {
			p[i] = cut(s[i], big, part);
			const uint64_t tiles = (uint64_t)p[i].tiles_n * p[i].tiles_m, n = tiles * std::max(p[i].partials, 1u);
			const double steps = p[i].partials ? p[i].k_split / 32 : ceil_div(s[i].k, 32) * s[i].n_products;
			longest = std::max(longest, steps * alone + ends);
			work += (double)n * (steps * step + ends) / slots;
			groups += n;
			partial_tiles += tiles * p[i].partials;
		}
		if (partial_tiles > MAX_PARTIAL_TILES) return;
		const double time = std::max(longest, work + (groups > slots ? 0.5 * longest : 0.0)) + (partial_tiles ? 0.027 * (double)partial_tiles + 1.8 : 0.0);
		if (least != 0.0 && time >= least) return;
		least = time;
		best_big = big;
		for (int i = 0; i < count; ++i) plan[i] = p[i];
	};
	consider(true, 0);
	for (uint64_t part = 512; part <= 1ull << 31; part *= 2) consider(false, part);
	return best_big;
}
// room for a group's splits, never less than any smaller batch of the same block takes: at most MAX_PARTIAL_TILES, and at most k / 512 for each tile and product
static uint64_t partial_room(const Size* s, int count) {
	uint64_t parts = 0;
	for (int i = 0; i < count; ++i)
		if (s[i].k >= 1024) parts += ceil_div(s[i].n, 128) * ceil_div(s[i].m, 128) * s[i].n_products * (s[i].k / 512);
	return std::min<uint64_t>(MAX_PARTIAL_TILES, parts) * (128 * 128 * 4);
}

// The tiles of h.  A round of BIG tiles that would leave half of the chip idle or more is made of half tiles instead: such a round takes 0.7 of the other (352 BIG tiles, 4096 x 1024 -
// 2816: hidden_backward_kernel 114 us, with 242 and 220 half tiles 87; half tiles alone 111).  A round of SMALL tiles takes 0.6 of a round of BIG ones: 500 rows forward 4096 - 10240 -
// 4096 194 us with SMALL tiles (2 rounds of 512), 157 with BIG ones (160, one round); 700 rows backward 1024 - 2816 - 1024 (264 and 66) 63 and 75.
static bool cover_of(uint32_t width, uint64_t rows, Cover& c, uint32_t& groups) {
	const uint32_t bn = (uint32_t)ceil_div(width, 128), bm = (uint32_t)ceil_div(rows, 256), sn = (uint32_t)ceil_div(width, 64), sm = (uint32_t)ceil_div(rows, 128);
	const uint64_t tiles = (uint64_t)bn * bm;
	const uint32_t whole = (uint32_t)(tiles / 256 * 256 / bn);   // rows of BIG tiles in the full rounds
	const uint64_t halves = ceil_div(rows - std::min<uint64_t>(rows, whole * 256ull), 128);
	const bool mixed = tiles >= 256 && halves && halves * bn <= 256;
	const double big = mixed ? tiles / 256 + 0.7 : ceil_div(tiles, 256), small = 0.6 * ceil_div((uint64_t)sn * sm, 512);
	c = big <= small ? Cover{bn, mixed ? whole : bm, 0, 0} : Cover{sn, sm, 0, 0};
	groups = c.half_first = c.tiles_n * c.tiles_m;
	if (big > small || !mixed) return big <= small;
	c.half_tiles_m = (uint32_t)halves;
	c.half_first = (groups + 7) & ~7u;
	groups = c.half_first + bn * c.half_tiles_m;
	return true;
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
// ---- few rows: a launch for h and one for y, and one that packs x.  Workgroups of 4 to 16 waves (8 for the pair of matrices, whose sums take twice the LDS): about 2048 waves, 8 a CU.
template <class T, int NM, int NB, int MB, bool PX, bool PO>
static void launch_few(hipStream_t st, const void* x, uint64_t x_ld, uint32_t rows, const void* w0, const void* w1, uint32_t n, uint32_t k, uint32_t per, void* out, uint64_t out_ld, int act) {
	const uint32_t groups = (uint32_t)ceil_div(PO ? (n + 31) & ~31u : n, per);
	uint32_t waves = 4;
	while (waves < (uint32_t)few_waves(NM, NB) && groups * waves < 2048 && waves * 256 < k) waves *= 2;
	hipLaunchKernelGGL((few_rows_kernel<T, NM, NB, MB, PX, PO>), dim3(groups), dim3(64 * waves), 0, st, (const T*)x, x_ld, rows, (const T*)w0, (const T*)w1, n, k, per, (T*)out, out_ld, act);
}
// Rows of the weights to a workgroup: 16, or, where that gives some CUs a workgroup more than others, the same for every CU in as few rounds of the chip as 48 rows (MB = 4, whose
// sums would not fit: 32) leave, in steps of 8.  24 rows through 4096 - 10240 - 4096 (640 workgroups of 16 rows, 256 of 40) 77.4 -> 72.9 us, through 1500 - 5000 - 1500 36.3 -> 30.6;
// 2048 - 8192 - 2048, which 16 divide, 32.4 with 16 and 31.6 with 32, one row 23.7 and 24.8.
template <class T, int NM, int MB, bool PX, bool PO>
static void pick_few(hipStream_t st, const void* x, uint64_t x_ld, uint32_t rows, const void* w0, const void* w1, uint32_t n, uint32_t k, void* out, uint64_t out_ld, int act) {
	const uint64_t rounds = ceil_div(n, 256 * (MB == 4 ? 32 : 48)), even = up8(ceil_div(n, 256 * rounds));
	const uint32_t per = even * rounds < ceil_div(n, 256 * 16) * 16 ? (uint32_t)std::max<uint64_t>(even, 16) : 16;
	if (per <= 16) launch_few<T, NM, 1, MB, PX, PO>(st, x, x_ld, rows, w0, w1, n, k, per, out, out_ld, act);
	else if (per <= 32) launch_few<T, NM, 2, MB, PX, PO>(st, x, x_ld, rows, w0, w1, n, k, per, out, out_ld, act);
	else if constexpr (MB < 4) launch_few<T, NM, 3, MB, PX, PO>(st, x, x_ld, rows, w0, w1, n, k, per, out, out_ld, act);
}
constexpr uint32_t FEW_PACK_H = 8, FEW_PACK_X = 5 << 16;
// Which of the two products' rows are packed.  h where more than a few rows are read of it: 12 rows, 2048 - 8192 - 2048, 28.9 -> 27.9 us, one row 24 -> 26.5.  x where that saves more
// than its launch takes: 32 rows of that block 33.4 us without and 34 with, 48 rows 41.9 and 39.4.
static uint32_t few_pitch(uint32_t width) { return (width + 31) & ~31u; }
static uint64_t few_padded(uint64_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }
static bool few_pack_h(uint64_t rows) { return rows > FEW_PACK_H; }
static bool few_pack_x(uint64_t rows, const NgpGatedFfn& b) { return few_pack_h(rows) && rows * ((uint64_t)b.n_in + b.n_hidden) >= FEW_PACK_X; }
template <class T, int MB>
static void launch_few_pair(hipStream_t st, const NgpGatedFfn& b, uint32_t rows, const void* x, uint64_t x_ld, const void* wg, const void* wu, const void* wd, void* y, uint64_t y_ld, void* h, void* packed) {
	const uint32_t pitch = few_pitch(b.n_hidden), d = b.n_in, f = b.n_hidden;
	if (few_pack_x(rows, b)) {
		hipLaunchKernelGGL((pack_few_kernel<T, MB>), dim3((d + 127) / 128 * MB), dim3(256), 0, st, (const T*)x, x_ld, rows, d, (T*)packed);
		pick_few<T, 2, MB, true, true>(st, packed, 0, rows, wg, wu, f, d, h, 0, b.activation);
	} else if (few_pack_h(rows)) pick_few<T, 2, MB, false, true>(st, x, x_ld, rows, wg, wu, f, d, h, 0, b.activation);
	else pick_few<T, 2, 1, false, false>(st, x, x_ld, rows, wg, wu, f, d, h, pitch, b.activation);
	if (few_pack_h(rows)) pick_few<T, 1, MB, true, false>(st, h, 0, rows, wd, nullptr, b.n_out, f, y, y_ld, 0);
	else pick_few<T, 1, 1, false, false>(st, h, pitch, rows, wd, nullptr, b.n_out, f, y, y_ld, 0);
}
template <class T>
static int run_few(hipStream_t st, const NgpGatedFfn& b, uint32_t rows, const void* x, uint64_t x_ld, const void* wg, const void* wu, const void* wd, void* y, uint64_t y_ld, void* h, void* packed) {
	if (rows <= 16) launch_few_pair<T, 1>(st, b, rows, x, x_ld, wg, wu, wd, y, y_ld, h, packed);
	else if (rows <= 32) launch_few_pair<T, 2>(st, b, rows, x, x_ld, wg, wu, wd, y, y_ld, h, packed);
	else launch_few_pair<T, 4>(st, b, rows, x, x_ld, wg, wu, wd, y, y_ld, h, packed);
	NGP_LAUNCH_CHECK("few_rows_kernel");
	return 0;
}

static bool vector_rows(const void* p, uint64_t ld, uint32_t cols) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && cols % 8 == 0; }

// What a call keeps in its workspace.  `any`: room for padded copies of every input, else of those whose width is no multiple of 8.
struct Space {
	uint32_t d8, f8, o8, fp;                                   // widths as the copies have them; fp: row pitch of h, dg and du
	void *x = nullptr, *wg = nullptr, *wu = nullptr, *wd = nullptr, *dy = nullptr, *h = nullptr, *d = nullptr;
	float* partial = nullptr;
	Size size[3];
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
			take_few(a, b, rows);
			bytes = a.used;
			return;
		}
		if (has_copies(b.n_in, any)) { x = a.take(rows * d8 * 2); wg = a.take((uint64_t)b.n_hidden * d8 * 2); wu = a.take((uint64_t)b.n_hidden * d8 * 2); }
		if (has_copies(b.n_hidden, any)) wd = a.take((uint64_t)b.n_out * f8 * 2);
		if (backward && has_copies(b.n_out, any)) dy = a.take(rows * o8 * 2);
		h = a.take(rows * fp * 2);
		if (backward) {
			d = a.take(rows * fp * 4);
			size[0] = {b.n_in, rows, b.n_hidden, 2};                       // dx
			size[1] = {b.n_in, 2 * (uint64_t)fp, rows, 1};                 // dw_gate over dw_up
			size[2] = {b.n_hidden, b.n_out, rows, 1};                      // dw_down
			partial = (float*)a.take(partial_room(size, 3));
		} else {
			size[0] = {b.n_out, rows, f8, 1};
			partial = (float*)a.take(partial_room(size, 1));
		}
		bytes = a.used;
		if (!backward) {   // never less than any smaller batch takes
			Arena few{nullptr};
			Space unused = *this;
			unused.take_few(few, b, FEW_ROWS);
			bytes = std::max(bytes, few.used);
		}
	}
	void take_few(Arena& a, const NgpGatedFfn& b, uint64_t rows) {
		h = a.take((few_pack_h(rows) ? few_padded(rows) : rows) * fp * 2);
		if (few_pack_x(rows, b)) x = a.take(few_padded(rows) * few_pitch(b.n_in) * 2);
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
	PadJobs pads{};
	uint32_t pad_groups = 0;
	// `t` as the DMA takes it, through `copy` where it is not ready (copy null: not reserved); pad() runs the copies
	Tensor ready(const Tensor& t, void* copy, uint32_t width8) {
		if (rc || dma_ready(t)) return t;
		if (!copy) { rc = refuse("ngp_hip_gated_ffn: a row that is not 16-byte aligned needs the workspace of NGP_FFN_ANY_LAYOUT"); return t; }
		PadJob& j = pads.job[pads.n++];
		j = PadJob{(const uint16_t*)t.p, (uint16_t*)copy, t.ld, t.rows * (width8 / 8), t.cols, width8, pad_groups};
		pad_groups += (uint32_t)ceil_div(j.pieces, PAD_BLOCK);
		return Tensor{copy, width8, t.rows, width8};
	}
	void pad() {
		if (rc || !pads.n) return;
		hipLaunchKernelGGL(pad_rows_kernel, dim3(pad_groups), dim3(256), 0, st, pads);
		ok("pad_rows_kernel");
	}
	// The group's products, item i of size sizes[which[i]]; `partial`: the room of partial_room.  The plan is made for all `count` sizes, whichever of them are asked for: a result's bits
	// do not depend on the others being wanted too.
	template <class T, bool FORWARD> void products(Group<T>& g, const int* which, const Size* sizes, int count, float* partial) {
		if (rc || !g.n) return;
		Plan plans[3];
		const bool big = plan_group(sizes, count, plans);
		uint32_t groups = 0, sum_groups = 0;
		bool sums = false;
		for (uint32_t i = 0; i < g.n; ++i) {
			Item<T>& it = g.item[i];
			const Plan& plan = plans[which[i]];
			it.n_products = sizes[which[i]].n_products;
			it.tiles_n = plan.tiles_n; it.tiles_m = plan.tiles_m; it.splits = plan.splits; it.k_split = plan.k_split; it.partials = plan.partials;
			it.partial = partial;
			partial += (uint64_t)it.partials * it.tiles_n * it.tiles_m * (128 * 128);
			it.first = groups;
			it.count = it.tiles_n * it.tiles_m * std::max(1u, it.partials);
			groups += (it.count + 7) & ~7u;
			sums |= it.partials != 0;
		}
		if (big) hipLaunchKernelGGL((group_kernel<T, BIG, FORWARD>), dim3(groups), dim3(Shape<BIG>::THREADS), 0, st, g);
		else hipLaunchKernelGGL((group_kernel<T, SMALL, FORWARD>), dim3(groups), dim3(Shape<SMALL>::THREADS), 0, st, g);
		if (!ok("group_kernel") || !sums) return;
		Group<T> s;
		s.n = 0;
		for (uint32_t i = 0; i < g.n; ++i) {
			if (!g.item[i].partials) continue;
			Item<T>& it = s.item[s.n++] = g.item[i];
			const uint32_t tiles = it.tiles_n * it.tiles_m;
			it.first = sum_groups;
			sum_groups += tiles;
			if (it.partials > SUM_FAN) {
				const uint64_t floats = (uint64_t)tiles * 128 * 128;
				hipLaunchKernelGGL(split_fold_kernel, dim3((uint32_t)(floats / 1024 * ceil_div(it.partials, SUM_FAN))), dim3(256), 0, st, it.partial, it.partials, floats);
			}
		}
		hipLaunchKernelGGL((group_sum_kernel<T>), dim3(sum_groups * SUM_GROUPS), dim3(256), 0, st, s);
		ok("group_sum_kernel");
	}
};

static Mat kc(const Tensor& t) { return Mat{t.p, t.ld, (uint32_t)t.rows, t.cols}; }            // rows of the tensor = rows of the operand
static Mat rc(const Tensor& t) { return Mat{t.p, t.ld, t.cols, (uint32_t)t.rows}; }            // rows of the tensor = k
template <class T> static Rows2<T> whole(void* p, uint64_t ld, uint64_t rows, uint32_t cols) { const Out<T> o{(T*)p, ld, (uint32_t)rows, cols}; return Rows2<T>{o, o, 0xffffffffu}; }

template <class T>
static int forward(hipStream_t st, const NgpGatedFfn& b, const Space& s, Tensor x, Tensor wg, Tensor wu, Tensor wd, void* y, uint64_t y_ld) {
	Launch l{st};
	x = l.ready(x, s.x, s.d8); wg = l.ready(wg, s.wg, s.d8); wu = l.ready(wu, s.wu, s.d8); wd = l.ready(wd, s.wd, s.f8);
	l.pad();
	if (l.rc) return l.rc;
	const Out<T> h{(T*)s.h, s.fp, (uint32_t)x.rows, s.fp};
	uint32_t groups;
	Cover cover;
	const bool big = cover_of(s.fp, x.rows, cover, groups);
	if (cover.half_tiles_m) hipLaunchKernelGGL((gate_up_kernel<T, BIG, true>), dim3(groups), dim3(Shape<BIG>::THREADS), 0, st, kc(x), kc(wg), kc(wu), h, b.activation, cover);
	else if (big) hipLaunchKernelGGL((gate_up_kernel<T, BIG, false>), dim3(groups), dim3(Shape<BIG>::THREADS), 0, st, kc(x), kc(wg), kc(wu), h, b.activation, cover);
	else hipLaunchKernelGGL((gate_up_kernel<T, SMALL, false>), dim3(groups), dim3(Shape<SMALL>::THREADS), 0, st, kc(x), kc(wg), kc(wu), h, b.activation, cover);
	l.ok("gate_up_kernel");
	const Tensor th{s.h, s.fp, x.rows, s.f8};
	Group<T> g;
	g.n = 1;
	g.item[0].p[0] = Pair{kc(wd), kc(th)};
	g.item[0].out = whole<T>(y, y_ld, x.rows, b.n_out);
	const int which[1] = {0};
	l.products<T, true>(g, which, s.size, 1, s.partial);
	return l.rc;
}

template <class T>
static int backward(hipStream_t st, const NgpGatedFfn& b, const Space& s, Tensor x, Tensor wg, Tensor wu, Tensor wd, Tensor dy, void* dx, uint64_t dx_ld, void* dwg, void* dwu, void* dwd) {
	Launch l{st};
	x = l.ready(x, s.x, s.d8); wg = l.ready(wg, s.wg, s.d8); wu = l.ready(wu, s.wu, s.d8); wd = l.ready(wd, s.wd, s.f8); dy = l.ready(dy, s.dy, s.o8);
	l.pad();
	if (l.rc) return l.rc;
	const uint32_t rows = (uint32_t)x.rows;
	T* const d = (T*)s.d;
	const Out<T> h{(T*)s.h, s.fp, rows, s.fp}, dg{d, 2ull * s.fp, rows, s.fp}, du{d + s.fp, 2ull * s.fp, rows, s.fp};
	uint32_t groups;
	Cover cover;
	const bool big = cover_of(s.fp, rows, cover, groups);
	if (cover.half_tiles_m) hipLaunchKernelGGL((hidden_backward_kernel<T, BIG, true>), dim3(groups), dim3(Shape<BIG>::THREADS), 0, st, kc(x), kc(wg), kc(wu), kc(dy), rc(wd), dg, du, h, b.activation, cover);
	else if (big) hipLaunchKernelGGL((hidden_backward_kernel<T, BIG, false>), dim3(groups), dim3(Shape<BIG>::THREADS), 0, st, kc(x), kc(wg), kc(wu), kc(dy), rc(wd), dg, du, h, b.activation, cover);
	else hipLaunchKernelGGL((hidden_backward_kernel<T, SMALL, false>), dim3(groups), dim3(Shape<SMALL>::THREADS), 0, st, kc(x), kc(wg), kc(wu), kc(dy), rc(wd), dg, du, h, b.activation, cover);
	l.ok("hidden_backward_kernel");
	const Tensor tdg{dg.p, dg.ld, rows, s.f8}, tdu{du.p, du.ld, rows, s.f8}, tboth{d, 2ull * s.fp, rows, 2 * s.fp}, th{s.h, s.fp, rows, s.fp};
	Group<T> g;
	int which[3];
	g.n = 0;
	auto add = [&](int size, const Pair& p0, const Pair& p1, const Rows2<T>& out, bool turned) {
		Item<T>& it = g.item[g.n];
		it.p[0] = p0; it.p[1] = p1; it.out = out; it.turned = turned;
		which[g.n++] = size;
	};
	if (dx) add(0, Pair{rc(wg), kc(tdg)}, Pair{rc(wu), kc(tdu)}, whole<T>(dx, dx_ld, rows, b.n_in), false);
	if (dwg) {
		const Out<T> og{(T*)dwg, b.n_in, b.n_hidden, b.n_in}, ou{(T*)dwu, b.n_in, b.n_hidden, b.n_in};
		const Pair gu{rc(x), rc(tboth)}, down{rc(th), rc(dy)};
		add(1, gu, gu, Rows2<T>{og, ou, s.fp}, true);
		add(2, down, down, whole<T>(dwd, b.n_hidden, b.n_out, b.n_hidden), true);
	}
	l.products<T, false>(g, which, s.size, 3, s.partial);
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
	if (n_rows > MAX_ROWS) return refuse("ngp_hip_gated_ffn_forward: more than 2^30 rows");
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
	if (n_rows <= FEW_ROWS) return b->dtype == NGP_DTYPE_F16 ? run_few<f16>((hipStream_t)stream, *b, (uint32_t)n_rows, x, x_stride, w_gate, w_up, w_down, y, y_stride, s.h, s.x)
	                                                         : run_few<b16>((hipStream_t)stream, *b, (uint32_t)n_rows, x, x_stride, w_gate, w_up, w_down, y, y_stride, s.h, s.x);
	if (b->dtype == NGP_DTYPE_F16) return forward<f16>((hipStream_t)stream, *b, s, tx, tg, tu, td, y, y_stride);
	return forward<b16>((hipStream_t)stream, *b, s, tx, tg, tu, td, y, y_stride);
}

int ngp_hip_gated_ffn_backward(void* stream, const NgpGatedFfn* b, uint64_t n_rows, const void* x, uint64_t x_stride, const void* w_gate, const void* w_up, const void* w_down,
                               const void* dy, uint64_t dy_stride, void* dx, uint64_t dx_stride, void* dw_gate, void* dw_up, void* dw_down, void* workspace, uint64_t workspace_bytes) {
	using namespace ffn;
	if (check_block(b, "ngp_hip_gated_ffn_backward")) return -1;
	if (n_rows > MAX_ROWS) return refuse("ngp_hip_gated_ffn_backward: more than 2^30 rows");
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
