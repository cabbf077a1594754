// gated_ffn_few.cuh — the forward pass of a few rows (up to 64) through a wide block: bound by reading the weights once.
//
// A workgroup owns 16 to 48 rows of the weights (of gate and up: the same), its waves share k, with 16-byte loads straight into the A operand of v_mfma_f32_16x16x32 (a load covers 64
// contiguous bytes of 16 weight rows); the rows of x are the B operand, 16 to a block, from L2.  Sums meet in LDS and are added in the waves' order.  No LDS staging, no alignment
// needed: a 16-byte load from a 2-byte boundary is one instruction on this hardware.
// Every workgroup reads all of x: 24 rows through 4096 - 10240 - 4096 in f16 took 87 us, 61 without that.  The rows lie a power of two apart and come in pieces of 64 bytes; packed as
// the fragments they are read as, 1 KiB each, it is 73 us (64 rows: 135 -> 104), although x is packed in a launch of its own; h is written packed by the product that makes it.
// One row: 252 MB of weights in 57 us, 4.4 TB/s.
// Included by gated_ffn.hip.
#pragma once

namespace ngp {
namespace ffn {

typedef i32x4 i32x4_any __attribute__((aligned(2)));

constexpr int FEW_ROWS = 64;
// k-blocks of 32 per wave and turn: about 64 registers of weights, or, where x is packed, twice 64 of both
constexpr int few_blocks(int w, int mb, bool packed) { return !packed ? (16 / w < 8 ? 16 / w : 8) : mb == 4 ? 2 : 16 / (w + mb) < 4 ? 16 / (w + mb) : 4; }
constexpr int few_waves(int nm, int nb) { return nm == 2 || nb > 1 ? 8 : 16; }

// Packed rows: element (m, k) of MB blocks of 16 rows where the lane that needs it finds it, 1 KiB to a fragment, k padded to 32
template <int MB> __device__ __forceinline__ uint64_t packed_at(uint32_t m, uint32_t k) { return (((uint64_t)(k >> 5) * MB + (m >> 4)) * 64 + ((k >> 3) & 3) * 16 + (m & 15)) * 8 + (k & 7); }
template <class T, int MB>
__global__ void __launch_bounds__(256) pack_few_kernel(const T* __restrict__ x, uint64_t x_ld, uint32_t rows, uint32_t k, T* __restrict__ out) {
	const uint32_t lane = threadIdx.x & 63, m = (blockIdx.x % MB) * 16 + (lane & 15), at = (blockIdx.x / MB * 4 + (threadIdx.x >> 6)) * 32 + 8 * (lane >> 4);
	if (at >= ((k + 31) & ~31u)) return;
	const T* r = x + min(m, rows - 1) * x_ld;
	*(i32x4*)(out + packed_at<MB>(m, at)) = at + 8 <= k ? i32x4(*(const i32x4_any*)(r + at)) : load8<T, false>(r, at, k);
}

// NM = 2: h = act(x w0^T) * (x w1^T), NM = 1: y = x w0^T; NB blocks of 16 rows of the weights, of which `per` rows in all are this workgroup's; MB blocks of 16 rows of x, which are
// packed (PX) or not; the result is to be packed (PO) or not
template <class T, int NM, int NB, int MB, bool PX, bool PO>
__global__ void __launch_bounds__(64 * few_waves(NM, NB)) few_rows_kernel(const T* __restrict__ x, uint64_t x_ld, uint32_t rows, const T* __restrict__ w0, const T* __restrict__ w1, uint32_t n, uint32_t k,
                                                                          uint32_t per, T* __restrict__ out, uint64_t out_ld, int act) {
	constexpr int W = NM * NB, BLOCKS = few_blocks(W, MB, PX), BATCH = BLOCKS * 32;
	__shared__ f32x4 sums[few_waves(NM, NB)][W][MB][64];
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
	const uint32_t n0 = blockIdx.x * per, n_end = n0 + per;
	const uint32_t kl = 8 * (lane >> 4);
	const T* w[W];   // [block][matrix]; rows behind this workgroup's are its last one again
#pragma unroll
	for (int i = 0; i < W; ++i) w[i] = (i % NM ? w1 : w0) + (uint64_t)min(n0 + i / NM * 16 + (lane & 15), min(n_end, n) - 1) * k;
	const T* xr[MB];
#pragma unroll
	for (int b = 0; b < MB; ++b) xr[b] = PX ? x + (b * 64 + (lane & 15)) * 8 : x + min((uint32_t)(b * 16 + (lane & 15)), rows - 1) * x_ld;
	f32x4 acc[W][MB];
#pragma unroll
	for (int j = 0; j < W; ++j)
#pragma unroll
		for (int b = 0; b < MB; ++b) acc[j][b] = f32x4{0, 0, 0, 0};
	auto load_x = [&](int b, uint32_t c) { return PX ? *(const i32x4*)(xr[b] + (uint64_t)c * (MB * 16) + kl * 16) : i32x4(*(const i32x4_any*)(xr[b] + c + kl)); };
	uint32_t kc;
	if constexpr (PX) {   // two batches of weights and rows in flight
		const uint32_t full = k / BATCH, mine = full > (uint32_t)wave ? (full - wave + waves - 1) / waves : 0;   // whole batches: wave, wave + waves, ..
		if (mine) {
			i32x4 f[2][W][BLOCKS], v[2][MB][BLOCKS];
			auto load = [&](int q, uint32_t i) {   // behind the last batch: that one again, not used
				const uint32_t at = (wave + min(i, mine - 1) * waves) * BATCH;
#pragma unroll
				for (int c = 0; c < BLOCKS; ++c) {
#pragma unroll
					for (int j = 0; j < W; ++j) f[q][j][c] = *(const i32x4_any*)(w[j] + at + c * 32 + kl);
#pragma unroll
					for (int b = 0; b < MB; ++b) v[q][b][c] = load_x(b, at + c * 32);
				}
			};
			load(0, 0);
			load(1, 1);
			for (uint32_t i = 0; i < mine; i += 2)
#pragma unroll
				for (int q = 0; q < 2; ++q) {
					if (i + q < mine)
#pragma unroll
						for (int c = 0; c < BLOCKS; ++c)
#pragma unroll
							for (int j = 0; j < W; ++j)
#pragma unroll
								for (int b = 0; b < MB; ++b) acc[j][b] = mfma16<T>(f[q][j][c], v[q][b][c], acc[j][b]);
					load(q, i + q + 2);
				}
		}
		kc = full % waves == (uint32_t)wave ? full * BATCH : k;
	} else
		for (kc = wave * BATCH; kc + BATCH <= k; kc += waves * BATCH) {
			i32x4 f[W][BLOCKS];
#pragma unroll
			for (int c = 0; c < BLOCKS; ++c)
#pragma unroll
				for (int j = 0; j < W; ++j) f[j][c] = *(const i32x4_any*)(w[j] + kc + c * 32 + kl);
#pragma unroll
			for (int c = 0; c < BLOCKS; ++c) {
				i32x4 v[MB];
#pragma unroll
				for (int b = 0; b < MB; ++b) v[b] = load_x(b, kc + c * 32);
#pragma unroll
				for (int j = 0; j < W; ++j)
#pragma unroll
					for (int b = 0; b < MB; ++b) acc[j][b] = mfma16<T>(f[j][c], v[b], acc[j][b]);
			}
		}
	if (kc < k)   // the wave whose turn the last, shorter chunk is
		for (uint32_t c = kc; c < k; c += 32) {
			const uint32_t at = c + kl;
			auto part = [&](const T* p) { return at + 8 <= k ? i32x4(*(const i32x4_any*)(p + at)) : load8<T, false>(p, at, k); };
			i32x4 f[W];
#pragma unroll
			for (int j = 0; j < W; ++j) f[j] = part(w[j]);
#pragma unroll
			for (int b = 0; b < MB; ++b) {
				const i32x4 v = PX ? load_x(b, c) : part(xr[b]);
#pragma unroll
				for (int j = 0; j < W; ++j) acc[j][b] = mfma16<T>(f[j], v, acc[j][b]);
			}
		}
#pragma unroll
	for (int j = 0; j < W; ++j)
#pragma unroll
		for (int b = 0; b < MB; ++b) sums[wave][j][b][lane] = acc[j][b];
	__syncthreads();
	// lane: row m = lane & 15 of block b, columns c .. + 3
	for (int i = wave; i < NB * MB; i += waves) {
		const int nb = i / MB, b = i % MB;
		f32x4 s = sums[0][nb * NM][b][lane], u = sums[0][nb * NM + NM - 1][b][lane];
		for (int v = 1; v < waves; ++v) {
			s += sums[v][nb * NM][b][lane];
			if (NM == 2) u += sums[v][nb * NM + NM - 1][b][lane];
		}
		const uint32_t m = b * 16 + (lane & 15), c = n0 + nb * 16 + 4 * (lane >> 4);
		if (NM == 2) with_activation(act, [&](auto a) {
#pragma unroll
			for (int e = 0; e < 4; ++e) s[e] = activate<decltype(a)::value>(s[e]).x * u[e];
		});
		if (m >= rows || c >= n_end) continue;
		if (PO) {   // zeros behind n: the next product's k goes on to a multiple of 32
			typedef T t4 __attribute__((ext_vector_type(4)));
			t4 v;
#pragma unroll
			for (int e = 0; e < 4; ++e) v[e] = c + e < n ? (T)s[e] : (T)0.0f;
			if (c < ((n + 31) & ~31u)) *(t4*)(out + packed_at<MB>(m, c)) = v;
			continue;
		}
		T* p = out + m * out_ld + c;
#pragma unroll
		for (int e = 0; e < 4; ++e)
			if (c + e < n) p[e] = (T)s[e];
	}
}

} // namespace ffn
} // namespace ngp
