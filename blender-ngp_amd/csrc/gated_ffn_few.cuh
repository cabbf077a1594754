// gated_ffn_few.cuh — the forward pass of a few rows (up to 64) through a wide block: bound by reading the weights once.
//
// A workgroup owns 16 rows of the weights (of gate and up: the same 16), its waves share k: each takes 256 of it in turn, eight 16-byte loads a lane and matrix in flight, straight
// into the A operand of v_mfma_f32_16x16x32 (a load covers 64 contiguous bytes of 16 weight rows); the rows of x are the B operand, 16 to a block, read the same way from L2.  Sums
// meet in LDS and are added in the waves' order.  No LDS staging, no alignment needed: a 16-byte load from a 2-byte boundary is one instruction on this hardware.
// Included by gated_ffn.hip.
#pragma once

namespace ngp {
namespace ffn {

typedef i32x4 i32x4_any __attribute__((aligned(2)));

constexpr int FEW_ROWS = 64, FEW_CHUNK = 8;   // k-blocks of 32 per wave and turn

// NM = 2: h = act(x w0^T) * (x w1^T), NM = 1: y = x w0^T; MB blocks of 16 rows of x
template <class T, int NM, int MB>
__global__ void __launch_bounds__(1024) few_rows_kernel(const T* __restrict__ x, uint64_t x_ld, uint32_t rows, const T* __restrict__ w0, const T* __restrict__ w1, uint32_t n, uint32_t k, T* __restrict__ out,
                                                        uint64_t out_ld, int act) {
	__shared__ f32x4 sums[NM == 2 ? 8 : 16][NM][MB][64];
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
	const uint32_t n0 = blockIdx.x * 16, r = min(n0 + (lane & 15), n - 1);
	const uint32_t kl = 8 * (lane >> 4);
	const T* w[NM];
	w[0] = w0 + (uint64_t)r * k;
	if (NM == 2) w[1] = w1 + (uint64_t)r * k;
	const T* xr[MB];
#pragma unroll
	for (int b = 0; b < MB; ++b) xr[b] = x + min((uint32_t)(b * 16 + (lane & 15)), rows - 1) * x_ld;
	f32x4 acc[NM][MB];
#pragma unroll
	for (int j = 0; j < NM; ++j)
#pragma unroll
		for (int b = 0; b < MB; ++b) acc[j][b] = f32x4{0, 0, 0, 0};
	uint32_t kc = wave * (FEW_CHUNK * 32);
	for (; kc + FEW_CHUNK * 32 <= k; kc += waves * (FEW_CHUNK * 32)) {
		i32x4 f[NM][FEW_CHUNK];
#pragma unroll
		for (int c = 0; c < FEW_CHUNK; ++c)
#pragma unroll
			for (int j = 0; j < NM; ++j) f[j][c] = *(const i32x4_any*)(w[j] + kc + c * 32 + kl);
#pragma unroll
		for (int c = 0; c < FEW_CHUNK; ++c) {
			i32x4 v[MB];
#pragma unroll
			for (int b = 0; b < MB; ++b) v[b] = *(const i32x4_any*)(xr[b] + kc + c * 32 + kl);
#pragma unroll
			for (int j = 0; j < NM; ++j)
#pragma unroll
				for (int b = 0; b < MB; ++b) acc[j][b] = mfma16<T>(f[j][c], v[b], acc[j][b]);
		}
	}
	if (kc < k)   // the wave whose turn the last, shorter chunk is
		for (uint32_t c = kc; c < k; c += 32) {
			const uint32_t at = c + kl;
			auto part = [&](const T* p) { return at + 8 <= k ? i32x4(*(const i32x4_any*)(p + at)) : load8<T, false>(p, at, k); };
			i32x4 f[NM];
#pragma unroll
			for (int j = 0; j < NM; ++j) f[j] = part(w[j]);
#pragma unroll
			for (int b = 0; b < MB; ++b) {
				const i32x4 v = part(xr[b]);
#pragma unroll
				for (int j = 0; j < NM; ++j) acc[j][b] = mfma16<T>(f[j], v, acc[j][b]);
			}
		}
#pragma unroll
	for (int j = 0; j < NM; ++j)
#pragma unroll
		for (int b = 0; b < MB; ++b) sums[wave][j][b][lane] = acc[j][b];
	__syncthreads();
	// lane: row m = lane & 15 of block b, columns n0 + 4 (lane >> 4) .. + 3
	for (int b = wave; b < MB; b += waves) {
		f32x4 s = sums[0][0][b][lane], u = sums[0][NM - 1][b][lane];
		for (int i = 1; i < waves; ++i) {
			s += sums[i][0][b][lane];
			if (NM == 2) u += sums[i][NM - 1][b][lane];
		}
		const uint32_t m = b * 16 + (lane & 15), c = n0 + 4 * (lane >> 4);
		if (NM == 2) with_activation(act, [&](auto a) {
#pragma unroll
			for (int e = 0; e < 4; ++e) s[e] = activate<decltype(a)::value>(s[e]).x * u[e];
		});
		if (m >= rows) continue;
		T* p = out + m * out_ld + c;
#pragma unroll
		for (int e = 0; e < 4; ++e)
			if (c + e < n) p[e] = (T)s[e];
	}
}

} // namespace ffn
} // namespace ngp
