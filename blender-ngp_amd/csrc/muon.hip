// muon.hip — the Muon step of the matrix parameters: momentum, orthogonalisation by Newton-Schulz products, weight update (include/ngp_hip.h: ngp_hip_muon_step).
//
//   m <- beta m + g;  u = g + beta m (Nesterov) or m;  X_0 = u / (|u|_F + eps);  X <- a X + (b A + c A^2) X with A = X X^T;  w <- (1 - lr wd) w - lr sqrt(max(1, rows / cols)) X
//
// X is taken with its short side n as rows (k = the long side): A is n x n.  An iteration is three products, 2 n^2 k + 2 n^3 + 2 n^2 k operations, of which the two symmetric ones
// (A, and B = a I + b A + c A^2) are computed on and below the diagonal only and written twice.
//
// Precision.  The quintic's slope at zero is 3.44: five iterations magnify what an early rounding does to a small singular value up to 480 times, so the products cannot run on
// operands of 11 (fp16) or 8 bits.  fp32 matrix instructions would do at 1/16 of the fp16 rate; instead every matrix is kept as two fp16 halves, v = hi + lo with
// hi = fp16(v) and lo = fp16(v - hi): 22 bits, and a product is three fp16 ones (hi hi + hi lo + lo hi, fp32 accumulation; lo lo is below the last bit kept).  Powers of two keep both
// halves inside fp16's normal range: X is held as 2^15 X (|X_ij| <= 1.21, typically 1 / sqrt(n k)), A and B as 2^13 of themselves (spectral norms at most 1.5 and 3.5).  fp32 arithmetic
// is as far from 64 bits: of the norm of X after 5 iterations, random 64 x 64 9e-7 here and 1.2e-6 there, 768 x 768 1.7e-6 and 2.8e-6, 768 x 768 of rank 1 1.4e-4 and 2.3e-4.
// Layout of such a matrix: row-major, per 32 columns 32 hi values and 32 lo values: 128 bytes of a row are both halves of 32 k.
//
// X is kept transposed, [k][n], and only so: A = X X^T reads it with k as the rows (transposed LDS reads on both sides), X^T <- X^T B with B, which is symmetric, along rows.  One
// orientation to write instead of two: for matrices that do not stay in the cache between launches the iterations are as much bound by memory as by the products.
#include <algorithm>
#include <math.h>
#include <stdio.h>
#include "ngp_device.cuh"
#include "matmul_mfma.cuh"

#pragma clang fp contract(fast)

namespace ngp {
namespace muon {

using namespace mm;

constexpr float SX = 32768.0f, SA = 8192.0f;                      // scales of X and of A, B
constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
constexpr uint32_t MAX_SIDE = 65536, SUM_BLOCKS = 1024;

struct Job {
	uint64_t offset;                    // of the matrix in the parameter vector, in elements
	uint32_t rows, cols, n, k;          // n = min, k = max of rows and cols
	uint32_t np;                        // n up to a multiple of 32
	f16 *xt[2], *a, *b;                 // X^T [k][2 np] (in slabs: one, [k][128]; two: an iteration reads one and writes the other), A and B [n][2 np]
	double* sums;
	float* partial;                     // the parts' sums of the tiles of A
	uint32_t parts;                     // of k, in the products that give A; of a matrix in slabs: the rows of one
};
enum { START_SUM, START_SPLIT, START_GRAM, START_SYM, START_APPLY, N_STARTS };
struct Step { float lr, momentum, decay, eps, inv_loss_scale; int nesterov, dtype; const void* grads; float* master; void* params; float* buffer; };
// As many matrices to a launch as its arguments, 4 KiB, hold beside Step, two numbers and the count: a longer list is more than one chain of launches, each waiting for the one before.
constexpr uint32_t ARGUMENT_BYTES = 4096, MAX_JOBS = (ARGUMENT_BYTES - sizeof(Step) - 32 - 4 * N_STARTS) / (sizeof(Job) + 4 * N_STARTS);
struct Jobs {
	Job job[MAX_JOBS];
	uint32_t start[N_STARTS][MAX_JOBS + 1];   // first workgroup of each job, per kind of kernel (the products: of the tile of the launch)
	uint32_t count;
};
static_assert(sizeof(Jobs) + sizeof(Step) + 16 <= ARGUMENT_BYTES && MAX_JOBS < 64, "fits the arguments of a launch; job_of has a lane for every end");

// the job of a workgroup, which becomes its number within the job: every lane compares one job's end
__device__ __forceinline__ uint32_t job_of(const Jobs& j, int kind, uint32_t& pid) {
	const uint32_t lane = threadIdx.x & 63, i = (uint32_t)__popcll(__ballot(lane < j.count && j.start[kind][lane < j.count ? lane + 1 : 0] <= pid));
	pid -= j.start[kind][i];
	return i;
}
__device__ __forceinline__ float load_grad(const Step& s, uint64_t i) {
	const float g = s.dtype == NGP_DTYPE_F32 ? ((const float*)s.grads)[i] : s.dtype == NGP_DTYPE_F16 ? (float)((const f16*)s.grads)[i] : (float)((const b16*)s.grads)[i];
	return g * s.inv_loss_scale;
}

// N gradients at once, and N weights: the choice of type is made once, and the loads (the stores) follow each other
template <int N> __device__ __forceinline__ void load_grads(const Step& s, const uint64_t (&at)[N], float (&g)[N]) {
	if (s.dtype == NGP_DTYPE_F32) {
#pragma unroll
		for (int i = 0; i < N; ++i) g[i] = ((const float*)s.grads)[at[i]];
	} else if (s.dtype == NGP_DTYPE_F16) {
#pragma unroll
		for (int i = 0; i < N; ++i) g[i] = (float)((const f16*)s.grads)[at[i]];
	} else {
#pragma unroll
		for (int i = 0; i < N; ++i) g[i] = (float)((const b16*)s.grads)[at[i]];
	}
#pragma unroll
	for (int i = 0; i < N; ++i) g[i] *= s.inv_loss_scale;
}
template <int N> __device__ __forceinline__ void set_weights(const Step& s, const uint64_t (&at)[N], const float (&w)[N], const bool (&in)[N]) {
#pragma unroll
	for (int i = 0; i < N; ++i)
		if (in[i]) s.master[at[i]] = w[i];
	if (!s.params) return;
	if (s.dtype == NGP_DTYPE_F16) {
#pragma unroll
		for (int i = 0; i < N; ++i)
			if (in[i]) ((f16*)s.params)[at[i]] = (f16)w[i];
	} else {
#pragma unroll
		for (int i = 0; i < N; ++i)
			if (in[i]) ((b16*)s.params)[at[i]] = (b16)w[i];
	}
}

__device__ __forceinline__ double block_sum(double v, double* lds) {   // 256 threads, a fixed order
	for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
	if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
	__syncthreads();
	v = lds[0] + lds[1] + lds[2] + lds[3];
	__syncthreads();
	return v;
}

// four gradients from i on (i and the vector's base aligned to four elements)
__device__ __forceinline__ f32x4 load_grad4(const Step& s, uint64_t i) {
	typedef f16 h4 __attribute__((ext_vector_type(4)));
	typedef b16 b4 __attribute__((ext_vector_type(4)));
	f32x4 g;
	if (s.dtype == NGP_DTYPE_F32) g = *(const f32x4*)((const float*)s.grads + i);
	else if (s.dtype == NGP_DTYPE_F16) g = __builtin_convertvector(*(const h4*)((const f16*)s.grads + i), f32x4);
	else g = __builtin_convertvector(*(const b4*)((const b16*)s.grads + i), f32x4);
	return g * s.inv_loss_scale;
}

// m <- beta m + g, and the squares of u.  In 64 bits: gradients of single precision may square to what fp32 cannot hold.  Bound by memory: 10 bytes an element of 16-bit gradients,
// 24 matrices of 768 x 768 in 25 us (5.6 TB/s).
__global__ void __launch_bounds__(256) momentum_kernel(Jobs jobs, Step s) {
	__shared__ double lds[4];
	uint32_t pid = blockIdx.x;
	const uint32_t ji = job_of(jobs, START_SUM, pid);
	const Job& j = jobs.job[ji];
	const uint32_t blocks = jobs.start[START_SUM][ji + 1] - jobs.start[START_SUM][ji];
	const uint64_t total = (uint64_t)j.rows * j.cols, step = (uint64_t)blocks * 256;
	const bool wide = ((j.offset & 3) | ((uintptr_t)s.buffer & 15) | ((uintptr_t)s.grads & (s.dtype == NGP_DTYPE_F32 ? 15 : 7))) == 0;
	const uint64_t quads = wide ? total / 4 : 0;
	double sum = 0.0;
	for (uint64_t q = (uint64_t)pid * 256 + threadIdx.x; q < quads; q += step) {
		const uint64_t i = j.offset + 4 * q;
		const f32x4 g = load_grad4(s, i), old = *(const f32x4*)(s.buffer + i);
		f32x4 m;
#pragma unroll
		for (int e = 0; e < 4; ++e) {
			m[e] = s.momentum * old[e] + g[e];
			const double u = s.nesterov ? g[e] + s.momentum * m[e] : m[e];
			sum += u * u;
		}
		*(f32x4*)(s.buffer + i) = m;
	}
	for (uint64_t i = 4 * quads + (uint64_t)pid * 256 + threadIdx.x; i < total; i += step) {
		const float g = load_grad(s, j.offset + i), m = s.momentum * s.buffer[j.offset + i] + g;
		s.buffer[j.offset + i] = m;
		const double u = s.nesterov ? g + s.momentum * m : m;
		sum += u * u;
	}
	sum = block_sum(sum, lds);
	if (threadIdx.x == 0) j.sums[pid] = sum;
}

__device__ __forceinline__ void split2(float v, f16& hi, f16& lo) { hi = (f16)v; lo = (f16)(v - (float)hi); }
__device__ __forceinline__ uint64_t split_col(uint32_t c) { return (uint64_t)(c >> 5) * 64 + (c & 31); }   // of the hi half; lo is 32 behind it

typedef f16 f16x4 __attribute__((ext_vector_type(4)));

// X_0^T in halves, zeros up to the padded width.  A workgroup takes 64 x 64 elements, through LDS where the matrix lies the other way round.  Bound by memory: 10 bytes an element,
// 24 matrices of 768 x 768 in 31 us (4.5 TB/s).
__global__ void __launch_bounds__(256) split_kernel(Jobs jobs, Step s) {
	__shared__ double lds[4];
	__shared__ float tile[64][65];   // [long][short]
	uint32_t pid = blockIdx.x;
	const uint32_t ji = job_of(jobs, START_SPLIT, pid);
	const Job& j = jobs.job[ji];
	const uint32_t blocks = jobs.start[START_SUM][ji + 1] - jobs.start[START_SUM][ji];
	double mine = 0.0;
	for (uint32_t i = threadIdx.x; i < blocks; i += 256) mine += j.sums[i];
	const double sum = block_sum(mine, lds);
	const double norm = sqrt(sum) + (double)s.eps, scale = norm == 0.0 ? 0.0 : (double)SX / norm;   // a zero update stays zero also without eps
	const uint32_t tiles_n = (j.np + 63) / 64, k0 = pid / tiles_n * 64, n0 = pid % tiles_n * 64;
	const bool turn = j.rows > j.cols;   // the matrix is X^T as it lies
#pragma unroll 4
	for (uint32_t e = threadIdx.x; e < 4096; e += 256) {   // e runs along the matrix's rows
		const uint32_t a = e >> 6, b = e & 63, k = k0 + (turn ? a : b), n = n0 + (turn ? b : a);
		const bool in = k < j.k && n < j.n;
		const uint64_t i = j.offset + (in ? (turn ? (uint64_t)k * j.cols + n : (uint64_t)n * j.cols + k) : 0);
		const float m = s.buffer[i], g = s.nesterov ? load_grad(s, i) : 0.0f;
		tile[k - k0][n - n0] = in ? (float)((double)(s.nesterov ? g + s.momentum * m : m) * scale) : 0.0f;
	}
	__syncthreads();
#pragma unroll
	for (uint32_t e = threadIdx.x; e < 1024; e += 256) {
		const uint32_t k = e >> 4, n = (e & 15) * 4;
		f16x4 hi, lo;
#pragma unroll
		for (int q = 0; q < 4; ++q) { f16 h, l; split2(tile[k][n + q], h, l); hi[q] = h; lo[q] = l; }
		if (k0 + k >= j.k || n0 + n >= j.np) continue;
		f16* p = j.xt[0] + (uint64_t)(k0 + k) * 2 * j.np + split_col(n0 + n);
		*(f16x4*)p = hi;
		*(f16x4*)(p + 32) = lo;
	}
}

// ---- products of split matrices ------------------------------------------------------------------------------------------------------------

// acc[nb][mb] = rows n0 .. of n times rows m0 .. of m (16 x 16 blocks), in steps of 32 k: 64 columns, both halves.  A ring of STAGES buffers, DMA spread between the MFMAs, counted
// waits: the scheme of mm::Product, with three MFMAs to a pair of fragments' halves.
// KC: the operands' rows have k along them (a step: 64 columns, both halves of 32 k).  RC: k is their rows (a step: 32 of them, both halves of the tile's columns).
template <int BN_, int BM_, int WN_, int WM_, int STAGES_> struct Geometry { static constexpr int BN = BN_, BM = BM_, WN = WN_, WM = WM_, STAGES = STAGES_, THREADS = 64 * WN_ * WM_; };
template <class G, int LAY>
struct SplitProduct {
	static constexpr int BN = G::BN, BM = G::BM, WN = G::WN, WM = G::WM, STAGES = G::STAGES;
	static constexpr int THREADS = G::THREADS, NB = BN / WN / 16, MB = BM / WM / 16, N = BN, M = BM, WAVES_N = WN, WAVES_M = WM;
	using NT = Tile<LAY, LAY == KC ? BN : 2 * BN, THREADS, LAY == KC ? 64 : 32>;
	using MT = Tile<LAY, LAY == KC ? BM : 2 * BM, THREADS, LAY == KC ? 64 : 32>;
	static constexpr int STAGE_BYTES = NT::BYTES + MT::BYTES, LOADS = NT::LOADS + MT::LOADS, LDS_BYTES = STAGES * STAGE_BYTES;
	static_assert(LDS_BYTES >= WN * WM * 32 * 144, "the epilogue's rows");

	// rows row0 .. + 15, half 0 (hi) or 1 (lo): lane l has row l & 15 and k = 8 (l >> 4) .. + 7
	template <class TT> static __device__ __forceinline__ i32x4 frag(const lds_char* p, int row0, int half, int lane) {
		if constexpr (LAY == RC) return TT::frag(p, (row0 >> 5) * 64 + half * 32 + (row0 & 31), lane);
		return *(const __attribute__((address_space(3))) i32x4*)(p + (row0 + (lane & 15)) * 128 + ((half * 4 + (lane >> 4)) ^ TT::swizzle(lane & 15)) * 16);
	}
	static __device__ __forceinline__ void run(f32x4 (&acc)[NB][MB], const Mat& n, const Mat& m, uint32_t n0, uint32_t m0, lds_char* lds) {   // RC: n.rows, m.rows in columns of both halves
		const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wave % WN, wm = wave / WN;
#pragma unroll
		for (int a = 0; a < NB; ++a)
#pragma unroll
			for (int b = 0; b < MB; ++b) acc[a][b] = f32x4{0, 0, 0, 0};
		NT nt;
		MT mt;
		nt.init(n, LAY == KC ? n0 : 2 * n0, 0, tid);
		mt.init(m, LAY == KC ? m0 : 2 * m0, 0, tid);
		const int steps = (int)(LAY == KC ? n.k / 64 : (n.k + 31) / 32);
		i32x4 rn, rm;
		int slot = 0;
		lds_char* to = lds;
		auto next_step = [&]() {
			rn = nt.next();
			rm = mt.next();
			to = lds + slot * STAGE_BYTES;
			slot = slot + 1 == STAGES ? 0 : slot + 1;
		};
		auto issue = [&](int i) {
			if (i < NT::LOADS) nt.issue(rn, i, to, wave);
			else mt.issue(rm, i - NT::LOADS, to + NT::BYTES, wave);
		};
		// Fragments are read a step ahead of the MFMAs that take them, and between MFMAs, as the DMA is issued: a burst of reads behind the barrier holds up every wave's MFMAs at once.
		i32x4 fm[2][2][MB], fn[2][2][NB];   // of two steps: hi, lo
		constexpr int READS = 2 * (MB + NB), COUNT = 3 * NB * MB;
		auto read = [&](int set, int d, const lds_char* p) {
			const int half = d / (MB + NB), i = d % (MB + NB);
			if (i < MB) fm[set][half][i] = frag<MT>(p + NT::BYTES, wm * (BM / WM) + i * 16, half, lane);
			else fn[set][half][i - MB] = frag<NT>(p, wn * (BN / WN) + (i - MB) * 16, half, lane);
		};
		int at = 0;
		auto step = [&](int set) {
			wait_and_sync<(STAGES - 2) * LOADS>();   // the next step has landed; this one is in registers everywhere, and its buffer free
			next_step();
			at = at + 1 == STAGES ? 0 : at + 1;
			const lds_char* p = lds + at * STAGE_BYTES;   // behind the last step: not used
			__builtin_amdgcn_sched_barrier(0);
#pragma unroll
			for (int i = 0; i < COUNT; ++i) {
				const int part = i / (NB * MB), a = i % (NB * MB) / MB, b = i % MB;
				acc[a][b] = mfma16<f16>(fn[set][part == 2][a], fm[set][part == 1][b], acc[a][b]);   // hi hi, hi lo, lo hi
#pragma unroll
				for (int d = 0; d < READS + LOADS; ++d)
					if (d * (COUNT - 2) / (READS + LOADS) == i) {
						__builtin_amdgcn_sched_barrier(0);
						if (d < READS) read(set ^ 1, d, p);
						else issue(d - READS);
						__builtin_amdgcn_sched_barrier(0);
					}
			}
			__builtin_amdgcn_sched_barrier(0);
		};
#pragma unroll
		for (int s = 0; s < STAGES; ++s) {   // the steps behind the last one read zeros
			next_step();
#pragma unroll
			for (int i = 0; i < LOADS; ++i) issue(i);
		}
		wait_and_sync<(STAGES - 1) * LOADS>();
#pragma unroll
		for (int d = 0; d < READS; ++d) read(0, d, lds);
		int s = 0;
		for (; s + 1 < steps; s += 2) {
			step(0);
			step(1);
		}
		if (s < steps) step(0);
		wait_and_sync();   // the DMA behind the last step too
	}
};
using Large = Geometry<128, 256, 2, 4, 3>;   // 144 KB of LDS
using Middle = Geometry<128, 128, 2, 2, 2>;  // 64 KB: two workgroups a CU, one's MFMAs beside the other's loads and stores
using Lone = Geometry<128, 128, 4, 2, 4>;    // 128 KB: where there is one tile a CU
using Little = Geometry<64, 64, 2, 2, 4>;    // 64 KB: two workgroups a CU

// A wave's 32 x 32 block (2 x 2 of 16) of a split matrix, through LDS of its own (32 rows of 144 bytes) into rows of 64 hi and 64 lo bytes: as it lies (rows m), or transposed (rows n)
__device__ __forceinline__ void put_split(const f32x4& v, bool turned, int nb, int mb, lds_char* lds, int lane) {   // block nb, mb of the four
	typedef __attribute__((address_space(3))) f16x4 lds_f16x4;
	typedef __attribute__((address_space(3))) f16 lds_f16;
	f16x4 hi, lo;
#pragma unroll
	for (int e = 0; e < 4; ++e) { f16 h, l; split2(v[e], h, l); hi[e] = h; lo[e] = l; }
	const int m = mb * 16 + (lane & 15), n = nb * 16 + 4 * (lane >> 4);
	if (!turned) {
		*(lds_f16x4*)(lds + m * 144 + n * 2) = hi;
		*(lds_f16x4*)(lds + m * 144 + 64 + n * 2) = lo;
	} else
#pragma unroll
		for (int e = 0; e < 4; ++e) {
			*(lds_f16*)(lds + (n + e) * 144 + m * 2) = hi[e];
			*(lds_f16*)(lds + (n + e) * 144 + 64 + m * 2) = lo[e];
		}
}
// rows row0 .. + 31 below `rows`, columns col0 .. + 31 (all below `cols` or none) of the split matrix p with rows of `pitch` elements
__device__ __forceinline__ void write_split(f16* p, uint32_t pitch, uint32_t rows, uint32_t cols, uint32_t row0, uint32_t col0, const lds_char* lds, int lane) {
	if (col0 >= cols) return;
#pragma unroll
	for (int r = 0; r < 32; r += 8) {
		const uint32_t row = row0 + r + (lane >> 3);
		const i32x4 q = *(const __attribute__((address_space(3))) i32x4*)(lds + (r + (lane >> 3)) * 144 + (lane & 7) * 16);
		if (row < rows) *(i32x4*)(p + (uint64_t)row * pitch + (uint64_t)col0 * 2 + (lane & 7) * 8) = q;
	}
}

// Square tiles on and below the diagonal, by rows; those below are written twice.
template <class G> inline uint32_t symmetric_tiles(uint32_t n) {
	static_assert(G::BN == G::BM, "square");
	const uint32_t t = (n + G::BM - 1) / G::BM;
	return t * (t + 1) / 2;
}
__device__ __forceinline__ void symmetric_tile(uint32_t pid, uint32_t& tm, uint32_t& tn) {
	for (tm = 0; pid > tm; ++tm) pid -= tm + 1;
	tn = pid;
}

// one tile of A = X X^T (POLY 0), or of B = a I + b A + c A^2 (POLY 1), from the sums in `acc`
template <class P, int POLY>
__device__ __forceinline__ void store_symmetric(const f32x4 (&acc)[P::NB][P::MB], const Job& j, uint32_t tm, uint32_t tn, lds_char* lds) {
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % P::WAVES_N, wm = wave / P::WAVES_N;
	lds_char* mine = lds + wave * (32 * 144);
	f16* const out = POLY ? j.b : j.a;
	i32x4 old[POLY ? P::NB / 2 : 1][POLY ? P::MB / 2 : 1][4];   // POLY: the tile of A, in whole rows of 32 columns, all of it under way at once
	if (POLY)
#pragma unroll
		for (int a = 0; a < P::NB; a += 2)
#pragma unroll
			for (int b = 0; b < P::MB; b += 2)
#pragma unroll
				for (int r = 0; r < 4; ++r) {
					const uint32_t n0 = tn * P::N + wn * (P::NB * 16) + a * 16, m = tm * P::M + wm * (P::MB * 16) + b * 16 + r * 8 + (lane >> 3);
					old[a / 2][b / 2][r] = i32x4{0, 0, 0, 0};
					if (m < j.n && n0 < j.np) old[a / 2][b / 2][r] = *(const i32x4*)(j.a + (uint64_t)m * 2 * j.np + (uint64_t)n0 * 2 + (lane & 7) * 8);
				}
#pragma unroll
	for (int a = 0; a < P::NB; a += 2)
#pragma unroll
		for (int b = 0; b < P::MB; b += 2) {
			if (POLY)
#pragma unroll
				for (int r = 0; r < 4; ++r) *(__attribute__((address_space(3))) i32x4*)(mine + (r * 8 + (lane >> 3)) * 144 + (lane & 7) * 16) = old[a / 2][b / 2][r];
			const uint32_t n0 = tn * P::N + wn * (P::NB * 16) + a * 16, m0 = tm * P::M + wm * (P::MB * 16) + b * 16;
			f32x4 v[2][2];
#pragma unroll
			for (int x = 0; x < 2; ++x)
#pragma unroll
				for (int y = 0; y < 2; ++y) {
					v[x][y] = acc[a + x][b + y];
					if (POLY) {
						const uint32_t m = m0 + y * 16 + (lane & 15), n = n0 + x * 16 + 4 * (lane >> 4);
						const lds_char* d = mine + (y * 16 + (lane & 15)) * 144 + (x * 16 + 4 * (lane >> 4)) * 2;
						const f16x4 hi = *(const __attribute__((address_space(3))) f16x4*)d, lo = *(const __attribute__((address_space(3))) f16x4*)(d + 64);
#pragma unroll
						for (int e = 0; e < 4; ++e) v[x][y][e] = NS_C / SA * v[x][y][e] + NS_B * ((float)hi[e] + (float)lo[e]) + (m == n + e && m < j.n ? NS_A * SA : 0.0f);
					} else v[x][y] *= SA / (SX * SX);
					put_split(v[x][y], false, x, y, mine, lane);
				}
			write_split(out, 2 * j.np, j.n, j.np, m0, n0, mine, lane);
			if (tn == tm) continue;
#pragma unroll
			for (int x = 0; x < 2; ++x)
#pragma unroll
				for (int y = 0; y < 2; ++y) put_split(v[x][y], true, x, y, mine, lane);
			write_split(out, 2 * j.np, j.n, j.np, n0, m0, mine, lane);
		}
}

// A, all of k or (a long, narrow X has few tiles) a part of it: then the sums are left as they lie in the registers, and gram_sum_kernel adds the parts in their order.
// Bound by the matrix pipes where the tiles fill the chip (two 8192 x 4096: 0.86 ms, 0.99 PFLOP/s of fp16 products, 0.97 of the tiles' work being needed), else by the latency of the
// DMA: one 1531 x 1000, 136 tiles of 64 x 64 and 48 steps, 16 us: 0.33 us a step with three of them on their way, 110 MB out of the L2s, of which 63 % is found there.
template <class G>
__global__ void __launch_bounds__(G::THREADS, (SplitProduct<G, RC>::LDS_BYTES <= 80 * 1024 ? 2 : 1)) gram_kernel(Jobs jobs, int from) {
	using P = SplitProduct<G, RC>;
	__shared__ __attribute__((aligned(1024))) char lds[P::LDS_BYTES];
	uint32_t pid = xcd_order(blockIdx.x, gridDim.x), tm, tn;
	const Job& j = jobs.job[job_of(jobs, START_GRAM, pid)];
	const uint32_t part = pid % j.parts, tile = pid / j.parts;
	symmetric_tile(tile, tm, tn);
	const uint32_t per = ((j.k + 31) / 32 + j.parts - 1) / j.parts * 32, k0 = part * per;
	const Mat mat{j.xt[from] + (uint64_t)k0 * 2 * j.np, 2ull * j.np, 2 * j.np, min(per, j.k - k0)};
	f32x4 acc[P::NB][P::MB];
	P::run(acc, mat, mat, tn * P::N, tm * P::M, lds_of(lds));
	if (j.parts == 1) { store_symmetric<P, 0>(acc, j, tm, tn, lds_of(lds)); return; }
	f32x4* q = (f32x4*)j.partial + (uint64_t)pid * (G::BN * G::BM / 4) + threadIdx.x;
#pragma unroll
	for (int i = 0; i < P::NB * P::MB; ++i) q[i * G::THREADS] = acc[i / P::MB][i % P::MB];
}
template <class G>
__global__ void __launch_bounds__(G::THREADS) gram_sum_kernel(Jobs jobs) {
	using P = SplitProduct<G, RC>;
	__shared__ __attribute__((aligned(16))) char lds[G::WN * G::WM * 32 * 144];
	uint32_t pid = blockIdx.x, tm, tn;
	const Job& j = jobs.job[job_of(jobs, START_SYM, pid)];
	if (j.parts == 1) return;
	symmetric_tile(pid, tm, tn);
	const f32x4* q = (const f32x4*)j.partial + (uint64_t)pid * j.parts * (G::BN * G::BM / 4) + threadIdx.x;
	f32x4 acc[P::NB][P::MB];
#pragma unroll
	for (int i = 0; i < P::NB * P::MB; ++i) acc[i / P::MB][i % P::MB] = q[i * G::THREADS];
#pragma unroll 4
	for (uint32_t part = 1; part < j.parts; ++part)
#pragma unroll
		for (int i = 0; i < P::NB * P::MB; ++i) acc[i / P::MB][i % P::MB] += q[part * (G::BN * G::BM / 4) + i * G::THREADS];
	store_symmetric<P, 0>(acc, j, tm, tn, lds_of(lds));
}

// B.  As gram_kernel: 0.43 ms and 13 us there
template <class G>
__global__ void __launch_bounds__(G::THREADS, (SplitProduct<G, KC>::LDS_BYTES <= 80 * 1024 ? 2 : 1)) poly_kernel(Jobs jobs) {
	using P = SplitProduct<G, KC>;
	__shared__ __attribute__((aligned(1024))) char lds[P::LDS_BYTES];
	uint32_t pid = xcd_order(blockIdx.x, gridDim.x), tm, tn;
	const Job& j = jobs.job[job_of(jobs, START_SYM, pid)];
	symmetric_tile(pid, tm, tn);
	const Mat mat{j.a, 2ull * j.np, j.n, 2 * j.np};
	f32x4 acc[P::NB][P::MB];
	P::run(acc, mat, mat, tn * P::N, tm * P::M, lds_of(lds));
	store_symmetric<P, 1>(acc, j, tm, tn, lds_of(lds));
}

// X^T <- X^T B, or (LAST) straight into the weights.  Bound by the matrix pipes: two 8192 x 4096 1.18 ms, 1.40 PFLOP/s of fp16 products; the last one, which reads and writes weights
// too, 1.5 ms.
template <class G, int LAST>
__global__ void __launch_bounds__(G::THREADS, (SplitProduct<G, KC>::LDS_BYTES <= 80 * 1024 ? 2 : 1)) apply_kernel(Jobs jobs, Step s, int from) {
	using P = SplitProduct<G, KC>;
	__shared__ __attribute__((aligned(1024))) char lds[P::LDS_BYTES];
	uint32_t pid = xcd_order(blockIdx.x, gridDim.x);
	const Job& j = jobs.job[job_of(jobs, START_APPLY, pid)];
	const uint32_t tiles_n = (j.n + P::N - 1) / P::N, tn = pid % tiles_n, tm = pid / tiles_n;
	f32x4 acc[P::NB][P::MB];
	P::run(acc, Mat{j.b, 2ull * j.np, j.n, 2 * j.np}, Mat{j.xt[from], 2ull * j.np, j.k, 2 * j.np}, tn * P::N, tm * P::M, lds_of(lds));
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % P::WAVES_N, wm = wave / P::WAVES_N;
	lds_char* mine = lds_of(lds) + wave * (32 * 144);
	const bool turn = j.rows > j.cols;
	const float keep = 1.0f - s.lr * s.decay, rate = s.lr * sqrtf(fmaxf(1.0f, (float)j.rows / (float)j.cols)) / (SA * SX);
#pragma unroll
	for (int a = 0; a < P::NB; a += 2)
#pragma unroll
		for (int b = 0; b < P::MB; b += 2) {
			const uint32_t n0 = tn * P::N + wn * (P::NB * 16) + a * 16, m0 = tm * P::M + wm * (P::MB * 16) + b * 16;
			if (!LAST) {
#pragma unroll
				for (int x = 0; x < 2; ++x)
#pragma unroll
					for (int y = 0; y < 2; ++y) put_split(acc[a + x][b + y] * (1.0f / SA), false, x, y, mine, lane);
				write_split(j.xt[1 - from], 2 * j.np, j.k, j.np, m0, n0, mine, lane);
				continue;
			}
			float w[16];
			uint64_t at[16];
			bool in[16];
#pragma unroll
			for (int i = 0; i < 16; ++i) {
				const uint32_t m = m0 + (i >> 2 & 1) * 16 + (lane & 15), n = n0 + (i >> 3) * 16 + 4 * (lane >> 4) + (i & 3);   // long, short
				in[i] = m < j.k && n < j.n;
				at[i] = j.offset + (in[i] ? (turn ? (uint64_t)m * j.cols + n : (uint64_t)n * j.cols + m) : 0);
				w[i] = s.master[at[i]];
			}
#pragma unroll
			for (int i = 0; i < 16; ++i) w[i] = keep * w[i] - rate * acc[a + (i >> 3)][b + (i >> 2 & 1)][i & 3];
			set_weights(s, at, w, in);
		}
}

// ---- a matrix in one workgroup ---------------------------------------------------------------------------------------------------------------
//
// Short side at most 64, long side at most 256 (the matrices of the framework's own networks): X^T, A and B stay in LDS in the same split layout, and the whole step is one launch
// whose time is the latency of its chain: 3 products an iteration, four barriers.  Five 64 x 64 matrices: 18 us; 76 as 17 launches of the kernels above.
struct TinyJobs { NgpMuonMatrix m[128]; };
constexpr uint32_t TINY_N = 64, TINY_K = 256;
constexpr int TINY_PITCH = 64 * 4 + 16;   // bytes of a row of 64 columns in two halves

__device__ __forceinline__ i32x4 tiny_along(const lds_char* p, int row0, int col0, int half, int lane) {   // 16 rows, 32 k along them from col0 (a multiple of 32)
	return *(const __attribute__((address_space(3))) i32x4*)(p + (row0 + (lane & 15)) * TINY_PITCH + col0 * 4 + half * 64 + (lane >> 4) * 16);
}
__device__ __forceinline__ i32x4 tiny_turned(const lds_char* p, int row0, int k0, int half, int lane) {    // 16 columns from row0, 32 k: the LDS rows from k0
	const lds_char* q = p + (k0 + 8 * (lane >> 4) + ((lane & 15) >> 2)) * TINY_PITCH + (row0 >> 5) * 128 + half * 64 + ((row0 & 31) + 4 * (lane & 3)) * 2;
	const i32x2 a = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)q));
	const i32x2 b = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(q + 4 * TINY_PITCH)));
	return i32x4{a.x, a.y, b.x, b.y};
}
__device__ __forceinline__ void tiny_put(lds_char* p, int row, int col, const f32x4& v) {   // four columns
	f16x4 hi, lo;
#pragma unroll
	for (int e = 0; e < 4; ++e) { f16 h, l; split2(v[e], h, l); hi[e] = h; lo[e] = l; }
	lds_char* q = p + row * TINY_PITCH + (col >> 5) * 128 + (col & 31) * 2;
	*(__attribute__((address_space(3))) f16x4*)q = hi;
	*(__attribute__((address_space(3))) f16x4*)(q + 64) = lo;
}
__device__ __forceinline__ f32x4 tiny_get(const lds_char* p, int row, int col) {
	const lds_char* q = p + row * TINY_PITCH + (col >> 5) * 128 + (col & 31) * 2;
	return __builtin_convertvector(*(const __attribute__((address_space(3))) f16x4*)q, f32x4) + __builtin_convertvector(*(const __attribute__((address_space(3))) f16x4*)(q + 64), f32x4);
}
__device__ __forceinline__ f32x4 mfma3(i32x4 nh, i32x4 nl, i32x4 mh, i32x4 ml, f32x4 c) {
	c = mfma16<f16>(nl, mh, c);
	c = mfma16<f16>(nh, ml, c);
	return mfma16<f16>(nh, mh, c);
}

struct TinyBlocks {   // of A and B: a wave's row of blocks and two of its four; a lane's row and first column in a block
	int m0, n0, lm, ln;
	__device__ __forceinline__ TinyBlocks(int wave, int lane) : m0(wave / 2 * 16), n0(wave % 2 * 32), lm(lane & 15), ln(4 * (lane >> 4)) {}
};
// the wave's blocks of X X^T, from 32 k_steps rows of X^T
__device__ __forceinline__ void tiny_gram(const lds_char* xt, int k_steps, const TinyBlocks& o, int lane, f32x4 (&acc)[2]) {
	acc[0] = acc[1] = f32x4{0, 0, 0, 0};
	for (int ks = 0; ks < k_steps; ++ks) {
		const i32x4 mh = tiny_turned(xt, o.m0, ks * 32, 0, lane), ml = tiny_turned(xt, o.m0, ks * 32, 1, lane);
#pragma unroll
		for (int b = 0; b < 2; ++b) acc[b] = mfma3(tiny_turned(xt, o.n0 + b * 16, ks * 32, 0, lane), tiny_turned(xt, o.n0 + b * 16, ks * 32, 1, lane), mh, ml, acc[b]);
	}
}
// A from the blocks of X X^T into `ma`, then B into `mb`; every wave of the workgroup calls it
__device__ __forceinline__ void tiny_polynomial(lds_char* ma, lds_char* mb, const TinyBlocks& o, int lane, f32x4 (&acc)[2]) {
#pragma unroll
	for (int b = 0; b < 2; ++b) tiny_put(ma, o.m0 + o.lm, o.n0 + b * 16 + o.ln, acc[b] * (SA / (SX * SX)));
	__syncthreads();
	acc[0] = acc[1] = f32x4{0, 0, 0, 0};
#pragma unroll
	for (int ks = 0; ks < 2; ++ks) {
		const i32x4 mh = tiny_along(ma, o.m0, ks * 32, 0, lane), ml = tiny_along(ma, o.m0, ks * 32, 1, lane);
#pragma unroll
		for (int b = 0; b < 2; ++b) acc[b] = mfma3(tiny_along(ma, o.n0 + b * 16, ks * 32, 0, lane), tiny_along(ma, o.n0 + b * 16, ks * 32, 1, lane), mh, ml, acc[b]);
	}
#pragma unroll
	for (int b = 0; b < 2; ++b) {
		const int row = o.m0 + o.lm, col = o.n0 + b * 16 + o.ln;
		f32x4 v = NS_C / SA * acc[b] + NS_B * tiny_get(ma, row, col);
#pragma unroll
		for (int e = 0; e < 4; ++e)
			if (row == col + e) v[e] += NS_A * SA;
		tiny_put(mb, row, col, v);
	}
	__syncthreads();
}
// rows r .. r + 15 of X^T B
__device__ __forceinline__ void tiny_apply(const lds_char* xt, const lds_char* mb, int r, int lane, f32x4 (&x)[4]) {
#pragma unroll
	for (int b = 0; b < 4; ++b) x[b] = f32x4{0, 0, 0, 0};
#pragma unroll
	for (int ks = 0; ks < 2; ++ks) {
		const i32x4 mh = tiny_along(xt, r, ks * 32, 0, lane), ml = tiny_along(xt, r, ks * 32, 1, lane);
#pragma unroll
		for (int b = 0; b < 4; ++b) x[b] = mfma3(tiny_along(mb, b * 16, ks * 32, 0, lane), tiny_along(mb, b * 16, ks * 32, 1, lane), mh, ml, x[b]);
	}
}
// the weights of those rows, r counted from the matrix's first
__device__ __forceinline__ void tiny_weights(const Step& s, uint64_t offset, uint32_t rows, uint32_t cols, uint32_t r, const TinyBlocks& o, const f32x4 (&x)[4]) {
	const bool turn = rows > cols;
	const uint32_t n = turn ? cols : rows, k = turn ? rows : cols, row = r + o.lm;
	const float keep = 1.0f - s.lr * s.decay, rate = s.lr * sqrtf(fmaxf(1.0f, (float)rows / (float)cols)) / (SA * SX);
	float w[16];
	uint64_t at[16];
	bool in[16];
#pragma unroll
	for (int i = 0; i < 16; ++i) {
		const uint32_t c = (i >> 2) * 16 + o.ln + (i & 3);
		in[i] = row < k && c < n;
		at[i] = offset + (in[i] ? (turn ? (uint64_t)row * cols + c : (uint64_t)c * cols + row) : 0);
		w[i] = s.master[at[i]];
	}
#pragma unroll
	for (int i = 0; i < 16; ++i) w[i] = keep * w[i] - rate * x[i >> 2][i & 3];
	set_weights(s, at, w, in);
}

__global__ void __launch_bounds__(512) tiny_kernel(TinyJobs jobs, Step s, uint32_t iterations) {
	__shared__ __attribute__((aligned(16))) char xt_[TINY_K * TINY_PITCH], a_[TINY_N * TINY_PITCH], b_[TINY_N * TINY_PITCH];
	__shared__ double sums[8];
	lds_char *const xt = lds_of(xt_), *const ma = lds_of(a_), *const mb = lds_of(b_);
	const NgpMuonMatrix job = jobs.m[blockIdx.x];
	const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
	const bool turn = job.rows > job.cols;                                    // the matrix lies as X^T
	const uint32_t n = turn ? job.cols : job.rows, k = turn ? job.rows : job.cols, total = job.rows * job.cols;
	const int k_steps = (int)((k + 31) / 32);
	constexpr int EACH = TINY_N * TINY_K / 512;
	float u[EACH];
	double sum = 0.0;
#pragma unroll
	for (int c = 0; c < EACH; c += 8) {   // eight loads, then eight stores
		if (c * 512 >= total) {
#pragma unroll
			for (int q = c; q < c + 8; ++q) u[q] = 0.0f;
			continue;
		}
		float old[8], g[8];
		uint64_t at[8];
#pragma unroll
		for (int q = 0; q < 8; ++q) {
			at[q] = job.offset + min((uint32_t)((c + q) * 512 + tid), total - 1);
			old[q] = s.buffer[at[q]];
		}
		load_grads(s, at, g);
#pragma unroll
		for (int q = 0; q < 8; ++q) {
			const uint32_t i = (c + q) * 512 + tid;
			const float m = s.momentum * old[q] + g[q];
			if (i < total) s.buffer[at[q]] = m;
			const double d = i < total ? (s.nesterov ? g[q] + s.momentum * m : m) : 0.0f;
			u[c + q] = (float)d;
			sum += d * d;
		}
	}
	for (int i = tid; i < k_steps * 32 * (TINY_PITCH / 16); i += 512) *(__attribute__((address_space(3))) i32x4*)(xt + i * 16) = i32x4{0, 0, 0, 0};
	for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
	if (lane == 0) sums[wave] = sum;
	__syncthreads();
	sum = sums[0];
	for (int i = 1; i < 8; ++i) sum += sums[i];
	const double norm = sqrt(sum) + (double)s.eps, scale = norm == 0.0 ? 0.0 : (double)SX / norm;
#pragma unroll
	for (int q = 0; q < EACH; ++q) {
		const uint32_t i = q * 512 + tid;
		if (q * 512 < total && i < total) {
			const uint32_t r = i / job.cols, c = i % job.cols, row = turn ? r : c, col = turn ? c : r;   // of X^T
			f16 hi, lo;
			split2((float)((double)u[q] * scale), hi, lo);
			lds_char* p = xt + row * TINY_PITCH + (col >> 5) * 128 + (col & 31) * 2;
			*(__attribute__((address_space(3))) f16*)p = hi;
			*(__attribute__((address_space(3))) f16*)(p + 64) = lo;
		}
	}
	__syncthreads();
	const TinyBlocks own(wave, lane);
	for (uint32_t it = 0; it < iterations; ++it) {
		f32x4 acc[2];
		tiny_gram(xt, k_steps, own, lane, acc);
		tiny_polynomial(ma, mb, own, lane, acc);
		f32x4 x[2][4];   // rows 16 wave .. and 128 + 16 wave .. of X^T B
#pragma unroll
		for (int h = 0; h < 2; ++h) {
			if (h * 128 + wave * 16 >= k_steps * 32) break;
			tiny_apply(xt, mb, h * 128 + wave * 16, lane, x[h]);
		}
		const bool last = it + 1 == iterations;   // a wave reads and writes its own rows of X^T alone: no barrier between
#pragma unroll
		for (int h = 0; h < 2; ++h) {
			const int r = h * 128 + wave * 16;
			if (r >= k_steps * 32) break;
			if (last) tiny_weights(s, job.offset, job.rows, job.cols, r, own, x[h]);
			else
#pragma unroll
				for (int b = 0; b < 4; ++b) tiny_put(xt, r + own.lm, b * 16 + own.ln, x[h][b] * (1.0f / SA));
		}
		__syncthreads();
	}
}
static bool is_tiny(const NgpMuonMatrix& m) { return std::min(m.rows, m.cols) <= TINY_N && std::max(m.rows, m.cols) <= TINY_K; }

// ---- a matrix of a short side up to 64, in slabs of its long one -------------------------------------------------------------------------------
//
// Between two iterations only A, 64 x 64, has to be known to all: a launch to an iteration, in which every workgroup adds the slabs' parts of A in their order, works out B for itself,
// multiplies its 128 or 256 rows of X^T and leaves their part of the next A.  Bound by the chain inside a launch, 10 us from
// the slab's and the parts' way in to the slab's way out, no gap between them: one 1640 x 24 64 us, 98 by the kernels above.
constexpr uint32_t MAX_SLABS = 32, BATCH_SLABS = 256, PART_FLOATS = TINY_N * TINY_N;
static uint32_t slab_rows(uint32_t k) { return k <= TINY_K / 2 * MAX_SLABS ? TINY_K / 2 : TINY_K; }
static uint32_t slabs_of(const NgpMuonMatrix& m) {   // 0: not in slabs
	const uint32_t k = std::max(m.rows, m.cols);
	return std::min(m.rows, m.cols) > TINY_N || k <= TINY_K || k > TINY_K * MAX_SLABS ? 0 : (k + slab_rows(k) - 1) / slab_rows(k);
}
// Only as many as a round of the chip takes, or short ones: twelve 6264 x 48 in slabs are two batches, 245 us, and 191 by the kernels above.
static bool in_slabs(uint32_t n, const NgpMuonMatrix* m) {
	uint32_t slabs = 0, most = 0;
	for (uint32_t i = 0; i < n; ++i) { slabs += slabs_of(m[i]); most = std::max(most, slabs_of(m[i])); }   // of the whole list, in whatever order: at most 2^21
	return slabs <= BATCH_SLABS || most <= MAX_SLABS / 2;
}

// it 0: X_0 and its A; it 1 ..: an iteration; the last: into the weights
__global__ void __launch_bounds__(512) slim_kernel(Jobs jobs, Step s, uint32_t it, int last) {
	__shared__ __attribute__((aligned(16))) char xt_[TINY_K * TINY_PITCH], a_[TINY_N * TINY_PITCH], b_[TINY_N * TINY_PITCH];
	__shared__ double sums[8];
	lds_char *const xt = lds_of(xt_), *const ma = lds_of(a_), *const mb = lds_of(b_);
	const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
	uint32_t slab = blockIdx.x;
	const uint32_t ji = job_of(jobs, START_GRAM, slab);
	const Job& j = jobs.job[ji];
	const uint32_t height = j.parts, r0 = slab * height, here = min(height, j.k - r0), slabs = (j.k + height - 1) / height;
	const int k_steps = (int)((here + 31) / 32);
	char* const x = (char*)j.xt[0] + (uint64_t)r0 * 256;
	f32x4* const part = (f32x4*)(j.partial + ((uint64_t)(it & 1) * slabs + slab) * PART_FLOATS) + tid;
	const TinyBlocks own(wave, lane);
	f32x4 acc[2];
	if (it == 0) {
		const uint32_t blocks = jobs.start[START_SUM][ji + 1] - jobs.start[START_SUM][ji];
		double sum = 0.0;
		for (uint32_t i = tid; i < blocks; i += 512) sum += j.sums[i];
		for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
		if (lane == 0) sums[wave] = sum;
		for (int i = tid; i < k_steps * 32 * (TINY_PITCH / 16); i += 512) *(__attribute__((address_space(3))) i32x4*)(xt + i * 16) = i32x4{0, 0, 0, 0};
		__syncthreads();
		sum = sums[0];
		for (int i = 1; i < 8; ++i) sum += sums[i];
		const double norm = sqrt(sum) + (double)s.eps, scale = norm == 0.0 ? 0.0 : (double)SX / norm;
		const bool turn = j.rows > j.cols;   // the matrix lies as X^T
#pragma unroll 8
		for (uint32_t e = tid; e < here * j.n; e += 512) {   // along the matrix's rows
			const uint32_t row = turn ? e / j.n : e % here, col = turn ? e % j.n : e / here;
			const uint64_t i = j.offset + (turn ? (uint64_t)(r0 + row) * j.cols + col : (uint64_t)col * j.cols + r0 + row);
			const float m = s.buffer[i], g = s.nesterov ? load_grad(s, i) : 0.0f;
			f16 hi, lo;
			split2((float)((double)(s.nesterov ? g + s.momentum * m : m) * scale), hi, lo);
			lds_char* p = xt + row * TINY_PITCH + (col >> 5) * 128 + (col & 31) * 2;
			*(__attribute__((address_space(3))) f16*)p = hi;
			*(__attribute__((address_space(3))) f16*)(p + 64) = lo;
		}
		__syncthreads();
	} else {
		for (int i = tid; i < k_steps * 32 * 16; i += 512) *(__attribute__((address_space(3))) i32x4*)(xt + (i >> 4) * TINY_PITCH + (i & 15) * 16) = *(const i32x4*)(x + i * 16);
		const f32x4* q = (const f32x4*)(j.partial + (uint64_t)(~it & 1) * slabs * PART_FLOATS) + tid;   // the parts that the launch before left
		acc[0] = acc[1] = f32x4{0, 0, 0, 0};
#pragma unroll 16
		for (uint32_t i = 0; i < slabs; ++i)
#pragma unroll
			for (int b = 0; b < 2; ++b) acc[b] += q[i * (PART_FLOATS / 4) + b * 512];
		tiny_polynomial(ma, mb, own, lane, acc);
#pragma unroll
		for (int h = 0; h < 2; ++h) {   // a wave reads and writes its own rows of X^T alone: no barrier between
			const int r = h * 128 + wave * 16;
			if (r >= k_steps * 32) break;
			f32x4 y[4];
			tiny_apply(xt, mb, r, lane, y);
			if (last) tiny_weights(s, j.offset, j.rows, j.cols, r0 + r, own, y);
			else
#pragma unroll
				for (int b = 0; b < 4; ++b) tiny_put(xt, r + own.lm, b * 16 + own.ln, y[b] * (1.0f / SA));
		}
		if (last) return;
		__syncthreads();
	}
	for (int i = tid; i < k_steps * 32 * 16; i += 512) *(i32x4*)(x + i * 16) = *(const __attribute__((address_space(3))) i32x4*)(xt + (i >> 4) * TINY_PITCH + (i & 15) * 16);
	tiny_gram(xt, k_steps, own, lane, acc);
#pragma unroll
	for (int b = 0; b < 2; ++b) part[b * 512] = acc[b];
}

// ---- host ------------------------------------------------------------------------------------------------------------------------------

static inline uint64_t up256(uint64_t v) { return (v + 255) & ~255ull; }

static int refuse(const char* what) { set_last_error(what, hipErrorInvalidValue); return -1; }

static const char* bad_matrices(uint32_t count, const NgpMuonMatrix* m) {
	if (count == 0) return nullptr;
	if (!m) return "no matrices";
	if (count > 65536) return "more than 65536 matrices";
	for (uint32_t i = 0; i < count; ++i) {
		if (m[i].rows < 1 || m[i].cols < 1 || m[i].rows > MAX_SIDE || m[i].cols > MAX_SIDE) return "rows and cols must be 1 .. 65536";
		if (m[i].offset > 1ull << 48) return "an offset above 2^48 elements";
		if (i && m[i].offset < m[i - 1].offset + (uint64_t)m[i - 1].rows * m[i - 1].cols) return "matrices must be in the order of their offsets and must not overlap";
	}
	return nullptr;
}

// The tile whose rounds of the chip cost least.  A round, in units of one 128 x 128 tile a CU in eight waves: two of four waves (24 of 768 x 768: 957 -> 845 us) 1.7, one 128 x 256
// 1.68 (two 8192 x 4096: 1.25 ms a launch where 128 x 128 take 1.7; not for the symmetric products: 0.87 ms both, more of a larger tile lies above the diagonal), two 64 x 64
// 0.8.  In a sweep of 16 shapes this is within 2.5 % of the best of the four (profiles/muon_tiles.txt); a step of 2000 x 2000 723 -> 657 us, 1500 x 1500 425 -> 390, 4000 x 8000 6.92 -> 6.56 ms against
// fixed bounds on the number of tiles.
enum { LITTLE_TILE, LONE_TILE, MIDDLE_TILE, LARGE_TILE };
static double rounds(uint32_t tiles, uint32_t slots) { return (double)((tiles + slots - 1) / slots); }
static int tile_for(uint32_t little, uint32_t middle, double large, double* least = nullptr) {
	const double cost[4] = {0.8 * rounds(little, 512), rounds(middle, 256), 1.7 * rounds(middle, 512), large};
	const int tile = (int)(std::min_element(cost, cost + 4) - cost);
	if (least) *least = tile == LITTLE_TILE && little <= 256 ? 0.4 : cost[tile];   // one workgroup a CU, for the estimate below
	return tile;
}
template <class G> static uint32_t apply_tiles(uint32_t n, uint32_t k) { return ((n + G::BN - 1) / G::BN) * ((k + G::BM - 1) / G::BM); }

// An iteration of a batch, estimated in microseconds: the rounds of its three products by their steps, and what starting them takes.  Within a tenth for 1 to 36 matrices of 768 x 768, 20
// and 25 of 128 x 616, 25 and 32 of 300 x 500; one 1531 x 1000 takes a fifth less.
struct Load {
	uint32_t count = 0, little_sym = 0, middle_sym = 0, little_apply = 0, middle_apply = 0, large_apply = 0;
	double long_steps = 0.0, short_steps = 0.0;   // of the symmetric tiles, summed
	void add(const NgpMuonMatrix& m) {
		const uint32_t n = std::min(m.rows, m.cols), k = std::max(m.rows, m.cols), sym = symmetric_tiles<Middle>(n);
		++count;
		little_sym += symmetric_tiles<Little>(n); middle_sym += sym;
		little_apply += apply_tiles<Little>(n, k); middle_apply += apply_tiles<Middle>(n, k); large_apply += apply_tiles<Large>(n, k);
		long_steps += (double)sym * ((k + 31) / 32); short_steps += (double)sym * ((n + 31) / 32);
	}
	double time() const {
		if (!count) return 0.0;
		double symmetric, apply;
		tile_for(little_sym, middle_sym, HUGE_VAL, &symmetric);
		tile_for(little_apply, middle_apply, 1.68 * rounds(large_apply, 256), &apply);
		return 12.0 + 0.9 * (symmetric * (long_steps + short_steps) + apply * short_steps) / middle_sym;
	}
};

// The matrices of a list that are too large for one workgroup, in batches of at most MAX_JOBS in their order: those in slabs (`slim`, at most BATCH_SLABS: more would be a second round
// of the chip), or the others, `limit` to a batch: the limit of least estimated time.  Few matrices more than fill the rounds of the chip are better a batch of their own (37 of
// 768 x 768: 24 and 13 take 1390 us, 19 and 18 1510, 36 and one 1529), few more small ones are not (25 of 128 x 616: 131 us at once, 238 as 24 and one; 32 of 300 x 500 245 and 351).
struct Batches {
	uint32_t n;
	const NgpMuonMatrix* m;
	bool slabs, slim;   // slabs: in_slabs of the list
	uint32_t first = 0, limit = MAX_JOBS;
	Batches(uint32_t n_, const NgpMuonMatrix* m_, bool slabs_, bool slim_) : n(n_), m(m_), slabs(slabs_), slim(slim_) {
		if (slim || n <= MAX_JOBS / 2) return;
		double least = HUGE_VAL;
		for (uint32_t l = MAX_JOBS; l >= MAX_JOBS / 2; --l) {
			double time = 0.0;
			uint32_t count = 0;
			Load load;
			for (uint32_t i = 0; i < n; ++i) {
				if (!mine(m[i])) continue;
				if (load.count == l) { time += load.time(); load = Load(); }
				load.add(m[i]);
				++count;
			}
			time += load.time();
			if (time < 1.02 * least) { least = std::min(least, time); limit = l; }   // the smaller one of two alike: the estimate is a little low for the largest batches
			l = std::min(l, count);   // one batch from there up
			if (l <= MAX_JOBS / 2) return;
		}
	}
	bool mine(const NgpMuonMatrix& e) const { return !is_tiny(e) && (slabs && slabs_of(e) != 0) == slim; }
	bool next(Jobs& jobs) {
		jobs.count = 0;
		for (uint32_t total = 0; first < n && jobs.count < limit; ++first) {
			if (!mine(m[first])) continue;
			if (slim && (total += slabs_of(m[first])) > BATCH_SLABS) break;
			Job& j = jobs.job[jobs.count++];
			j.offset = m[first].offset; j.rows = m[first].rows; j.cols = m[first].cols;
		}
		return jobs.count != 0;
	}
};

// their buffers in `base` (null: the size alone)
static uint64_t lay_out(Jobs& jobs, bool slim, char* base) {
	uint64_t used = 0;
	auto take = [&](uint64_t bytes) { char* p = base ? base + used : nullptr; used += up256(bytes); return p; };
	for (int kind = 0; kind < N_STARTS; ++kind) jobs.start[kind][0] = 0;
	uint32_t tiles = 0;
	for (uint32_t i = 0; i < jobs.count; ++i) tiles += symmetric_tiles<Little>(std::min(jobs.job[i].rows, jobs.job[i].cols));
	for (uint32_t i = 0; i < jobs.count; ++i) {
		Job& j = jobs.job[i];
		j.n = std::min(j.rows, j.cols); j.k = std::max(j.rows, j.cols);
		j.np = (j.n + 31) & ~31u;
		const uint32_t blocks = (uint32_t)std::min<uint64_t>(SUM_BLOCKS, ((uint64_t)j.rows * j.cols + 4095) / 4096);
		jobs.start[START_SUM][i + 1] = jobs.start[START_SUM][i] + blocks;
		if (slim) {
			j.parts = slab_rows(j.k);
			const uint32_t slabs = (j.k + j.parts - 1) / j.parts;
			j.xt[0] = (f16*)take((uint64_t)slabs * j.parts * 256);
			j.partial = (float*)take((uint64_t)2 * slabs * PART_FLOATS * 4);
			j.sums = (double*)take(blocks * 8);
			jobs.start[START_GRAM][i + 1] = jobs.start[START_GRAM][i] + slabs;
			continue;
		}
		j.xt[0] = (f16*)take((uint64_t)j.k * j.np * 4);
		j.xt[1] = (f16*)take((uint64_t)j.k * j.np * 4);
		j.a = (f16*)take((uint64_t)j.n * j.np * 4);
		j.b = (f16*)take((uint64_t)j.n * j.np * 4);
		j.sums = (double*)take(blocks * 8);
		// Few tiles: k in parts of at least 8 steps, two workgroups a CU (each holds 64 KiB of LDS).  The step of one 96 x 8192 373 -> 149 us, 256 x 4096 251 -> 152 us, 700 x 6000 (66
		// tiles) 455 -> 363 us; with 136 tiles, 1531 x 1000, it costs: 244 -> 250 us, and with a
		// short side to sum over, twenty 128 x 616: 128 -> 134 us.
		j.parts = tiles >= 128 || j.k < 768 ? 1 : std::max(1u, std::min(512 / tiles, (j.k + 31) / 32 / 8));
		const uint32_t steps = (j.k + 31) / 32, per = (steps + j.parts - 1) / j.parts;
		j.parts = (steps + per - 1) / per;
		j.partial = (float*)take(j.parts > 1 ? (uint64_t)j.parts * symmetric_tiles<Little>(j.n) * (Little::BN * Little::BM * 4) : 0);
		jobs.start[START_SPLIT][i + 1] = jobs.start[START_SPLIT][i] + ((j.np + 63) / 64) * ((j.k + 63) / 64);
	}
	return used;
}

// of the largest batch: they run one behind the other
static uint64_t workspace_of(Batches b) {
	uint64_t most = 0;
	Jobs jobs;
	while (b.next(jobs)) most = std::max(most, lay_out(jobs, b.slim, nullptr));
	return most;
}

template <class G> static uint32_t count_symmetric(Jobs& jobs) {
	for (uint32_t i = 0; i < jobs.count; ++i) {
		const uint32_t tiles = symmetric_tiles<G>(jobs.job[i].n);
		jobs.start[START_SYM][i + 1] = jobs.start[START_SYM][i] + tiles;
		jobs.start[START_GRAM][i + 1] = jobs.start[START_GRAM][i] + tiles * jobs.job[i].parts;
	}
	return jobs.start[START_SYM][jobs.count];
}
template <class G> static uint32_t count_apply(Jobs& jobs) {
	for (uint32_t i = 0; i < jobs.count; ++i) {
		const Job& j = jobs.job[i];
		jobs.start[START_APPLY][i + 1] = jobs.start[START_APPLY][i] + apply_tiles<G>(j.n, j.k);
	}
	return jobs.start[START_APPLY][jobs.count];
}

// B of the X that `from` names
template <class G> static void symmetric_products(hipStream_t st, Jobs& jobs, int from) {
	const uint32_t tiles = count_symmetric<G>(jobs), groups = jobs.start[START_GRAM][jobs.count];
	hipLaunchKernelGGL(gram_kernel<G>, dim3(groups), dim3(G::THREADS), 0, st, jobs, from);
	if (groups > tiles) hipLaunchKernelGGL(gram_sum_kernel<G>, dim3(tiles), dim3(G::THREADS), 0, st, jobs);
	hipLaunchKernelGGL(poly_kernel<G>, dim3(tiles), dim3(G::THREADS), 0, st, jobs);
}
template <class G> static void apply(hipStream_t st, Jobs& jobs, const Step& s, int from, bool last) {
	const dim3 groups(count_apply<G>(jobs));
	if (last) hipLaunchKernelGGL((apply_kernel<G, 1>), groups, dim3(G::THREADS), 0, st, jobs, s, from);
	else hipLaunchKernelGGL((apply_kernel<G, 0>), groups, dim3(G::THREADS), 0, st, jobs, s, from);
}

} // namespace muon
} // namespace ngp

using namespace ngp;

extern "C" {

uint64_t ngp_hip_muon_workspace_bytes(uint32_t n_matrices, const NgpMuonMatrix* matrices_host) {
	using namespace muon;
	if (const char* bad = bad_matrices(n_matrices, matrices_host)) { refuse(bad); return 0; }
	const bool slabs = in_slabs(n_matrices, matrices_host);
	return std::max(workspace_of(Batches(n_matrices, matrices_host, slabs, true)), workspace_of(Batches(n_matrices, matrices_host, slabs, false)));
}

int ngp_hip_muon_step(void* stream, uint32_t n_matrices, const NgpMuonMatrix* matrices_host, float learning_rate, float momentum, float weight_decay, float epsilon, int nesterov,
                      uint32_t n_iterations, float loss_scale, int dtype, const void* grads, float* master, void* params, float* momentum_buffer, void* workspace, uint64_t workspace_bytes) {
	using namespace muon;
	char msg[256];
	const char* bad = bad_matrices(n_matrices, matrices_host);
	if (!bad && (n_iterations < 1 || n_iterations > 32)) bad = "n_iterations must be 1 .. 32";
	if (!bad && !(loss_scale > 0.0f)) bad = "loss_scale must be positive";
	if (!bad && !(epsilon >= 0.0f)) bad = "epsilon must not be negative";
	if (!bad && dtype != NGP_DTYPE_F16 && dtype != NGP_DTYPE_BF16 && dtype != NGP_DTYPE_F32) bad = "dtype must be F16, BF16 or F32";
	if (!bad && dtype == NGP_DTYPE_F32 && params) bad = "dtype F32 has no params: the master copy is the parameters";
	if (!bad && n_matrices && (!grads || !master || !momentum_buffer)) bad = "null tensor";
	if (!bad && ((((uintptr_t)master | (uintptr_t)momentum_buffer) & 3) || (((uintptr_t)grads | (uintptr_t)params) & (dtype == NGP_DTYPE_F32 ? 3 : 1)))) bad = "a tensor is not aligned to its elements";
	const uint32_t n = bad ? 0 : n_matrices;
	const bool slabs = in_slabs(n, matrices_host);
	Batches slim(n, matrices_host, slabs, true), tiled(n, matrices_host, slabs, false);
	const uint64_t need = std::max(workspace_of(slim), workspace_of(tiled));
	if (!bad && need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)) bad = "workspace null, not 16-byte aligned or too small (ngp_hip_muon_workspace_bytes)";
	if (bad) { snprintf(msg, sizeof(msg), "ngp_hip_muon_step: %s", bad); return refuse(msg); }
	hipStream_t st = (hipStream_t)stream;
	const Step s{learning_rate, momentum, weight_decay, epsilon, 1.0f / loss_scale, nesterov, dtype, grads, master, params, momentum_buffer};
	for (uint32_t first = 0; first < n_matrices;) {
		TinyJobs tiny;
		uint32_t count = 0;
		for (; first < n_matrices && count < 128; ++first)
			if (is_tiny(matrices_host[first])) tiny.m[count++] = matrices_host[first];
		if (count) hipLaunchKernelGGL(tiny_kernel, dim3(count), dim3(512), 0, st, tiny, s, n_iterations);
		NGP_LAUNCH_CHECK("tiny_kernel");
	}
	Jobs jobs;
	while (slim.next(jobs)) {
		lay_out(jobs, true, (char*)workspace);
		const uint32_t c = jobs.count;
		hipLaunchKernelGGL(momentum_kernel, dim3(jobs.start[START_SUM][c]), dim3(256), 0, st, jobs, s);
		for (uint32_t it = 0; it <= n_iterations; ++it) hipLaunchKernelGGL(slim_kernel, dim3(jobs.start[START_GRAM][c]), dim3(512), 0, st, jobs, s, it, (int)(it == n_iterations));
		NGP_LAUNCH_CHECK("slim_kernel");
	}
	while (tiled.next(jobs)) {
		lay_out(jobs, false, (char*)workspace);
		const uint32_t c = jobs.count;
		hipLaunchKernelGGL(momentum_kernel, dim3(jobs.start[START_SUM][c]), dim3(256), 0, st, jobs, s);
		hipLaunchKernelGGL(split_kernel, dim3(jobs.start[START_SPLIT][c]), dim3(256), 0, st, jobs, s);
		const uint32_t little_symmetric = count_symmetric<Little>(jobs), middle_symmetric = count_symmetric<Middle>(jobs);
		const uint32_t little_apply = count_apply<Little>(jobs), middle_apply = count_apply<Middle>(jobs), large_apply = count_apply<Large>(jobs);
		const int apply_tile = tile_for(little_apply, middle_apply, 1.68 * rounds(large_apply, 256));
		int symmetric_tile = tile_for(little_symmetric, middle_symmetric, HUGE_VAL);
		for (uint32_t i = 0; i < jobs.count; ++i)
			if (jobs.job[i].parts > 1) symmetric_tile = LITTLE_TILE;   // the parts are laid out for it
		for (uint32_t i = 0; i < n_iterations; ++i) {
			const int from = (int)(i & 1);
			const bool last = i + 1 == n_iterations;
			if (symmetric_tile == MIDDLE_TILE) symmetric_products<Middle>(st, jobs, from);
			else if (symmetric_tile == LONE_TILE) symmetric_products<Lone>(st, jobs, from);
			else symmetric_products<Little>(st, jobs, from);
			if (apply_tile == LARGE_TILE) apply<Large>(st, jobs, s, from, last);
			else if (apply_tile == MIDDLE_TILE) apply<Middle>(st, jobs, s, from, last);
			else if (apply_tile == LONE_TILE) apply<Lone>(st, jobs, s, from, last);
			else apply<Little>(st, jobs, s, from, last);
		}
		NGP_LAUNCH_CHECK("ngp_hip_muon_step");
	}
	return 0;
}

} // extern "C"
