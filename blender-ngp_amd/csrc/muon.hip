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
// halves inside fp16's normal range: X is held as 2^15 X (|X_ij| <= 1.21, typically 1 / sqrt(n k)), A and B as 2^13 of themselves (spectral norms at most 1.5 and 3.5).
// Layout of such a matrix: row-major, per 32 columns 32 hi values and 32 lo values: one 64-wide step of the product core brings both halves of 32 k.
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
constexpr uint32_t MAX_JOBS = 24, MAX_SIDE = 65536, SUM_BLOCKS = 256;

struct Job {
	uint64_t offset;                    // of the matrix in the parameter vector, in elements
	uint32_t rows, cols, n, k;          // n = min, k = max of rows and cols
	uint32_t np, kp;                    // n and k up to a multiple of 32
	f16 *x, *xt[2], *a, *b;             // X [n][2 kp], its transpose [k][2 np] (two: an iteration reads one and writes the other), A and B [n][2 np]
	double* sums;
};
enum { START_SUM, START_SPLIT, START_SYM, START_APPLY, N_STARTS };
struct Jobs {
	Job job[MAX_JOBS];
	uint32_t start[N_STARTS][MAX_JOBS + 1];   // first workgroup of each job, per kind of kernel
	uint32_t count;
};

struct Step { float lr, momentum, decay, eps, inv_loss_scale; int nesterov, dtype; const void* grads; float* master; void* params; float* buffer; };

__device__ __forceinline__ uint32_t job_of(const Jobs& j, int kind, uint32_t& pid) {
	uint32_t i = 0;
	while (i + 1 < j.count && pid >= j.start[kind][i + 1]) ++i;
	pid -= j.start[kind][i];
	return i;
}
// workgroups in the order of the XCDs they run on (see matmul_mfma.cuh tile_of)
__device__ __forceinline__ uint32_t xcd_order(uint32_t pid, uint32_t total) {
	const uint32_t xcd = pid & 7, per = total >> 3, rem = total & 7;
	return xcd * per + (xcd < rem ? xcd : rem) + (pid >> 3);
}

__device__ __forceinline__ float load_grad(const Step& s, uint64_t i) {
	const float g = s.dtype == NGP_DTYPE_F32 ? ((const float*)s.grads)[i] : s.dtype == NGP_DTYPE_F16 ? (float)((const f16*)s.grads)[i] : (float)((const b16*)s.grads)[i];
	return g * s.inv_loss_scale;
}

__device__ __forceinline__ double block_sum(double v, double* lds) {   // 256 threads, a fixed order
	for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
	if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
	__syncthreads();
	v = lds[0] + lds[1] + lds[2] + lds[3];
	__syncthreads();
	return v;
}

// m <- beta m + g, and the squares of u.  In 64 bits: gradients of single precision may square to what fp32 cannot hold.
__global__ void __launch_bounds__(256) momentum_kernel(Jobs jobs, Step s) {
	__shared__ double lds[4];
	uint32_t pid = blockIdx.x;
	const uint32_t ji = job_of(jobs, START_SUM, pid);
	const Job& j = jobs.job[ji];
	const uint32_t blocks = jobs.start[START_SUM][ji + 1] - jobs.start[START_SUM][ji];
	const uint64_t total = (uint64_t)j.rows * j.cols;
	double sum = 0.0;
	for (uint64_t i = (uint64_t)pid * 256 + threadIdx.x; i < total; i += (uint64_t)blocks * 256) {
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

// X_0 in halves, in both orientations, zeros up to the padded widths.  A workgroup takes 64 x 64 elements of X.
__global__ void __launch_bounds__(256) split_kernel(Jobs jobs, Step s) {
	__shared__ double lds[4];
	__shared__ float tile[64][65];
	uint32_t pid = blockIdx.x;
	const uint32_t ji = job_of(jobs, START_SPLIT, pid);
	const Job& j = jobs.job[ji];
	const uint32_t blocks = jobs.start[START_SUM][ji + 1] - jobs.start[START_SUM][ji];
	const double sum = block_sum(threadIdx.x < blocks ? j.sums[threadIdx.x] : 0.0, lds);
	const double norm = sqrt(sum) + (double)s.eps, scale = norm == 0.0 ? 0.0 : (double)SX / norm;   // a zero update stays zero also without eps
	const uint32_t tiles_k = (j.kp + 63) / 64, m0 = pid / tiles_k * 64, n0 = pid % tiles_k * 64;
	const bool turn = j.rows > j.cols;   // X = u^T
	for (uint32_t e = threadIdx.x; e < 4096; e += 256) {   // e runs along the rows of u
		const uint32_t a = e >> 6, b = e & 63, m = m0 + (turn ? b : a), n = n0 + (turn ? a : b);
		float v = 0.0f;
		if (m < j.n && n < j.k) {
			const uint64_t i = j.offset + (turn ? (uint64_t)n * j.cols + m : (uint64_t)m * j.cols + n);
			const float buf = s.buffer[i];
			v = (float)((double)(s.nesterov ? load_grad(s, i) + s.momentum * buf : buf) * scale);
		}
		tile[m - m0][n - n0] = v;
	}
	__syncthreads();
	for (uint32_t e = threadIdx.x; e < 4096; e += 256) {
		const uint32_t m = m0 + (e >> 6), n = n0 + (e & 63);
		f16 hi, lo;
		if (m < j.n && n < j.kp) {
			split2(tile[e >> 6][e & 63], hi, lo);
			f16* p = j.x + (uint64_t)m * 2 * j.kp + split_col(n);
			p[0] = hi; p[32] = lo;
		}
		const uint32_t mt = m0 + (e & 63), nt = n0 + (e >> 6);
		if (mt < j.np && nt < j.k) {
			split2(tile[e & 63][e >> 6], hi, lo);
			f16* p = j.xt[0] + (uint64_t)nt * 2 * j.np + split_col(mt);
			p[0] = hi; p[32] = lo;
		}
	}
}

// ---- products of split matrices ------------------------------------------------------------------------------------------------------------

struct Shape { static constexpr int N = 128, M = 128, WN = 2, WM = 2, THREADS = 256; };
constexpr int BK = 64;   // 32 k, both halves
using T = Tile<KC, 128, 256, BK>;
constexpr int NB = 2, MB = 2;

// acc[nb][mb] = rows n0 .. of n times rows m0 .. of m; steps of 32 k
__device__ __forceinline__ void split_product(f32x16 (&acc)[NB][MB], const Mat& n, const Mat& m, uint32_t n0, uint32_t m0, lds_char* lds) {
	const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wave % Shape::WN, wm = wave / Shape::WN;
#pragma unroll
	for (int a = 0; a < NB; ++a)
#pragma unroll
		for (int b = 0; b < MB; ++b)
#pragma unroll
			for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.0f;
	T nt, mt;
	nt.init(n, n0, tid);
	mt.init(m, m0, tid);
	const int steps = (int)(n.k / BK);
	auto issue = [&](int stage) {
		const i32x4 rn = nt.next(), rm = mt.next();
#pragma unroll
		for (int i = 0; i < T::LOADS; ++i) {
			nt.issue(rn, i, lds + stage * 2 * T::BYTES, wave);
			mt.issue(rm, i, lds + stage * 2 * T::BYTES + T::BYTES, wave);
		}
	};
	issue(0);
	for (int s = 0; s < steps; ++s) {
		wait_and_sync();
		if (s + 1 < steps) issue((s + 1) & 1);
		const lds_char* p = lds + (s & 1) * 2 * T::BYTES;
#pragma unroll
		for (int ks = 0; ks < 2; ++ks) {
			i32x4 nh[NB], nl[NB], mh[MB], ml[MB];
#pragma unroll
			for (int b = 0; b < NB; ++b) { nh[b] = T::frag32(p, wn * 64 + b * 32, ks, lane); nl[b] = T::frag32(p, wn * 64 + b * 32, ks + 2, lane); }
#pragma unroll
			for (int b = 0; b < MB; ++b) { mh[b] = T::frag32(p + T::BYTES, wm * 64 + b * 32, ks, lane); ml[b] = T::frag32(p + T::BYTES, wm * 64 + b * 32, ks + 2, lane); }
#pragma unroll
			for (int a = 0; a < NB; ++a)
#pragma unroll
				for (int b = 0; b < MB; ++b) {
					acc[a][b] = mfma<f16>(nl[a], mh[b], acc[a][b]);
					acc[a][b] = mfma<f16>(nh[a], ml[b], acc[a][b]);
					acc[a][b] = mfma<f16>(nh[a], mh[b], acc[a][b]);
				}
		}
	}
}

typedef f16 f16x4 __attribute__((ext_vector_type(4)));

// a 32 x 32 block into a split matrix, as it lies (row m) and / or transposed (row n); lane layout: matmul_mfma.cuh store_rows
__device__ __forceinline__ void store_split(const f32x16& v, f16* p, uint32_t cols2, uint32_t rows, uint32_t cols, f16* pt, uint32_t colst2, uint32_t rowst, uint32_t colst, uint32_t n0, uint32_t m0, int lane) {
	const uint32_t m = m0 + (lane & 31);
#pragma unroll
	for (int q = 0; q < 4; ++q) {
		const uint32_t n = n0 + 8 * q + 4 * (lane >> 5);
		f16x4 hi, lo;
#pragma unroll
		for (int e = 0; e < 4; ++e) { f16 h, l; split2(v[4 * q + e], h, l); hi[e] = h; lo[e] = l; }
		if (p && m < rows && n < cols) {   // cols is a multiple of 32: a quad never straddles it
			f16* d = p + (uint64_t)m * cols2 + split_col(n);
			*(f16x4*)d = hi; *(f16x4*)(d + 32) = lo;
		}
		if (pt && m < colst)
#pragma unroll
			for (int e = 0; e < 4; ++e)
				if (n + e < rowst) {
					f16* d = pt + (uint64_t)(n + e) * colst2 + split_col(m);
					d[0] = hi[e]; d[32] = lo[e];
				}
	}
}

// A = X X^T (POLY 0), or B = a I + b A + c A^2 (POLY 1): tiles on and below the diagonal
template <int POLY>
__global__ void __launch_bounds__(256, 2) symmetric_kernel(Jobs jobs) {
	__shared__ __attribute__((aligned(1024))) char lds[4 * T::BYTES];
	uint32_t pid = xcd_order(blockIdx.x, gridDim.x);
	const Job& j = jobs.job[job_of(jobs, START_SYM, pid)];
	uint32_t tm = (uint32_t)((sqrtf(8.0f * pid + 1.0f) - 1.0f) * 0.5f);
	while (tm * (tm + 1) / 2 > pid) --tm;
	while ((tm + 1) * (tm + 2) / 2 <= pid) ++tm;
	const uint32_t tn = pid - tm * (tm + 1) / 2;
	const uint32_t width = 2 * (POLY ? j.np : j.kp);
	const Mat mat{POLY ? j.a : j.x, width, j.n, width};
	f32x16 acc[NB][MB];
	split_product(acc, mat, mat, tn * 128, tm * 128, lds_of(lds));
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % Shape::WN, wm = wave / Shape::WN;
#pragma unroll
	for (int a = 0; a < NB; ++a)
#pragma unroll
		for (int b = 0; b < MB; ++b) {
			const uint32_t n0 = tn * 128 + wn * 64 + a * 32, m0 = tm * 128 + wm * 64 + b * 32, m = m0 + (lane & 31);
			f32x16 v;
#pragma unroll
			for (int q = 0; q < 4; ++q) {
				const uint32_t n = n0 + 8 * q + 4 * (lane >> 5);
				f16x4 hi = {0, 0, 0, 0}, lo = {0, 0, 0, 0};
				if (POLY && m < j.n && n < j.np) {
					const f16* d = j.a + (uint64_t)m * 2 * j.np + split_col(n);
					hi = *(const f16x4*)d; lo = *(const f16x4*)(d + 32);
				}
#pragma unroll
				for (int e = 0; e < 4; ++e) {
					if (POLY) v[4 * q + e] = NS_C / SA * acc[a][b][4 * q + e] + NS_B * ((float)hi[e] + (float)lo[e]) + (m == n + e && m < j.n ? NS_A * SA : 0.0f);
					else v[4 * q + e] = acc[a][b][4 * q + e] * (SA / (SX * SX));
				}
			}
			f16* const out = POLY ? j.b : j.a;
			store_split(v, out, 2 * j.np, j.n, j.np, tm != tn ? out : nullptr, 2 * j.np, j.n, j.np, n0, m0, lane);
		}
}

// X <- B X: into both orientations, or (LAST) straight into the weights
template <int LAST>
__global__ void __launch_bounds__(256, 2) apply_kernel(Jobs jobs, Step s, int from) {
	__shared__ __attribute__((aligned(1024))) char lds[4 * T::BYTES];
	uint32_t pid = xcd_order(blockIdx.x, gridDim.x);
	const Job& j = jobs.job[job_of(jobs, START_APPLY, pid)];
	const uint32_t tiles_m = (j.n + 127) / 128, tm = pid % tiles_m, tn = pid / tiles_m;
	f32x16 acc[NB][MB];
	split_product(acc, Mat{j.xt[from], 2ull * j.np, j.k, 2 * j.np}, Mat{j.b, 2ull * j.np, j.n, 2 * j.np}, tn * 128, tm * 128, lds_of(lds));
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % Shape::WN, wm = wave / Shape::WN;
	const bool turn = j.rows > j.cols;
	const float keep = 1.0f - s.lr * s.decay, rate = s.lr * sqrtf(fmaxf(1.0f, (float)j.rows / (float)j.cols)) / (SA * SX);
#pragma unroll
	for (int a = 0; a < NB; ++a)
#pragma unroll
		for (int b = 0; b < MB; ++b) {
			const uint32_t n0 = tn * 128 + wn * 64 + a * 32, m0 = tm * 128 + wm * 64 + b * 32, m = m0 + (lane & 31);
			if (!LAST) {
				f32x16 v;
#pragma unroll
				for (int i = 0; i < 16; ++i) v[i] = acc[a][b][i] * (1.0f / SA);
				store_split(v, j.x, 2 * j.kp, j.n, j.kp, j.xt[1 - from], 2 * j.np, j.k, j.np, n0, m0, lane);
				continue;
			}
			if (m >= j.n) continue;
#pragma unroll
			for (int i = 0; i < 16; ++i) {
				const uint32_t n = n0 + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
				if (n >= j.k) continue;
				const uint64_t at = j.offset + (turn ? (uint64_t)n * j.cols + m : (uint64_t)m * j.cols + n);
				const float w = keep * s.master[at] - rate * acc[a][b][i];
				s.master[at] = w;
				if (s.params) {
					if (s.dtype == NGP_DTYPE_F16) ((f16*)s.params)[at] = (f16)w;
					else ((b16*)s.params)[at] = (b16)w;
				}
			}
		}
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

// the buffers of matrices [first, first + jobs.count) in `base` (null: the size alone)
static uint64_t lay_out(Jobs& jobs, const NgpMuonMatrix* m, char* base) {
	uint64_t used = 0;
	auto take = [&](uint64_t bytes) { char* p = base ? base + used : nullptr; used += up256(bytes); return p; };
	for (int kind = 0; kind < N_STARTS; ++kind) jobs.start[kind][0] = 0;
	for (uint32_t i = 0; i < jobs.count; ++i) {
		Job& j = jobs.job[i];
		j.offset = m[i].offset; j.rows = m[i].rows; j.cols = m[i].cols;
		j.n = std::min(j.rows, j.cols); j.k = std::max(j.rows, j.cols);
		j.np = (j.n + 31) & ~31u; j.kp = (j.k + 31) & ~31u;
		const uint32_t blocks = (uint32_t)std::min<uint64_t>(SUM_BLOCKS, ((uint64_t)j.rows * j.cols + 4095) / 4096);
		j.x = (f16*)take((uint64_t)j.n * j.kp * 4);
		j.xt[0] = (f16*)take((uint64_t)j.k * j.np * 4);
		j.xt[1] = (f16*)take((uint64_t)j.k * j.np * 4);
		j.a = (f16*)take((uint64_t)j.n * j.np * 4);
		j.b = (f16*)take((uint64_t)j.n * j.np * 4);
		j.sums = (double*)take(blocks * 8);
		const uint32_t tn = (j.n + 127) / 128, tk = (j.k + 127) / 128;
		const uint32_t n[N_STARTS] = {blocks, ((j.np + 63) / 64) * ((j.kp + 63) / 64), tn * (tn + 1) / 2, tn * tk};
		for (int kind = 0; kind < N_STARTS; ++kind) jobs.start[kind][i + 1] = jobs.start[kind][i] + n[kind];
	}
	return used;
}

} // namespace muon
} // namespace ngp

using namespace ngp;

extern "C" {

uint64_t ngp_hip_muon_workspace_bytes(uint32_t n_matrices, const NgpMuonMatrix* matrices_host) {
	using namespace muon;
	if (const char* bad = bad_matrices(n_matrices, matrices_host)) { refuse(bad); return 0; }
	uint64_t most = 0;
	Jobs jobs;
	for (uint32_t first = 0; first < n_matrices; first += MAX_JOBS) {
		jobs.count = std::min(MAX_JOBS, n_matrices - first);
		most = std::max(most, lay_out(jobs, matrices_host + first, nullptr));
	}
	return most;
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
	if (!bad && n_matrices && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < ngp_hip_muon_workspace_bytes(n_matrices, matrices_host))) bad = "workspace null, not 16-byte aligned or too small (ngp_hip_muon_workspace_bytes)";
	if (bad) { snprintf(msg, sizeof(msg), "ngp_hip_muon_step: %s", bad); return refuse(msg); }
	hipStream_t st = (hipStream_t)stream;
	const Step s{learning_rate, momentum, weight_decay, epsilon, 1.0f / loss_scale, nesterov, dtype, grads, master, params, momentum_buffer};
	for (uint32_t first = 0; first < n_matrices; first += MAX_JOBS) {
		Jobs jobs;
		jobs.count = std::min(MAX_JOBS, n_matrices - first);
		lay_out(jobs, matrices_host + first, (char*)workspace);
		const uint32_t c = jobs.count;
		hipLaunchKernelGGL(momentum_kernel, dim3(jobs.start[START_SUM][c]), dim3(256), 0, st, jobs, s);
		hipLaunchKernelGGL(split_kernel, dim3(jobs.start[START_SPLIT][c]), dim3(256), 0, st, jobs, s);
		for (uint32_t i = 0; i < n_iterations; ++i) {
			hipLaunchKernelGGL(symmetric_kernel<0>, dim3(jobs.start[START_SYM][c]), dim3(256), 0, st, jobs);
			hipLaunchKernelGGL(symmetric_kernel<1>, dim3(jobs.start[START_SYM][c]), dim3(256), 0, st, jobs);
			if (i + 1 < n_iterations) hipLaunchKernelGGL(apply_kernel<0>, dim3(jobs.start[START_APPLY][c]), dim3(256), 0, st, jobs, s, (int)(i & 1));
			else hipLaunchKernelGGL(apply_kernel<1>, dim3(jobs.start[START_APPLY][c]), dim3(256), 0, st, jobs, s, (int)(i & 1));
		}
		NGP_LAUNCH_CHECK("ngp_hip_muon_step");
	}
	return 0;
}

} // extern "C"
