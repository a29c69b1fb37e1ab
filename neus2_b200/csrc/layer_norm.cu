// Layer norm over rows of any width, forward and backward.
//
// A group of TPR threads owns a row at a time and keeps it in registers: one read, one write per value.  Groups of up to a warp
// reduce with shuffles, wider ones through shared memory behind a barrier of their own; blocks are persistent, so gamma and beta
// (and in the backward pass the sums for their gradients) stay on the SM over all rows of a group.  The variance is the mean square
// of the centred row, not a difference of sums.
//
// Bound by memory where rows are wide (forward, 16384 rows of 4096 bf16: 55 us, 4.9 TB/s), by the instructions around a row where they are
// short (262144 rows of 64 fp16: 14.3 us, 4.8 TB/s) and by launches and the join where they are few (backward, 8192 rows of 1024 bf16 with
// a skip connection: 19.9 us of which the join takes 3.5; 33 rows of 1111 fp32: 4.3 us).
#include <type_traits>

#include "dense.cuh"

namespace n2b {
namespace ln {

static __device__ uint32_t g_error;  // bit 0: a bounded wait ran out

// VEC entries moved by one access: 16 bytes, or one entry where rows do not start on 16-byte boundaries.
template <typename T, int VEC>
struct Pack;
template <>
struct Pack<float, 4> {
	using Raw = float4;
	static __device__ __forceinline__ void get(const Raw& r, float (&v)[4]) { v[0] = r.x, v[1] = r.y, v[2] = r.z, v[3] = r.w; }
	static __device__ __forceinline__ Raw put(const float (&v)[4]) { return make_float4(v[0], v[1], v[2], v[3]); }
};
template <>
struct Pack<__half, 8> {
	using Raw = uint4;
	static __device__ __forceinline__ void get(const Raw& r, float (&v)[8]) {
		const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
		for (int i = 0; i < 4; ++i) {
			const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
			v[2 * i] = f.x, v[2 * i + 1] = f.y;
		}
	}
	static __device__ __forceinline__ Raw put(const float (&v)[8]) {
		uint32_t w[4];
#pragma unroll
		for (int i = 0; i < 4; ++i) {
			const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
			w[i] = *reinterpret_cast<const uint32_t*>(&h);
		}
		return make_uint4(w[0], w[1], w[2], w[3]);
	}
};
template <>
struct Pack<__nv_bfloat16, 8> {
	using Raw = uint4;
	static __device__ __forceinline__ void get(const Raw& r, float (&v)[8]) {
		const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
		for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
	}
	static __device__ __forceinline__ Raw put(const float (&v)[8]) {
		uint32_t w[4];
#pragma unroll
		for (int i = 0; i < 4; ++i) {
			const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
			w[i] = *reinterpret_cast<const uint32_t*>(&h);
		}
		return make_uint4(w[0], w[1], w[2], w[3]);
	}
};
template <typename T>
struct Pack<T, 1> {
	using Raw = T;
	static __device__ __forceinline__ void get(const Raw& r, float (&v)[1]) { v[0] = to_f(r); }
	static __device__ __forceinline__ Raw put(const float (&v)[1]) { return from_f<T>(v[0]); }
};

// Makes the compiler forget what it knows about a packed value: it unpacks it again where it is used next, instead of keeping the
// unpacked (or centred) entries of a whole row in registers over a reduction.
__device__ __forceinline__ void forget(uint4& v) { asm volatile("" : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w)); }
__device__ __forceinline__ void forget(float4& v) { asm volatile("" : "+f"(v.x), "+f"(v.y), "+f"(v.z), "+f"(v.w)); }
__device__ __forceinline__ void forget(float& v) { asm volatile("" : "+f"(v)); }
template <typename H>
__device__ __forceinline__ void forget(H& v) { asm volatile("" : "+h"(*reinterpret_cast<uint16_t*>(&v))); }

template <typename Raw>
__device__ __forceinline__ Raw zero() { return Raw{}; }
template <>
__device__ __forceinline__ __half zero<__half>() { return __ushort_as_half(0); }
template <>
__device__ __forceinline__ __nv_bfloat16 zero<__nv_bfloat16>() { return __ushort_as_bfloat16(0); }

__device__ __forceinline__ float param_at(const void* p, uint32_t dtype, uint32_t c) {
	if (dtype == NEUS2B_F32) return ((const float*)p)[c];
	return dtype == NEUS2B_F16 ? to_f(((const __half*)p)[c]) : to_f(((const __nv_bfloat16*)p)[c]);
}

// Sums over the TPR threads of a group, in a fixed order, the same values in all of them.  s: shared memory of the group, [2][TPR / 32];
// `turn` alternates so that one barrier per sum is enough.
template <int TPR>
__device__ __forceinline__ float group_sum(float a) {
#pragma unroll
	for (int o = (TPR < 32 ? TPR : 32) / 2; o; o >>= 1) a += __shfl_xor_sync(~0u, a, o);
	return a;
}
template <int TPR>
__device__ __forceinline__ float group_sum(float a, float2* s, int group, int& turn) {
	a = group_sum<TPR>(a);
	if (TPR > 32) {
		constexpr int W = TPR / 32;
		float2* t = s + turn * W;
		turn ^= 1;
		if ((threadIdx.x & 31) == 0) t[(threadIdx.x % TPR) >> 5].x = a;
		asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(TPR) : "memory");
		a = 0.f;
#pragma unroll
		for (int w = 0; w < W; ++w) a += t[w].x;
	}
	return a;
}
template <int TPR>
__device__ __forceinline__ void group_sums(float& a, float& b, float2* s, int group, int& turn) {
	a = group_sum<TPR>(a);
	b = group_sum<TPR>(b);
	if (TPR > 32) {
		constexpr int W = TPR / 32;
		float2* t = s + turn * W;
		turn ^= 1;
		if ((threadIdx.x & 31) == 0) t[(threadIdx.x % TPR) >> 5] = make_float2(a, b);
		asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(TPR) : "memory");
		a = b = 0.f;
#pragma unroll
		for (int w = 0; w < W; ++w) a += t[w].x, b += t[w].y;
	}
}

// gamma or beta of the group's columns in shared memory: entry (access k, thread t, i) of a row is the row's column (k TPR + t) VEC + i; four
// consecutive ones lie together and the threads' fours side by side, so that a warp's reads do not collide.
template <int VEC, int TPR>
__device__ __forceinline__ int param_slot(int k, int t, int i) {
	constexpr int Q = VEC < 4 ? VEC : 4;
	return ((k * (VEC / Q) + i / Q) * TPR + t) * Q + i % Q;
}
template <int VEC, int TPR, int VPT>
__device__ __forceinline__ void stage_param(float* s, const void* p, uint32_t dtype, uint32_t W, int threads) {
	for (int c = threadIdx.x; c < VEC * TPR * VPT; c += threads) {
		const int u = c / VEC;
		s[param_slot<VEC, TPR>(u / TPR, u % TPR, c % VEC)] = p && (uint32_t)c < W ? param_at(p, dtype, c) : 0.f;
	}
}
template <int VEC, int TPR>
__device__ __forceinline__ void staged(const float* s, int k, int t, float (&v)[VEC]) {
	if (VEC >= 4) {
#pragma unroll
		for (int q = 0; q < VEC / 4; ++q) {
			const float4 f = *reinterpret_cast<const float4*>(s + param_slot<VEC, TPR>(k, t, 4 * q));
			v[4 * q] = f.x, v[4 * q + 1 < VEC ? 4 * q + 1 : 0] = f.y, v[4 * q + 2 < VEC ? 4 * q + 2 : 0] = f.z, v[4 * q + 3 < VEC ? 4 * q + 3 : 0] = f.w;
		}
	} else {
#pragma unroll
		for (int i = 0; i < VEC; ++i) v[i] = s[param_slot<VEC, TPR>(k, t, i)];
	}
}

// ---- rows on their way: every group has a ring of `depth` rows in shared memory that bulk copies fill ahead of it
__device__ __forceinline__ uint32_t sptr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
	asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void init_barrier(uint32_t bar) {
	asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;\n\tfence.mbarrier_init.release.cluster;" ::"r"(bar) : "memory");
}
// both addresses on 16-byte boundaries, bytes a multiple of 16
__device__ __forceinline__ void copy_row(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
	asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// `given_up`: set in shared memory by the first thread of the block whose wait ran out.  From there on the block waits for no row for long,
// orders none, and goes on with what is there, through the barriers that its other threads wait at: the call's results are void, and the
// error flag says so.
__device__ __forceinline__ void wait_row(uint32_t bar, uint32_t parity, volatile uint32_t& given_up) {
	if (wait_phase(bar, parity, [&] { return given_up != 0; })) return;
	given_up = 1;
	atomicOr(&g_error, 1u);
}
template <int TPR>
__device__ __forceinline__ void group_barrier(int group) {
	if (TPR > 32) asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(TPR) : "memory");
	else __syncwarp();
}

// Up to 16 (8) entries a thread, gamma and beta stay in registers and the next row is fetched ahead; above that they are read from shared
// memory, the registers hold the packed row, and the rows of the SM's other warps are fetch-ahead enough.
template <typename T, int VEC, int TPR, int VPT, bool RING>
struct Forward {
	static constexpr bool kStaged = VEC * VPT > (RING || VEC == 1 ? 8 : 16);
	static constexpr int kWords = VPT * (VEC * (int)sizeof(T) > 4 ? VEC * (int)sizeof(T) / 4 : 1);  // registers of a packed row
	static constexpr int kThreads = !RING ? 256 : TPR == 64 ? 768 : 1024, kGroups = kThreads / TPR;  // (a group's barrier is one of 15)
	static constexpr int kBlocks = RING ? 1 : !kStaged && VEC * VPT > 8 ? 3 : kWords <= 16 ? 4 : kWords <= 32 ? 3 : 2;
};

template <typename T, int VEC, int TPR, int VPT, bool RING>
__global__ void __launch_bounds__(Forward<T, VEC, TPR, VPT, RING>::kThreads, Forward<T, VEC, TPR, VPT, RING>::kBlocks)
    forward_kernel(neus2b_layer_norm_desc d, int depth, const T* x, uint64_t x_ld, const void* __restrict__ gamma, const void* __restrict__ beta, T* y, uint64_t y_ld,
                   float* __restrict__ mean_out, float* __restrict__ rstd_out) {
	using P = Pack<T, VEC>;
	using Raw = typename P::Raw;
	using F = Forward<T, VEC, TPR, VPT, RING>;
	constexpr int G = F::kGroups;
	constexpr bool kAhead = !F::kStaged && !RING;
	constexpr int kMaxDepth = 4;
	__shared__ uint64_t bars[RING ? G * kMaxDepth : 1];
	__shared__ volatile uint32_t given_up;
	__shared__ float2 sums[G][2 * (TPR > 32 ? TPR / 32 : 1)];
	extern __shared__ float4 params4[];  // kStaged: gamma, beta; RING: the rings
	float* const sg = reinterpret_cast<float*>(params4);
	float* const sb = sg + VEC * TPR * VPT;
	const int group = threadIdx.x / TPR, t = threadIdx.x % TPR;
	const uint32_t W = d.width;
	const float inv_w = 1.f / (float)W;
	let_next_start();
	wait_for_previous();
	float ga[F::kStaged ? 1 : VPT * VEC], be[F::kStaged ? 1 : VPT * VEC];
	if (F::kStaged) {
		stage_param<VEC, TPR, VPT>(sg, gamma, d.param_dtype, W, F::kThreads);
		stage_param<VEC, TPR, VPT>(sb, beta, d.param_dtype, W, F::kThreads);
		__syncthreads();
	} else {
#pragma unroll
		for (int k = 0; k < VPT * VEC; ++k) {
			const uint32_t c = ((k / VEC) * TPR + t) * VEC + k % VEC;
			ga[F::kStaged ? 0 : k] = c < W ? param_at(gamma, d.param_dtype, c) : 0.f;
			be[F::kStaged ? 0 : k] = c < W && beta ? param_at(beta, d.param_dtype, c) : 0.f;
		}
	}
	Raw cur[VPT], ahead[kAhead ? VPT : 1];
	auto fetch = [&](Raw* raw, const T* row, bool there) {
#pragma unroll
		for (int k = 0; k < VPT; ++k) raw[k] = there && (k * TPR + t) * VEC < W ? *reinterpret_cast<const Raw*>(row + k * TPR * VEC) : zero<Raw>();
	};
	int turn = 0, slot = 0;
	uint32_t parity = 0, r = blockIdx.x * G + group;
	const uint32_t step = gridDim.x * G;
	const uint32_t row_bytes = W * (uint32_t)sizeof(T);
	unsigned char* const ring = reinterpret_cast<unsigned char*>(params4) + (F::kStaged ? 2 * VEC * TPR * VPT * sizeof(float) : 0) + (size_t)group * depth * row_bytes;
	const T* xp = x + (uint64_t)r * x_ld + t * VEC;  // the thread's first access of the row, and of the row it writes
	T* yp = y + (uint64_t)r * y_ld + t * VEC;
	const uint64_t x_step = (uint64_t)step * x_ld, y_step = (uint64_t)step * y_ld;
	if (kAhead) fetch(ahead, xp, r < d.n);
	if (RING && threadIdx.x == 0) given_up = 0;
	if (RING && t == 0) {
		for (int i = 0; i < depth; ++i) init_barrier(sptr(&bars[group * kMaxDepth + i]));
		for (int i = 0; i < depth; ++i) {
			const uint64_t row = (uint64_t)r + (uint64_t)i * step;
			if (row >= d.n) break;
			const uint32_t bar = sptr(&bars[group * kMaxDepth + i]);
			expect_bytes(bar, row_bytes);
			copy_row(sptr(ring + (size_t)i * row_bytes), x + row * x_ld, row_bytes, bar);
		}
	}
	if (RING) __syncthreads();
	// every group of the block runs the same number of rounds: the shuffles of narrow groups take the whole warp
	for (uint32_t r0 = blockIdx.x * G; r0 < d.n; r0 += step, r += step, xp += x_step, yp += y_step) {
		if (kAhead) {
#pragma unroll
			for (int k = 0; k < VPT; ++k) cur[k] = ahead[kAhead ? k : 0];
			fetch(ahead, xp + x_step, (uint64_t)r + step < d.n);
		} else if (RING) {
			const uint32_t bar = sptr(&bars[group * kMaxDepth + slot]);
			unsigned char* const row = ring + (size_t)slot * row_bytes;
			if (r < d.n) wait_row(bar, parity, given_up);
#pragma unroll
			for (int k = 0; k < VPT; ++k) {  // (a group that has no row left computes on an old one and stores nothing)
				const uint32_t c = (k * TPR + t) * VEC;
				cur[k] = c < W ? *reinterpret_cast<const Raw*>(row + c * sizeof(T)) : zero<Raw>();
			}
			group_barrier<TPR>(group);  // the row is in registers: its place is free
			const uint64_t next = (uint64_t)r + (uint64_t)depth * step;
			if (t == 0 && next < d.n && !given_up) {
				expect_bytes(bar, row_bytes);
				copy_row(sptr(row), x + next * x_ld, row_bytes, bar);
			}
			if (++slot == depth) slot = 0, parity ^= 1u;
		} else {
			fetch(cur, xp, r < d.n);
		}
		float s = 0.f;
#pragma unroll
		for (int k = 0; k < VPT; ++k) {
			float e[VEC];
			P::get(cur[k], e);
#pragma unroll
			for (int i = 0; i < VEC; ++i) s += e[i];
		}
		s = group_sum<TPR>(s, sums[group], group, turn);
		float mean = s * inv_w;
		mean = fmaf(fmaf(-mean, (float)W, s), inv_w, mean);  // the quotient, corrected by what the product with 1 / W left
		float q = 0.f;
#pragma unroll
		for (int k = 0; k < VPT; ++k) {
			if (F::kStaged) forget(cur[k]);
			float e[VEC], part = 0.f;
			P::get(cur[k], e);
#pragma unroll
			for (int i = 0; i < VEC; ++i) part = fmaf(e[i] - mean, e[i] - mean, part);
			if ((k * TPR + t) * VEC < W) q += part;  // an access lies inside the row or outside of it
		}
		q = group_sum<TPR>(q, sums[group], group, turn);
		const float rstd = rsqrtf(fmaf(q, inv_w, d.epsilon));
		if (F::kStaged) asm volatile("" ::: "memory");  // gamma and beta are read again for every row, not kept in registers
		if (r < d.n) {
#pragma unroll
			for (int k = 0; k < VPT; ++k) {
				const uint32_t c = (k * TPR + t) * VEC;
				float e[VEC], g[VEC], b[VEC];
				if (F::kStaged) forget(cur[k]);
				P::get(cur[k], e);
				if (F::kStaged) {
					staged<VEC, TPR>(sg, k, t, g);
					staged<VEC, TPR>(sb, k, t, b);
				}
#pragma unroll
				for (int i = 0; i < VEC; ++i)
					e[i] = fmaf((e[i] - mean) * rstd, F::kStaged ? g[i] : ga[F::kStaged ? 0 : k * VEC + i], F::kStaged ? b[i] : be[F::kStaged ? 0 : k * VEC + i]);
				if (c < W) *reinterpret_cast<Raw*>(yp + k * TPR * VEC) = P::put(e);
			}
			if (mean_out && t == 0) mean_out[r] = mean, rstd_out[r] = rstd;
		}
	}
}

// Up to so many rows are one cluster's, which needs neither a second launch nor a workspace: such a call is bound by the host (32 rows of 1111
// fp32: 14.8 us of its time, two launches 19.5; on the device 6.6 us and 4.2, 32 rows of 8192 bf16 12.8 and 16.4).
constexpr uint32_t kFewRows = 32, kCluster = 8;

template <int TPR, int E, bool RING>
struct Backward {
	static constexpr int kThreads = RING ? (E <= 8 ? 1024 : 512) : TPR > 128 ? TPR : 128, kGroups = kThreads / TPR;
	static constexpr int kBlocks = (E <= 8 ? 1024 : 512) / kThreads;
	static constexpr int kGrid = kSMs * kBlocks;
};

// partial: [gridDim.x][2][width], the block's sums for dgamma and dbeta; or null, and the grid is one cluster whose blocks keep their sums at
// byte `sums_at` of their shared memory and join them there.  A block adds its groups' sums in order.  The next
// row's statistics are fetched ahead like the row itself.
template <typename T, int VEC, int TPR, int VPT, bool RING>
__global__ void __launch_bounds__(Backward<TPR, VEC * VPT, RING>::kThreads, Backward<TPR, VEC * VPT, RING>::kBlocks)
    backward_kernel(neus2b_layer_norm_desc d, int depth, const T* __restrict__ x, uint64_t x_ld, const void* __restrict__ gamma, const float* __restrict__ mean,
                    const float* __restrict__ rstd, const T* dy, uint64_t dy_ld, const T* skip, uint64_t skip_ld, T* dx, uint64_t dx_ld,
                    float* __restrict__ partial, uint32_t sums_at, float* dgamma, float* dbeta, int accumulate) {
	using P = Pack<T, VEC>;
	using Raw = typename P::Raw;
	constexpr int E = VPT * VEC;
	using B = Backward<TPR, E, RING>;
	constexpr int kMaxDepth = 4;
	__shared__ uint64_t bars[RING ? B::kGroups * kMaxDepth : 1];
	__shared__ volatile uint32_t given_up;
	constexpr int G = B::kGroups;
	__shared__ float2 sums[G][2 * (TPR > 32 ? TPR / 32 : 1)];
	extern __shared__ float4 rings4[];  // the rings; afterwards, where G > 1, the threads' sums [2 E][threads]
	const int group = threadIdx.x / TPR, t = threadIdx.x % TPR;
	const uint32_t W = d.width;
	const float inv_w = 1.f / (float)W;
	let_next_start();
	wait_for_previous();
	float ga[E];
#pragma unroll
	for (int k = 0; k < E; ++k) {
		const uint32_t c = ((k / VEC) * TPR + t) * VEC + k % VEC;
		ga[k] = c < W ? param_at(gamma, d.param_dtype, c) : 0.f;
	}
	float dg[E], db[E];
#pragma unroll
	for (int k = 0; k < E; ++k) dg[k] = db[k] = 0.f;
	int turn = 0, slot = 0;
	uint32_t parity = 0, r = blockIdx.x * G + group;
	const uint32_t step = gridDim.x * G;
	const bool add = skip && dx;
	const uint32_t row_bytes = W * (uint32_t)sizeof(T), slot_bytes = row_bytes * (add ? 3 : 2);  // x, dy, skip
	unsigned char* const ring = reinterpret_cast<unsigned char*>(rings4) + (size_t)group * depth * slot_bytes;
	auto order = [&](uint64_t row, int i) {
		const uint32_t bar = sptr(&bars[group * kMaxDepth + i]), dst = sptr(ring + (size_t)i * slot_bytes);
		expect_bytes(bar, slot_bytes);
		copy_row(dst, x + row * x_ld, row_bytes, bar);
		copy_row(dst + row_bytes, dy + row * dy_ld, row_bytes, bar);
		if (add) copy_row(dst + 2 * row_bytes, skip + row * skip_ld, row_bytes, bar);
	};
	if (RING && threadIdx.x == 0) given_up = 0;
	if (RING && t == 0) {
		for (int i = 0; i < depth; ++i) init_barrier(sptr(&bars[group * kMaxDepth + i]));
		for (int i = 0; i < depth; ++i) {
			const uint64_t row = (uint64_t)r + (uint64_t)i * step;
			if (row < d.n) order(row, i);
		}
	}
	if (RING) __syncthreads();
	float mu = 0.f, rs = 0.f;
	if (r < d.n) mu = mean[r], rs = rstd[r];
	for (uint32_t r0 = blockIdx.x * G; r0 < d.n; r0 += step, r += step) {
		Raw rx[VPT], ry[VPT], rk[VPT];
		const float m = mu, sc = rs;
		if ((uint64_t)r + step < d.n) mu = mean[r + step], rs = rstd[r + step];  // of the next row, ahead of its turn
		const unsigned char* const row = ring + (size_t)slot * slot_bytes;
		if (RING && r < d.n) wait_row(sptr(&bars[group * kMaxDepth + slot]), parity, given_up);
#pragma unroll
		for (int k = 0; k < VPT; ++k) {  // zeros outside of the row and behind the last one: they add nothing to any sum
			const uint32_t c = (k * TPR + t) * VEC;
			const bool in = r < d.n && c < W;
			auto get = [&](int which, const T* p, uint64_t ld) {
				return *reinterpret_cast<const Raw*>(RING ? row + which * row_bytes + c * sizeof(T) : (const unsigned char*)(p + r * ld + c));
			};
			rx[k] = in ? get(0, x, x_ld) : zero<Raw>();
			ry[k] = in ? get(1, dy, dy_ld) : zero<Raw>();
			rk[k] = in && add ? get(2, skip, skip_ld) : zero<Raw>();
		}
		if (RING) {
			group_barrier<TPR>(group);  // the rows are in registers: their place is free
			const uint64_t next = (uint64_t)r + (uint64_t)depth * step;
			if (t == 0 && next < d.n && !given_up) order(next, slot);
			if (++slot == depth) slot = 0, parity ^= 1u;
		}
		float s1 = 0.f, s2 = 0.f;
		float xh[E], a[E];
#pragma unroll
		for (int k = 0; k < VPT; ++k) {
			float ex[VEC], ey[VEC];
			P::get(rx[k], ex);
			P::get(ry[k], ey);
#pragma unroll
			for (int i = 0; i < VEC; ++i) {
				const int e = k * VEC + i;
				xh[e] = (ex[i] - m) * sc, a[e] = ey[i] * ga[e];
				dg[e] = fmaf(ey[i], xh[e], dg[e]);
				db[e] += ey[i];
				s1 += a[e];
				s2 = fmaf(a[e], xh[e], s2);
			}
		}
		if (dx) {
			group_sums<TPR>(s1, s2, sums[group], group, turn);
			s1 *= inv_w, s2 *= inv_w;
			if (r < d.n) {
#pragma unroll
				for (int k = 0; k < VPT; ++k) {
					const uint32_t c = (k * TPR + t) * VEC;
					float v[VEC], sk[VEC];
					P::get(rk[k], sk);
#pragma unroll
					for (int i = 0; i < VEC; ++i) v[i] = fmaf(sc, a[k * VEC + i] - s1 - xh[k * VEC + i] * s2, sk[i]);
					if (c < W) *reinterpret_cast<Raw*>(dx + r * dx_ld + c) = P::put(v);
				}
			}
		}
	}
	if (!partial && !dgamma && !dbeta) return;
	float* const mine = reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(rings4) + sums_at);
	float* out = partial ? partial + (uint64_t)blockIdx.x * 2 * W : mine;
	if constexpr (G > 1) {  // every thread's sums go to shared memory, and the block's threads share the columns
		float* const all = reinterpret_cast<float*>(rings4);
		__syncthreads();
#pragma unroll
		for (int k = 0; k < E; ++k) all[k * B::kThreads + threadIdx.x] = dg[k], all[(E + k) * B::kThreads + threadIdx.x] = db[k];
		__syncthreads();
		for (int i = threadIdx.x; i < 2 * E * TPR; i += B::kThreads) {
			const int k = i / TPR, e = k % E;
			const uint32_t c = ((e / VEC) * TPR + i % TPR) * VEC + e % VEC;
			float v = 0.f;
#pragma unroll
			for (int g = 0; g < G; ++g) v += all[k * B::kThreads + g * TPR + i % TPR];
			if (c < W) out[(k < E ? 0 : W) + c] = v;
		}
	} else {
#pragma unroll
		for (int k = 0; k < E; ++k) {
			const uint32_t c = ((k / VEC) * TPR + t) * VEC + k % VEC;
			if (c < W) out[c] = dg[k], out[W + c] = db[k];
		}
	}
	if (partial) return;
	__syncwarp();
	cluster_sync();
	for (uint32_t i = blockIdx.x * B::kThreads + threadIdx.x; i < 2 * W; i += gridDim.x * B::kThreads) {
		float part[kCluster], v = 0.f;
#pragma unroll
		for (uint32_t b = 0; b < kCluster; ++b) part[b] = b < gridDim.x ? load_peer(sptr(mine + i), b) : 0.f;
#pragma unroll
		for (uint32_t b = 0; b < kCluster; ++b) v += part[b];
		float* const o = i < W ? dgamma : dbeta;
		const uint32_t c = i < W ? i : i - W;
		if (o) o[c] = accumulate ? o[c] + v : v;
	}
	__syncwarp();
	cluster_sync();  // (before this block's memory goes)
}

// sums of the blocks' parts: a block takes 32 columns of [parts][2 width], its 32 rows of threads share the parts and join in order
__global__ void __launch_bounds__(1024) join_kernel(const float* __restrict__ partial, uint32_t parts, uint32_t width, float* __restrict__ dgamma,
                                                     float* __restrict__ dbeta, int accumulate) {
	__shared__ float s[32][33];
	let_next_start();
	wait_for_previous();
	const uint32_t c = blockIdx.x * 32 + threadIdx.x;
	float v = 0.f;
	if (c < 2 * width)
		for (uint32_t p = threadIdx.y; p < parts; p += 32) v += partial[(uint64_t)p * 2 * width + c];
	s[threadIdx.y][threadIdx.x] = v;
	__syncthreads();
	if (threadIdx.y == 0 && c < 2 * width) {
		for (int k = 1; k < 32; ++k) v += s[k][threadIdx.x];
		float* o = c < width ? (dgamma ? dgamma + c : nullptr) : (dbeta ? dbeta + (c - width) : nullptr);
		if (o) *o = accumulate ? *o + v : v;
	}
}

// ---- rows that do not fit into the registers of a block: read once for each sum and once for the result (from L2), entry by entry.  Forward
// these are rows above 8192 entries off 16-byte boundaries, and above 16384 on them; backward rows above 4096 entries
// off the boundaries and above 8192 on them, where the parameters' sums take x and dL/dy a second time, 32 columns a block: 4096 x 12288
// bf16 259 us, 4096 x 6001 fp16 129 us, five to six times the time of their bytes.

// sum over the block, the same value in every thread
__device__ __forceinline__ float block_sum(float v, float* s) {
#pragma unroll
	for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
	__syncthreads();
	if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
	__syncthreads();
	v = 0.f;
	for (int w = 0; w < (int)(blockDim.x >> 5); ++w) v += s[w];
	return v;
}

constexpr int kWideThreads = 512;  // with four loads on their way each (1385 rows of 9837 fp16: 27 us; 256 threads, one load: 36)
template <typename T>
__global__ void __launch_bounds__(kWideThreads) wide_forward_kernel(neus2b_layer_norm_desc d, const T* x, uint64_t x_ld, const void* __restrict__ gamma,
                                                            const void* __restrict__ beta, T* y, uint64_t y_ld, float* __restrict__ mean_out,
                                                            float* __restrict__ rstd_out) {
	__shared__ float s[kWideThreads / 32];
	const uint32_t W = d.width;
	for (uint32_t r = blockIdx.x; r < d.n; r += gridDim.x) {
		const T* xr = x + r * x_ld;
		float v = 0.f;
#pragma unroll 4
		for (uint32_t c = threadIdx.x; c < W; c += kWideThreads) v += to_f(xr[c]);
		const float mean = block_sum(v, s) / (float)W;
		v = 0.f;
#pragma unroll 4
		for (uint32_t c = threadIdx.x; c < W; c += kWideThreads) {
			const float t = to_f(xr[c]) - mean;
			v = fmaf(t, t, v);
		}
		const float rstd = 1.f / sqrtf(block_sum(v, s) / (float)W + d.epsilon);
#pragma unroll 4
		for (uint32_t c = threadIdx.x; c < W; c += kWideThreads) {
			const float g = param_at(gamma, d.param_dtype, c), b = beta ? param_at(beta, d.param_dtype, c) : 0.f;
			y[r * y_ld + c] = from_f<T>(fmaf((to_f(xr[c]) - mean) * rstd, g, b));
		}
		if (mean_out && threadIdx.x == 0) mean_out[r] = mean, rstd_out[r] = rstd;
	}
}

template <typename T>
__global__ void __launch_bounds__(kWideThreads) wide_backward_kernel(neus2b_layer_norm_desc d, const T* __restrict__ x, uint64_t x_ld,
                                                             const void* __restrict__ gamma, const float* __restrict__ mean,
                                                             const float* __restrict__ rstd, const T* dy, uint64_t dy_ld, const T* skip,
                                                             uint64_t skip_ld, T* dx, uint64_t dx_ld) {
	__shared__ float s[kWideThreads / 32];
	const uint32_t W = d.width;
	for (uint32_t r = blockIdx.x; r < d.n; r += gridDim.x) {
		const float mu = mean[r], rs = rstd[r];
		float s1 = 0.f, s2 = 0.f;
#pragma unroll 4
		for (uint32_t c = threadIdx.x; c < W; c += kWideThreads) {
			const float a = param_at(gamma, d.param_dtype, c) * to_f(dy[r * dy_ld + c]);
			s1 += a;
			s2 = fmaf(a, (to_f(x[r * x_ld + c]) - mu) * rs, s2);
		}
		s1 = block_sum(s1, s) / (float)W;
		s2 = block_sum(s2, s) / (float)W;
#pragma unroll 4
		for (uint32_t c = threadIdx.x; c < W; c += kWideThreads) {
			const float a = param_at(gamma, d.param_dtype, c) * to_f(dy[r * dy_ld + c]);
			const float xh = (to_f(x[r * x_ld + c]) - mu) * rs;
			dx[r * dx_ld + c] = from_f<T>(rs * (a - s1 - xh * s2) + (skip ? to_f(skip[r * skip_ld + c]) : 0.f));
		}
	}
}

// dgamma, dbeta of 32 columns
template <typename T>
__global__ void __launch_bounds__(1024) wide_params_kernel(uint32_t n, uint32_t width, const T* __restrict__ x, uint64_t x_ld,
                                                            const float* __restrict__ mean, const float* __restrict__ rstd,
                                                            const T* __restrict__ dy, uint64_t dy_ld, float* __restrict__ dgamma,
                                                            float* __restrict__ dbeta, int accumulate) {
	__shared__ float sg[32][33], sb[32][33];
	const uint32_t c = blockIdx.x * 32 + threadIdx.x;
	float g = 0.f, b = 0.f;
	if (c < width)
		for (uint32_t r = threadIdx.y; r < n; r += 32) {
			const float v = to_f(dy[r * dy_ld + c]);
			b += v;
			g = fmaf(v, (to_f(x[r * x_ld + c]) - mean[r]) * rstd[r], g);
		}
	sg[threadIdx.y][threadIdx.x] = g;
	sb[threadIdx.y][threadIdx.x] = b;
	__syncthreads();
	if (threadIdx.y == 0 && c < width) {
		for (int k = 1; k < 32; ++k) g += sg[k][threadIdx.x], b += sb[k][threadIdx.x];
		if (dgamma) dgamma[c] = accumulate ? dgamma[c] + g : g;
		if (dbeta) dbeta[c] = accumulate ? dbeta[c] + b : b;
	}
}


constexpr uint32_t kWidest = 8192;  // entries that a backward variant holds at most
constexpr uint32_t kWidestUnaligned = 4096;  // of rows off 16-byte boundaries
// Blocks a SM that a backward variant for rows of this width runs at most, whether they start on 16-byte boundaries or not.
constexpr uint32_t most_blocks(uint32_t width) { return width <= 256 ? 8 : width <= 2048 ? 4 : width <= kWidestUnaligned ? 2 : 1; }
constexpr int kTooWide = -1000;     // no variant holds the row

template <typename T, int VEC, int TPR, int VPT>
struct Variant {
	static constexpr int kVec = VEC, kTpr = TPR, kVpt = VPT;
};

// The narrowest group that holds the row, `u` accesses of VEC entries, for rows that are read with plain loads: short ones, and those that
// do not start on 16-byte boundaries (VEC 1).
template <typename T, int VEC, typename F>
int with_forward_variant(uint32_t width, F f) {
	const uint32_t u = (width + VEC - 1) / VEC;
	// Short rows are bound by the instructions around them (sums over the group, statistics): two accesses a thread halve these
	// (262144 rows of 64 fp16: 15.2 -> 14.1 us).
	if (u <= 8) return f(Variant<T, VEC, 4, 2>());
	if (u <= 16) return f(Variant<T, VEC, 8, 2>());
	if (u <= 32) return f(Variant<T, VEC, 16, 2>());
	if constexpr (VEC == 1) {
		if (u <= 64) return f(Variant<T, VEC, 32, 2>());
		if (u <= 128) return f(Variant<T, VEC, 32, 4>());
		if (u <= 256) return f(Variant<T, VEC, 32, 8>());
		if (u <= 512) return f(Variant<T, VEC, 32, 16>());
		if (u <= 1024) return f(Variant<T, VEC, 32, 32>());
		if (u <= 2048) return f(Variant<T, VEC, 256, 8>());
		if (u <= 4096) return f(Variant<T, VEC, 256, 16>());
		if (u <= 8192) return f(Variant<T, VEC, 256, 32>());
	}
	if constexpr (VEC == 4) {  // too wide for a ring beside gamma and beta in shared memory
		if (u > 2048 && u <= 4096) return f(Variant<T, VEC, 256, 16>());
	}
	return kTooWide;
}
template <typename T, int VEC, typename F>
int with_backward_variant(uint32_t width, F f) {
	const uint32_t u = (width + VEC - 1) / VEC;
	if (u <= 8) return f(Variant<T, VEC, 8, 1>());
	if (u <= 16) return f(Variant<T, VEC, 16, 1>());
	if (u <= 32) return f(Variant<T, VEC, 32, 1>());
	if constexpr (VEC == 1) {
		if (u <= 64) return f(Variant<T, VEC, 32, 2>());
		if (u <= 128) return f(Variant<T, VEC, 32, 4>());
		if (u <= 512) return f(Variant<T, VEC, 32, 16>());
		if (u <= 1024) return f(Variant<T, VEC, 64, 16>());
		if (u <= 2048) return f(Variant<T, VEC, 128, 16>());
		if (u <= 4096) return f(Variant<T, VEC, 256, 16>());
	}
	return kTooWide;
}
// Rows of 512 bytes and more are worth a bulk copy each.  The ring variants are those of the widths from there on.
constexpr size_t kRingRow = 512;
template <typename T, int VEC, typename F>
int with_forward_ring(uint32_t width, F f) {
	const uint32_t u = (width + VEC - 1) / VEC;
	if (u <= 64) return f(Variant<T, VEC, 32, 2>());
	if (u <= 128) return f(Variant<T, VEC, 32, 4>());
	if (u <= 256) return f(Variant<T, VEC, 64, 4>());
	if (u <= 512) return f(Variant<T, VEC, 128, 4>());
	if (u <= 1024) return f(Variant<T, VEC, 256, 4>());
	if (u <= 2048) return f(Variant<T, VEC, 512, 4>());
	return kTooWide;
}
template <typename T, int VEC, typename F>
int with_backward_ring(uint32_t width, F f) {
	const uint32_t u = (width + VEC - 1) / VEC;
	constexpr int M = VEC == 8 ? 2 : 4;  // 16 entries a thread
	if constexpr (VEC == 8) {
		if (u <= 32) return f(Variant<T, VEC, 32, 1>());  // 8, and twice the threads: 65536 rows of 256 bf16 32 us, before 40
	}
	if (u <= 32 * M) return f(Variant<T, VEC, 32, M>());
	if (u <= 64 * M) return f(Variant<T, VEC, 64, M>());
	if (u <= 128 * M) return f(Variant<T, VEC, 128, M>());
	if (u <= 256 * M) return f(Variant<T, VEC, 256, M>());
	if (u <= 512 * M) return f(Variant<T, VEC, 512, M>());
	return kTooWide;
}
// Dynamic shared memory of a block at most; what a launch may ask for is set to this whatever it takes, so that calls of several threads agree.
constexpr int kRoom = 216 * 1024;
// rows ahead of a group, `round` bytes for one of every group: as many as fit, 4 at most
static int ring_depth(size_t fixed, size_t round) {
	const size_t room = kRoom, d = fixed < room ? (room - fixed) / round : 0;
	return d < 4 ? (int)d : 4;
}
static bool rows16(const void* p, uint64_t ld, size_t bytes) { return !p || (((uintptr_t)p | (ld * bytes)) & 15) == 0; }

}  // namespace ln

using namespace ln;

int read_layer_norm_error(uint32_t* flags) {
	const cudaError_t e = cudaMemcpyFromSymbol(flags, ln::g_error, sizeof(*flags));
	return e == cudaSuccess ? NEUS2B_OK : (int)e;
}
int write_layer_norm_error(uint32_t flags) {
	const cudaError_t e = cudaMemcpyToSymbol(ln::g_error, &flags, sizeof(flags));
	return e == cudaSuccess ? NEUS2B_OK : (int)e;
}

static int check_desc(const neus2b_layer_norm_desc* d) {
	if (!d || d->width == 0 || !(d->epsilon > 0.f) || isinf(d->epsilon)) return NEUS2B_E_INVALID;
	if (d->n > (1u << 31) || d->width > (1u << 30)) return NEUS2B_E_TOO_LARGE;
	if (d->dtype > NEUS2B_BF16 || (d->param_dtype != NEUS2B_F32 && d->param_dtype != d->dtype)) return NEUS2B_E_UNSUPPORTED;
	return NEUS2B_OK;
}
// An output in place of an input has to have its rows where the input has them.
static bool clash(const void* out, uint64_t out_stride, const void* in, uint64_t in_stride, uint32_t n) { return out && out == in && n > 1 && out_stride != in_stride; }
static bool bad_rows(const void* p, uint64_t stride, uint32_t width, size_t align) { return !p || stride < width || ((uintptr_t)p & (align - 1)); }

}  // namespace n2b

using namespace n2b;

extern "C" int neus2b_layer_norm_forward(const neus2b_layer_norm_desc* desc, const void* d_x, uint64_t x_stride, const void* d_gamma, const void* d_beta,
                                         void* d_y, uint64_t y_stride, float* d_mean, float* d_rstd, neus2b_stream_t stream) {
	if (int rc = check_desc(desc)) return rc;
	const size_t b = dtype_bytes(desc->dtype), pb = dtype_bytes(desc->param_dtype);
	if (!d_gamma || (((uintptr_t)d_gamma | (uintptr_t)d_beta) & (pb - 1)) || !d_mean != !d_rstd || (((uintptr_t)d_mean | (uintptr_t)d_rstd) & 3))
		return NEUS2B_E_INVALID;
	if (desc->n == 0) return NEUS2B_OK;
	if (bad_rows(d_x, x_stride, desc->width, b) || bad_rows(d_y, y_stride, desc->width, b)) return NEUS2B_E_INVALID;
	if (clash(d_y, y_stride, d_x, x_stride, desc->n)) return NEUS2B_E_INVALID;
	return with_float_type(desc->dtype, [&](auto t) {
		using T = decltype(t);
		constexpr int V = 16 / sizeof(T);
		const size_t row = desc->width * b;
		auto go = [&](auto v, auto ring) {
			using K = decltype(v);
			using F = Forward<T, K::kVec, K::kTpr, K::kVpt, decltype(ring)::value>;
			auto kernel = forward_kernel<T, K::kVec, K::kTpr, K::kVpt, decltype(ring)::value>;
			size_t smem = F::kStaged ? 2 * K::kTpr * K::kVpt * K::kVec * sizeof(float) : 0;
			int depth = 0;
			if (ring) {
				depth = ring_depth(smem, F::kGroups * row);
				if (!depth) return kTooWide;
				smem += (size_t)F::kGroups * row * depth;
			}
			if (smem > 32 * 1024) N2B_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRoom));
			int resident = 1;
			if (!ring) {
				static const int most = [&] {
					int q = 0;
					return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&q, kernel, F::kThreads, smem) == cudaSuccess && q > 0 ? q : F::kBlocks;
				}();
				resident = most;
			}
			const uint32_t need = (desc->n + F::kGroups - 1) / F::kGroups, most = kSMs * resident;
			return launch_behind(kernel, need < most ? need : most, F::kThreads, smem, stream, *desc, depth, (const T*)d_x, x_stride, d_gamma, d_beta, (T*)d_y, y_stride,
			                     d_mean, d_rstd);
		};
		const bool vec = rows16(d_x, x_stride, b) && rows16(d_y, y_stride, b) && desc->width % V == 0;
		int rc = kTooWide;
		if (vec && row >= kRingRow) rc = with_forward_ring<T, V>(desc->width, [&](auto v) { return go(v, std::true_type()); });
		if (rc == kTooWide) {
			auto plain = [&](auto v) { return go(v, std::false_type()); };
			rc = vec ? with_forward_variant<T, V>(desc->width, plain) : with_forward_variant<T, 1>(desc->width, plain);
		}
		if (rc != kTooWide) return rc;
		wide_forward_kernel<T><<<desc->n < 4u * kSMs ? desc->n : 4u * kSMs, kWideThreads, 0, stream>>>(*desc, (const T*)d_x, x_stride, d_gamma, d_beta, (T*)d_y,
		                                                                                 y_stride, d_mean, d_rstd);
		N2B_CHECK_LAUNCH();
		return NEUS2B_OK;
	});
}

extern "C" int neus2b_layer_norm_backward_workspace(const neus2b_layer_norm_desc* desc, uint64_t* bytes) {
	if (int rc = check_desc(desc)) return rc;
	if (!bytes) return NEUS2B_E_INVALID;
	const uint64_t most = (uint64_t)kSMs * most_blocks(desc->width), blocks = desc->n < most ? desc->n : most;
	*bytes = desc->width <= kWidest && desc->n > kFewRows ? blocks * 2 * desc->width * sizeof(float) : 0;
	return NEUS2B_OK;
}

extern "C" int neus2b_layer_norm_backward(const neus2b_layer_norm_desc* desc, const void* d_x, uint64_t x_stride, const void* d_gamma, const float* d_mean,
                                          const float* d_rstd, const void* d_dL_dy, uint64_t dy_stride, const void* d_skip, uint64_t skip_stride,
                                          void* d_dL_dx, uint64_t dx_stride, float* d_dgamma, float* d_dbeta, int grad_mode, void* d_workspace,
                                          uint64_t workspace_bytes, neus2b_stream_t stream) {
	uint64_t need = 0;
	if (int rc = neus2b_layer_norm_backward_workspace(desc, &need)) return rc;
	if (grad_mode < NEUS2B_GRAD_IGNORE || grad_mode > NEUS2B_GRAD_ACCUMULATE) return NEUS2B_E_INVALID;
	if (grad_mode == NEUS2B_GRAD_IGNORE) d_dgamma = d_dbeta = nullptr;
	if (!d_dgamma && !d_dbeta) need = 0;  // the workspace is theirs
	const uint32_t n = desc->n, width = desc->width;
	const size_t b = dtype_bytes(desc->dtype);
	if (((uintptr_t)d_dgamma | (uintptr_t)d_dbeta | (uintptr_t)d_mean | (uintptr_t)d_rstd) & 3) return NEUS2B_E_INVALID;
	if (!d_gamma || ((uintptr_t)d_gamma & (dtype_bytes(desc->param_dtype) - 1))) return NEUS2B_E_INVALID;
	if (n == 0) {
		if (grad_mode == NEUS2B_GRAD_OVERWRITE) {
			if (d_dgamma) N2B_CHECK_CUDA(cudaMemsetAsync(d_dgamma, 0, (size_t)width * 4, stream));
			if (d_dbeta) N2B_CHECK_CUDA(cudaMemsetAsync(d_dbeta, 0, (size_t)width * 4, stream));
		}
		return NEUS2B_OK;
	}
	if (!d_mean || !d_rstd || bad_rows(d_x, x_stride, width, b) || bad_rows(d_dL_dy, dy_stride, width, b) ||
	    (d_skip && bad_rows(d_skip, skip_stride, width, b)) || (d_dL_dx && bad_rows(d_dL_dx, dx_stride, width, b)))
		return NEUS2B_E_INVALID;
	if ((d_dL_dx && d_dL_dx == d_x) || clash(d_dL_dx, dx_stride, d_dL_dy, dy_stride, n) || clash(d_dL_dx, dx_stride, d_skip, skip_stride, n)) return NEUS2B_E_INVALID;
	const bool vec = rows16(d_x, x_stride, b) && rows16(d_dL_dy, dy_stride, b) && rows16(d_skip, skip_stride, b) && rows16(d_dL_dx, dx_stride, b) &&
	                 width * b % 16 == 0;
	if (!vec && width > kWidestUnaligned) need = 0;
	if (need && (!d_workspace || ((uintptr_t)d_workspace & 15) || workspace_bytes < need)) return NEUS2B_E_INVALID;
	return with_float_type(desc->dtype, [&](auto t) {
		using T = decltype(t);
		constexpr int V = 16 / sizeof(T);
		const bool params = d_dgamma || d_dbeta;
		const int accumulate = grad_mode == NEUS2B_GRAD_ACCUMULATE;
		if (!params && !d_dL_dx) return NEUS2B_OK;
		const size_t row = width * b;
		auto go = [&](auto v, auto ring) {
			using K = decltype(v);
			using B = Backward<K::kTpr, K::kVpt * K::kVec, decltype(ring)::value>;
			static_assert(B::kGrid <= kSMs * (int)most_blocks(K::kTpr * K::kVpt * K::kVec), "the workspace holds the sums of every block");
			const bool few = params && n <= kFewRows;
			const uint32_t need = (n + B::kGroups - 1) / B::kGroups, most = few ? kCluster : (uint32_t)B::kGrid, blocks = need < most ? need : most;
			constexpr size_t kSums = B::kGroups > 1 ? 2 * K::kVpt * K::kVec * B::kThreads * sizeof(float) : 0;
			const size_t kept = few ? (size_t)2 * width * sizeof(float) : 0;  // the block's sums
			size_t smem = 0;
			const size_t slot = row * (d_skip && d_dL_dx ? 3 : 2) * B::kGroups;
			int depth = 0;
			if (ring) {
				depth = ring_depth(kept + 16, slot);
				if (!depth) return kTooWide;
				smem = slot * depth;
			}
			smem = ((smem > kSums ? smem : kSums) + 15) / 16 * 16;
			const uint32_t sums_at = (uint32_t)smem;
			smem += kept;
			auto kernel = backward_kernel<T, K::kVec, K::kTpr, K::kVpt, decltype(ring)::value>;
			if (smem > 32 * 1024) N2B_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRoom));
			if (int rc = launch_behind_in_clusters(few ? blocks : 1, kernel, blocks, B::kThreads, smem, stream, *desc, depth, (const T*)d_x, x_stride, d_gamma, d_mean, d_rstd, (const T*)d_dL_dy, dy_stride,
			                           (const T*)d_skip, skip_stride, (T*)d_dL_dx, dx_stride, params && !few ? (float*)d_workspace : nullptr, sums_at, few ? d_dgamma : nullptr,
			                           few ? d_dbeta : nullptr, accumulate))
				return rc;
			if (params && !few) {
				return launch_behind(join_kernel, (2 * width + 31) / 32, dim3(32, 32), 0, stream, (const float*)d_workspace, blocks, width, d_dgamma, d_dbeta,
				                     accumulate);
			}
			return NEUS2B_OK;
		};
		int rc = kTooWide;
		if (vec && row >= kRingRow) rc = with_backward_ring<T, V>(width, [&](auto v) { return go(v, std::true_type()); });
		if (rc == kTooWide) {
			auto plain = [&](auto v) { return go(v, std::false_type()); };
			rc = vec ? with_backward_variant<T, V>(width, plain) : with_backward_variant<T, 1>(width, plain);
		}
		if (rc != kTooWide) return rc;
		if (params) {  // ahead of the input gradient, which may overwrite dL/dy
			wide_params_kernel<T><<<(width + 31) / 32, dim3(32, 32), 0, stream>>>(n, width, (const T*)d_x, x_stride, d_mean, d_rstd, (const T*)d_dL_dy,
			                                                                       dy_stride, d_dgamma, d_dbeta, accumulate);
			N2B_CHECK_LAUNCH();
		}
		if (d_dL_dx) {
			wide_backward_kernel<T><<<n < 4u * kSMs ? n : 4u * kSMs, kWideThreads, 0, stream>>>(*desc, (const T*)d_x, x_stride, d_gamma, d_mean, d_rstd,
			                                                                      (const T*)d_dL_dy, dy_stride, (const T*)d_skip, skip_stride,
			                                                                      (T*)d_dL_dx, dx_stride);
			N2B_CHECK_LAUNCH();
		}
		return NEUS2B_OK;
	});
}
