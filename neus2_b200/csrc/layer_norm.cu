// Layer norm over rows of any width, forward and backward.
//
// A group of TPR threads owns a row at a time and keeps it in registers: one read, one write per value.  Groups of up to a warp
// reduce with shuffles, wider ones through shared memory behind a barrier of their own; blocks are persistent, so gamma and beta
// (and in the backward pass the sums for their gradients) stay in registers over all rows of a group, and the next row is fetched
// before the current one is reduced.  The variance is the mean square of the centred row, not a difference of sums.
#include "dense.cuh"

namespace n2b {
namespace ln {

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

__device__ __forceinline__ float param_at(const void* p, uint32_t dtype, uint32_t c) {
	if (dtype == NEUS2B_F32) return ((const float*)p)[c];
	return dtype == NEUS2B_F16 ? to_f(((const __half*)p)[c]) : to_f(((const __nv_bfloat16*)p)[c]);
}

// Sums over the TPR threads of a group, in a fixed order, the same value in all of them.  s: shared memory of the group, [2][TPR / 32][2];
// `turn` alternates so that a barrier per sum is enough.
template <int TPR>
__device__ __forceinline__ void group_sum(float& a, float& b, float2* s, int group, int& turn) {
#pragma unroll
	for (int o = (TPR < 32 ? TPR : 32) / 2; o; o >>= 1) {
		a += __shfl_xor_sync(~0u, a, o);
		b += __shfl_xor_sync(~0u, b, o);
	}
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

template <int TPR>
struct Geometry {
	static constexpr int kThreads = TPR > 256 ? TPR : 256;
	static constexpr int kGroups = kThreads / TPR;
};

template <typename T, int VEC, int TPR, int VPT>
__global__ void __launch_bounds__(Geometry<TPR>::kThreads) forward_kernel(neus2b_layer_norm_desc d, const T* x, uint64_t x_ld,
                                                                          const void* __restrict__ gamma, const void* __restrict__ beta, T* y,
                                                                          uint64_t y_ld, float* __restrict__ mean_out, float* __restrict__ rstd_out) {
	using P = Pack<T, VEC>;
	constexpr int G = Geometry<TPR>::kGroups;
	__shared__ float2 sums[G][2 * (TPR > 32 ? TPR / 32 : 1)];
	const int group = threadIdx.x / TPR, t = threadIdx.x % TPR;
	const uint32_t W = d.width;
	float ga[VPT * VEC], be[VPT * VEC];
#pragma unroll
	for (int k = 0; k < VPT * VEC; ++k) {
		const uint32_t c = ((k / VEC) * TPR + t) * VEC + k % VEC;
		ga[k] = c < W ? param_at(gamma, d.param_dtype, c) : 0.f;
		be[k] = c < W && beta ? param_at(beta, d.param_dtype, c) : 0.f;
	}
	typename P::Raw raw[VPT];
	auto fetch = [&](uint32_t r) {
#pragma unroll
		for (int k = 0; k < VPT; ++k) {
			const uint32_t c = (k * TPR + t) * VEC;
			if (r < d.n && c < W) raw[k] = *reinterpret_cast<const typename P::Raw*>(x + r * x_ld + c);
		}
	};
	int turn = 0;
	uint32_t r = blockIdx.x * G + group;
	fetch(r);
	// every group of the block runs the same number of rounds: the shuffles of narrow groups take the whole warp
	for (uint32_t r0 = blockIdx.x * G; r0 < d.n; r0 += gridDim.x * G, r += gridDim.x * G) {
		float v[VPT * VEC];
		float s = 0.f, q = 0.f;
#pragma unroll
		for (int k = 0; k < VPT; ++k) {
			float e[VEC];
			P::get(raw[k], e);
#pragma unroll
			for (int i = 0; i < VEC; ++i) {
				v[k * VEC + i] = e[i];
				if ((k * TPR + t) * VEC + i < W) s += e[i];
			}
		}
		fetch(r + gridDim.x * G);
		group_sum<TPR>(s, q, sums[group], group, turn);
		const float mean = s / (float)W;
		q = s = 0.f;
#pragma unroll
		for (int k = 0; k < VPT * VEC; ++k) {
			v[k] -= mean;
			if (((k / VEC) * TPR + t) * VEC + k % VEC < W) q = fmaf(v[k], v[k], q);
		}
		group_sum<TPR>(q, s, sums[group], group, turn);
		const float rstd = 1.f / sqrtf(q / (float)W + d.epsilon);
		if (r < d.n) {
#pragma unroll
			for (int k = 0; k < VPT; ++k) {
				const uint32_t c = (k * TPR + t) * VEC;
				float e[VEC];
#pragma unroll
				for (int i = 0; i < VEC; ++i) e[i] = fmaf(v[k * VEC + i] * rstd, ga[k * VEC + i], be[k * VEC + i]);
				if (c < W) *reinterpret_cast<typename P::Raw*>(y + r * y_ld + c) = P::put(e);
			}
			if (mean_out && t == 0) mean_out[r] = mean, rstd_out[r] = rstd;
		}
	}
}

// partial: [gridDim.x][2][width], the block's sums for dgamma and dbeta.  A block adds its groups' sums in order.
template <typename T, int VEC, int TPR, int VPT>
__global__ void __launch_bounds__(Geometry<TPR>::kThreads) backward_kernel(neus2b_layer_norm_desc d, const T* __restrict__ x, uint64_t x_ld,
                                                                           const void* __restrict__ gamma, const float* __restrict__ mean,
                                                                           const float* __restrict__ rstd, const T* dy, uint64_t dy_ld, const T* skip,
                                                                           uint64_t skip_ld, T* dx, uint64_t dx_ld, float* __restrict__ partial) {
	using P = Pack<T, VEC>;
	using Raw = typename P::Raw;
	constexpr int G = Geometry<TPR>::kGroups, E = VPT * VEC;
	__shared__ float2 sums[G][2 * (TPR > 32 ? TPR / 32 : 1)];
	extern __shared__ float columns[];  // [2][TPR * E] where G > 1
	const int group = threadIdx.x / TPR, t = threadIdx.x % TPR;
	const uint32_t W = d.width;
	const float inv_w = 1.f / (float)W;
	float ga[E], dg[E], db[E];
#pragma unroll
	for (int k = 0; k < E; ++k) {
		const uint32_t c = ((k / VEC) * TPR + t) * VEC + k % VEC;
		ga[k] = c < W ? param_at(gamma, d.param_dtype, c) : 0.f;
		dg[k] = db[k] = 0.f;
	}
	Raw rx[VPT], ry[VPT];
	float mu = 0.f, rs = 0.f;
	auto fetch = [&](uint32_t r) {
		if (r >= d.n) return;
		mu = mean[r], rs = rstd[r];
#pragma unroll
		for (int k = 0; k < VPT; ++k) {
			const uint32_t c = (k * TPR + t) * VEC;
			if (c < W) {
				rx[k] = *reinterpret_cast<const Raw*>(x + r * x_ld + c);
				ry[k] = *reinterpret_cast<const Raw*>(dy + r * dy_ld + c);
			}
		}
	};
	int turn = 0;
	uint32_t r = blockIdx.x * G + group;
	fetch(r);
	for (uint32_t r0 = blockIdx.x * G; r0 < d.n; r0 += gridDim.x * G, r += gridDim.x * G) {
		const float m = mu, sc = rs;
		float s1 = 0.f, s2 = 0.f;
		float xh[E], a[E];
		Raw rk[VPT];
#pragma unroll
		for (int k = 0; k < VPT; ++k) {
			const uint32_t c = (k * TPR + t) * VEC;
			float ex[VEC], ey[VEC];
			P::get(rx[k], ex);
			P::get(ry[k], ey);
			if (skip && dx && r < d.n && c < W) rk[k] = *reinterpret_cast<const Raw*>(skip + r * skip_ld + c);
#pragma unroll
			for (int i = 0; i < VEC; ++i) {
				const int e = k * VEC + i;
				const bool in = r < d.n && c + i < W;
				xh[e] = in ? (ex[i] - m) * sc : 0.f;
				const float g = in ? ey[i] : 0.f;
				dg[e] = fmaf(g, xh[e], dg[e]);
				db[e] += g;
				a[e] = g * ga[e];
				s1 += a[e];
				s2 = fmaf(a[e], xh[e], s2);
			}
		}
		fetch(r + gridDim.x * G);
		if (dx) {
			group_sum<TPR>(s1, s2, sums[group], group, turn);
			s1 *= inv_w, s2 *= inv_w;
			if (r < d.n) {
#pragma unroll
				for (int k = 0; k < VPT; ++k) {
					const uint32_t c = (k * TPR + t) * VEC;
					float e[VEC], sk[VEC];
					if (skip) P::get(rk[k], sk);
#pragma unroll
					for (int i = 0; i < VEC; ++i) {
						e[i] = sc * (a[k * VEC + i] - s1 - xh[k * VEC + i] * s2);
						if (skip) e[i] += sk[i];
					}
					if (c < W) *reinterpret_cast<Raw*>(dx + r * dx_ld + c) = P::put(e);
				}
			}
		}
	}
	if (!partial) return;
	float* out = partial + (uint64_t)blockIdx.x * 2 * W;
	if (G > 1) {
		for (int g = 0; g < G; ++g) {
			if (group == g) {
#pragma unroll
				for (int k = 0; k < E; ++k) {
					const int c = ((k / VEC) * TPR + t) * VEC + k % VEC;
					if (g > 0) dg[k] += columns[c], db[k] += columns[TPR * E + c];
					if (g < G - 1) columns[c] = dg[k], columns[TPR * E + c] = db[k];
				}
			}
			__syncthreads();
		}
		if (group != G - 1) return;
	}
#pragma unroll
	for (int k = 0; k < E; ++k) {
		const uint32_t c = ((k / VEC) * TPR + t) * VEC + k % VEC;
		if (c < W) out[c] = dg[k], out[W + c] = db[k];
	}
}

// sums of the blocks' parts: a block takes 32 columns of [parts][2 width], its 32 rows of threads share the parts and join in order
__global__ void __launch_bounds__(1024) join_kernel(const float* __restrict__ partial, uint32_t parts, uint32_t width, float* __restrict__ dgamma,
                                                     float* __restrict__ dbeta, int accumulate) {
	__shared__ float s[32][33];
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

// ---- rows that do not fit into the registers of a block: read once for each sum and once for the result (from L2)

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

template <typename T>
__global__ void __launch_bounds__(256) wide_forward_kernel(neus2b_layer_norm_desc d, const T* x, uint64_t x_ld, const void* __restrict__ gamma,
                                                            const void* __restrict__ beta, T* y, uint64_t y_ld, float* __restrict__ mean_out,
                                                            float* __restrict__ rstd_out) {
	__shared__ float s[8];
	const uint32_t W = d.width;
	for (uint32_t r = blockIdx.x; r < d.n; r += gridDim.x) {
		const T* xr = x + r * x_ld;
		float v = 0.f;
		for (uint32_t c = threadIdx.x; c < W; c += 256) v += to_f(xr[c]);
		const float mean = block_sum(v, s) / (float)W;
		v = 0.f;
		for (uint32_t c = threadIdx.x; c < W; c += 256) {
			const float t = to_f(xr[c]) - mean;
			v = fmaf(t, t, v);
		}
		const float rstd = 1.f / sqrtf(block_sum(v, s) / (float)W + d.epsilon);
		for (uint32_t c = threadIdx.x; c < W; c += 256) {
			const float g = param_at(gamma, d.param_dtype, c), b = beta ? param_at(beta, d.param_dtype, c) : 0.f;
			y[r * y_ld + c] = from_f<T>(fmaf((to_f(xr[c]) - mean) * rstd, g, b));
		}
		if (mean_out && threadIdx.x == 0) mean_out[r] = mean, rstd_out[r] = rstd;
	}
}

template <typename T>
__global__ void __launch_bounds__(256) wide_backward_kernel(neus2b_layer_norm_desc d, const T* __restrict__ x, uint64_t x_ld,
                                                             const void* __restrict__ gamma, const float* __restrict__ mean,
                                                             const float* __restrict__ rstd, const T* dy, uint64_t dy_ld, const T* skip,
                                                             uint64_t skip_ld, T* dx, uint64_t dx_ld) {
	__shared__ float s[8];
	const uint32_t W = d.width;
	for (uint32_t r = blockIdx.x; r < d.n; r += gridDim.x) {
		const float mu = mean[r], rs = rstd[r];
		float s1 = 0.f, s2 = 0.f;
		for (uint32_t c = threadIdx.x; c < W; c += 256) {
			const float a = param_at(gamma, d.param_dtype, c) * to_f(dy[r * dy_ld + c]);
			s1 += a;
			s2 = fmaf(a, (to_f(x[r * x_ld + c]) - mu) * rs, s2);
		}
		s1 = block_sum(s1, s) / (float)W;
		s2 = block_sum(s2, s) / (float)W;
		for (uint32_t c = threadIdx.x; c < W; c += 256) {
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


constexpr int kBackwardBlocks = 2 * kSMs;
constexpr uint32_t kWidest = 8192;  // entries that a backward variant holds at most
constexpr int kTooWide = -1000;  // no variant holds the row

template <typename T, int VEC, int TPR, int VPT>
struct Variant {
	using Type = T;
	static constexpr int kVec = VEC, kTpr = TPR, kVpt = VPT;
};

// The narrowest group that holds the row: a row of `width` entries is width / VEC accesses.  Forward pass: up to four accesses of 16
// bytes a thread; backward pass: two, since a thread keeps five values for every entry.
template <typename T, int VEC, typename F>
int with_forward_variant(uint32_t width, F f) {
	const uint32_t u = (width + VEC - 1) / VEC;
	if (u <= 8) return f(Variant<T, VEC, 8, 1>());
	if (u <= 16) return f(Variant<T, VEC, 16, 1>());
	if (u <= 32) return f(Variant<T, VEC, 32, 1>());
	if (u <= 64) return f(Variant<T, VEC, 32, 2>());
	if (u <= 128) return f(Variant<T, VEC, 32, 4>());
	if (u <= 256) return f(Variant<T, VEC, 128, 2>());
	if (u <= 512) return f(Variant<T, VEC, 256, 2>());
	if (u <= 1024) return f(Variant<T, VEC, 256, 4>());
	if (u <= 2048) return f(Variant<T, VEC, 512, 4>());
	if (VEC < 8 && u <= 4096) return f(Variant<T, VEC, VEC < 8 ? 1024 : 512, 4>());
	if (VEC < 4 && u <= 8192) return f(Variant<T, VEC, VEC < 4 ? 1024 : 512, VEC < 4 ? 8 : 4>());
	return kTooWide;
}
template <typename T, int VEC, typename F>
int with_backward_variant(uint32_t width, F f) {
	const uint32_t u = (width + VEC - 1) / VEC;
	constexpr int X = VEC == 8 ? 1 : VEC == 4 ? 2 : 4;  // accesses that make up 8 entries, 4 at most
	if (u <= 8) return f(Variant<T, VEC, 8, 1>());
	if (u <= 16) return f(Variant<T, VEC, 16, 1>());
	if (u <= 32) return f(Variant<T, VEC, 32, 1>());
	if (u <= 32 * X) return f(Variant<T, VEC, 32, X>());
	if (u <= 64 * X) return f(Variant<T, VEC, 64, X>());
	if (u <= 128 * X) return f(Variant<T, VEC, 128, X>());
	if (u <= 256 * X) return f(Variant<T, VEC, 256, X>());
	if (u <= 512 * X) return f(Variant<T, VEC, 256, 2 * X>());
	if (u <= 1024 * X) return f(Variant<T, VEC, 512, 2 * X>());
	return kTooWide;
}
// backward blocks, and so partial sums, of a call
template <int TPR>
static uint32_t backward_blocks(uint32_t n) {
	const uint32_t need = (n + Geometry<TPR>::kGroups - 1) / Geometry<TPR>::kGroups;
	return need < (uint32_t)kBackwardBlocks ? need : kBackwardBlocks;
}
static bool rows16(const void* p, uint64_t ld, size_t bytes) { return !p || (((uintptr_t)p | (ld * bytes)) & 15) == 0; }

}  // namespace ln

using namespace ln;

static int check_desc(const neus2b_layer_norm_desc* d) {
	if (!d || d->width == 0 || !(d->epsilon > 0.f) || isinf(d->epsilon)) return NEUS2B_E_INVALID;
	if (d->dtype > NEUS2B_BF16 || (d->param_dtype != NEUS2B_F32 && d->param_dtype != d->dtype)) return NEUS2B_E_UNSUPPORTED;
	return NEUS2B_OK;
}
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
	return with_float_type(desc->dtype, [&](auto t) {
		using T = decltype(t);
		constexpr int V = 16 / sizeof(T);
		auto go = [&](auto v) {
			using K = decltype(v);
			constexpr int G = Geometry<K::kTpr>::kGroups;
			auto kernel = forward_kernel<T, K::kVec, K::kTpr, K::kVpt>;
			const uint32_t need = (desc->n + G - 1) / G, most = kSMs * (2048 / Geometry<K::kTpr>::kThreads);
			kernel<<<need < most ? need : most, Geometry<K::kTpr>::kThreads, 0, stream>>>(*desc, (const T*)d_x, x_stride, d_gamma, d_beta, (T*)d_y, y_stride, d_mean,
			                                                                          d_rstd);
			N2B_CHECK_LAUNCH();
			return NEUS2B_OK;
		};
		const bool vec = rows16(d_x, x_stride, b) && rows16(d_y, y_stride, b) && desc->width % V == 0;
		const int rc = vec ? with_forward_variant<T, V>(desc->width, go) : with_forward_variant<T, 1>(desc->width, go);
		if (rc != kTooWide) return rc;
		wide_forward_kernel<T><<<desc->n < 8u * kSMs ? desc->n : 8u * kSMs, 256, 0, stream>>>(*desc, (const T*)d_x, x_stride, d_gamma, d_beta, (T*)d_y,
		                                                                                 y_stride, d_mean, d_rstd);
		N2B_CHECK_LAUNCH();
		return NEUS2B_OK;
	});
}

extern "C" int neus2b_layer_norm_backward_workspace(const neus2b_layer_norm_desc* desc, uint64_t* bytes) {
	if (int rc = check_desc(desc)) return rc;
	if (!bytes) return NEUS2B_E_INVALID;
	// the most blocks that any variant runs: narrow groups share a block, so no variant has more than this
	const uint64_t blocks = desc->n < (uint32_t)kBackwardBlocks ? desc->n : kBackwardBlocks;
	*bytes = desc->width <= kWidest ? blocks * 2 * desc->width * sizeof(float) : 0;
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
	if (need && (!d_workspace || ((uintptr_t)d_workspace & 15) || workspace_bytes < need)) return NEUS2B_E_INVALID;
	return with_float_type(desc->dtype, [&](auto t) {
		using T = decltype(t);
		constexpr int V = 16 / sizeof(T);
		const bool params = d_dgamma || d_dbeta;
		const int accumulate = grad_mode == NEUS2B_GRAD_ACCUMULATE;
		if (!params && !d_dL_dx) return NEUS2B_OK;
		auto go = [&](auto v) {
			using K = decltype(v);
			constexpr int G = Geometry<K::kTpr>::kGroups;
			const uint32_t blocks = backward_blocks<K::kTpr>(n);
			const size_t smem = G > 1 ? 2 * K::kTpr * K::kVpt * K::kVec * sizeof(float) : 0;
			auto kernel = backward_kernel<T, K::kVec, K::kTpr, K::kVpt>;
			kernel<<<blocks, Geometry<K::kTpr>::kThreads, smem, stream>>>(*desc, (const T*)d_x, x_stride, d_gamma, d_mean, d_rstd, (const T*)d_dL_dy, dy_stride,
			                                                            (const T*)d_skip, skip_stride, (T*)d_dL_dx, dx_stride,
			                                                            params ? (float*)d_workspace : nullptr);
			N2B_CHECK_LAUNCH();
			if (params) {
				join_kernel<<<(2 * width + 31) / 32, dim3(32, 32), 0, stream>>>((const float*)d_workspace, blocks, width, d_dgamma, d_dbeta, accumulate);
				N2B_CHECK_LAUNCH();
			}
			return NEUS2B_OK;
		};
		const bool vec = rows16(d_x, x_stride, b) && rows16(d_dL_dy, dy_stride, b) && rows16(d_skip, skip_stride, b) && rows16(d_dL_dx, dx_stride, b) && width % V == 0;
		const int rc = vec ? with_backward_variant<T, V>(width, go) : with_backward_variant<T, 1>(width, go);
		if (rc != kTooWide) return rc;
		if (params) {  // ahead of the input gradient, which may overwrite dL/dy
			wide_params_kernel<T><<<(width + 31) / 32, dim3(32, 32), 0, stream>>>(n, width, (const T*)d_x, x_stride, d_mean, d_rstd, (const T*)d_dL_dy,
			                                                                       dy_stride, d_dgamma, d_dbeta, accumulate);
			N2B_CHECK_LAUNCH();
		}
		if (d_dL_dx) {
			wide_backward_kernel<T><<<n < 8u * kSMs ? n : 8u * kSMs, 256, 0, stream>>>(*desc, (const T*)d_x, x_stride, d_gamma, d_mean, d_rstd,
			                                                                      (const T*)d_dL_dy, dy_stride, (const T*)d_skip, skip_stride,
			                                                                      (T*)d_dL_dx, dx_stride);
			N2B_CHECK_LAUNCH();
		}
		return NEUS2B_OK;
	});
}
