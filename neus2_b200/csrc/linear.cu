// Linear layers of any width: y = act(x W^T + b) + r, and the two products of the backward pass.
#include "dense.cuh"

namespace n2b {

// What happens to a sum on its way out.  forward: z = sum + bias, [z stored], act(z) + add; input gradient: sum * act'(slope_z) + add;
// weight gradient: fp32, optionally added to what is there.
struct Epilogue {
	void* out;
	uint64_t out_ld;
	const void *bias, *add, *slope_z;
	uint64_t add_ld, slope_ld;
	void* preact;
	uint64_t preact_ld;
	int act, out_f32, accumulate;
};

template <typename T>
__device__ __forceinline__ void epilogue_one(const Epilogue& e, uint64_t r, uint32_t c, float v) {
	if (e.out_f32) {
		float* o = (float*)e.out + r * e.out_ld + c;
		*o = e.accumulate ? *o + v : v;
		return;
	}
	if (e.bias) v += to_f(((const T*)e.bias)[c]);
	if (e.preact) ((T*)e.preact)[r * e.preact_ld + c] = from_f<T>(v);
	v = e.slope_z ? v * act_slope(e.act, to_f(((const T*)e.slope_z)[r * e.slope_ld + c])) : act_value(e.act, v);
	if (e.add) v += to_f(((const T*)e.add)[r * e.add_ld + c]);
	((T*)e.out)[r * e.out_ld + c] = from_f<T>(v);
}

// C[m][n] = sum_k a(m, k) b(n, k), a(m, k) = a[m * am + k * ak]: 64 x 64 tiles, 4 x 4 sums per thread.
template <typename T>
__global__ void __launch_bounds__(256) product_kernel(uint32_t M, uint32_t N, uint32_t K, const T* __restrict__ a, uint64_t am, uint64_t ak,
                                                       const T* __restrict__ b, uint64_t bn, uint64_t bk, Epilogue e) {
	__shared__ float sa[16][65], sb[16][65];
	const uint32_t tiles_n = (N + 63) / 64, tiles = ((M + 63) / 64) * tiles_n;
	const int tid = threadIdx.x, tr = tid / 16, tc = tid % 16;
	for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
		const uint32_t m0 = tile / tiles_n * 64, n0 = tile % tiles_n * 64;
		float acc[4][4] = {};
		for (uint32_t k0 = 0; k0 < K; k0 += 16) {
			for (int i = tid; i < 1024; i += 256) {
				const int r = ak == 1 ? i / 16 : i % 64, k = ak == 1 ? i % 16 : i / 64;
				sa[k][r] = (m0 + r < M && k0 + k < K) ? to_f(a[(m0 + r) * am + (k0 + k) * ak]) : 0.f;
				const int r2 = bk == 1 ? i / 16 : i % 64, k2 = bk == 1 ? i % 16 : i / 64;
				sb[k2][r2] = (n0 + r2 < N && k0 + k2 < K) ? to_f(b[(n0 + r2) * bn + (k0 + k2) * bk]) : 0.f;
			}
			__syncthreads();
#pragma unroll
			for (int k = 0; k < 16; ++k)
#pragma unroll
				for (int i = 0; i < 4; ++i)
#pragma unroll
					for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][tr + 16 * i], sb[k][tc + 16 * j], acc[i][j]);
			__syncthreads();
		}
		for (int i = 0; i < 4; ++i)
			for (int j = 0; j < 4; ++j) {
				const uint32_t r = m0 + tr + 16 * i, c = n0 + tc + 16 * j;
				if (r < M && c < N) epilogue_one<T>(e, r, c, acc[i][j]);
			}
	}
}

// dz = dy * act'(z)
template <typename T>
__global__ void __launch_bounds__(256) slope_kernel(uint64_t n, uint32_t width, int act, const T* __restrict__ z, uint64_t z_ld,
                                                     const T* __restrict__ dy, uint64_t dy_ld, T* __restrict__ dz) {
	for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < n * width; i += gridDim.x * 256ull) {
		const uint64_t r = i / width;
		const uint32_t c = (uint32_t)(i - r * width);
		dz[i] = from_f<T>(to_f(dy[r * dy_ld + c]) * act_slope(act, to_f(z[r * z_ld + c])));
	}
}

// sums of the columns, one block for 32 of them
template <typename T>
__global__ void __launch_bounds__(1024) column_sum_kernel(uint32_t n, uint32_t width, const T* __restrict__ a, uint64_t ld, float* __restrict__ out,
                                                          int accumulate) {
	__shared__ float s[32][33];
	const uint32_t c = blockIdx.x * 32 + threadIdx.x;
	float v = 0.f;
	if (c < width)
		for (uint32_t r = threadIdx.y; r < n; r += 32) v += to_f(a[r * ld + c]);
	s[threadIdx.y][threadIdx.x] = v;
	__syncthreads();
	if (threadIdx.y == 0 && c < width) {
		for (int k = 1; k < 32; ++k) v += s[k][threadIdx.x];
		out[c] = accumulate ? out[c] + v : v;
	}
}

static bool bad_desc(const neus2b_linear_desc* d) {
	return !d || d->in_width == 0 || d->out_width == 0 || d->activation > NEUS2B_ACT_SILU;
}
static bool bad_matrix(const void* p, uint64_t stride, uint32_t width, size_t align) { return !p || stride < width || ((uintptr_t)p & (align - 1)); }
static bool bad_optional(const void* p, uint64_t stride, uint32_t width, size_t align) { return p && bad_matrix(p, stride, width, align); }

template <typename T>
static int product(uint32_t M, uint32_t N, uint32_t K, const T* a, uint64_t am, uint64_t ak, const T* b, uint64_t bn, uint64_t bk,
                   const Epilogue& e, cudaStream_t s) {
	const uint64_t tiles = (uint64_t)((M + 63) / 64) * ((N + 63) / 64);
	product_kernel<T><<<(uint32_t)(tiles < 8 * kSMs ? tiles : 8 * kSMs), 256, 0, s>>>(M, N, K, a, am, ak, b, bn, bk, e);
	N2B_CHECK_LAUNCH();
	return NEUS2B_OK;
}

}  // namespace n2b

using namespace n2b;

extern "C" int neus2b_linear_forward(const neus2b_linear_desc* desc, const void* d_x, uint64_t x_stride, const void* d_w, const void* d_bias,
                                     const void* d_residual, uint64_t residual_stride, void* d_y, uint64_t y_stride, void* d_preact,
                                     uint64_t preact_stride, neus2b_stream_t stream) {
	if (bad_desc(desc)) return NEUS2B_E_INVALID;
	if (!is_half_type(desc->dtype)) return NEUS2B_E_UNSUPPORTED;
	const uint32_t in = desc->in_width, out = desc->out_width;
	if (bad_matrix(d_w, in, in, 2) || ((uintptr_t)d_bias & 1)) return NEUS2B_E_INVALID;
	if (desc->n == 0) return NEUS2B_OK;
	if (bad_matrix(d_x, x_stride, in, 2) || bad_matrix(d_y, y_stride, out, 2) || bad_optional(d_residual, residual_stride, out, 2) ||
	    bad_optional(d_preact, preact_stride, out, 2))
		return NEUS2B_E_INVALID;
	return with_half_type(desc->dtype, [&](auto t) {
		using T = decltype(t);
		Epilogue e{};
		e.out = d_y, e.out_ld = y_stride, e.bias = d_bias, e.add = d_residual, e.add_ld = residual_stride;
		e.preact = d_preact, e.preact_ld = preact_stride, e.act = (int)desc->activation;
		return product<T>(desc->n, out, in, (const T*)d_x, x_stride, 1, (const T*)d_w, in, 1, e, stream);
	});
}

extern "C" int neus2b_linear_backward_workspace(const neus2b_linear_desc* desc, uint64_t* bytes) {
	if (bad_desc(desc) || !bytes) return NEUS2B_E_INVALID;
	if (!is_half_type(desc->dtype)) return NEUS2B_E_UNSUPPORTED;
	*bytes = desc->activation == NEUS2B_ACT_NONE ? 0 : (uint64_t)desc->n * desc->out_width * 2;
	return NEUS2B_OK;
}

extern "C" int neus2b_linear_backward(const neus2b_linear_desc* desc, const void* d_x, uint64_t x_stride, const void* d_w, const void* d_preact,
                                      uint64_t preact_stride, const void* d_dL_dy, uint64_t dy_stride, uint32_t below_activation,
                                      const void* d_below_preact, uint64_t below_stride, const void* d_skip, uint64_t skip_stride, void* d_dL_dx,
                                      uint64_t dx_stride, float* d_wgrad, float* d_bgrad, int grad_mode, void* d_workspace,
                                      uint64_t workspace_bytes, neus2b_stream_t stream) {
	uint64_t need = 0;
	if (int rc = neus2b_linear_backward_workspace(desc, &need)) return rc;
	if (below_activation > NEUS2B_ACT_SILU || grad_mode < NEUS2B_GRAD_IGNORE || grad_mode > NEUS2B_GRAD_ACCUMULATE) return NEUS2B_E_INVALID;
	const uint32_t n = desc->n, in = desc->in_width, out = desc->out_width;
	if (grad_mode == NEUS2B_GRAD_IGNORE) d_wgrad = d_bgrad = nullptr;
	if (((uintptr_t)d_wgrad | (uintptr_t)d_bgrad) & 3) return NEUS2B_E_INVALID;
	if (n == 0) {
		if (grad_mode == NEUS2B_GRAD_OVERWRITE) {
			if (d_wgrad) N2B_CHECK_CUDA(cudaMemsetAsync(d_wgrad, 0, (size_t)in * out * 4, stream));
			if (d_bgrad) N2B_CHECK_CUDA(cudaMemsetAsync(d_bgrad, 0, (size_t)out * 4, stream));
		}
		return NEUS2B_OK;
	}
	if (bad_matrix(d_dL_dy, dy_stride, out, 2) || (d_wgrad && bad_matrix(d_x, x_stride, in, 2)) || (d_dL_dx && bad_matrix(d_w, in, in, 2)) ||
	    bad_optional(d_dL_dx, dx_stride, in, 2) || bad_optional(d_skip, skip_stride, in, 2))
		return NEUS2B_E_INVALID;
	if (desc->activation != NEUS2B_ACT_NONE && bad_matrix(d_preact, preact_stride, out, 2)) return NEUS2B_E_INVALID;
	if (d_dL_dx && below_activation != NEUS2B_ACT_NONE && bad_matrix(d_below_preact, below_stride, in, 2)) return NEUS2B_E_INVALID;
	if (need && (!d_workspace || ((uintptr_t)d_workspace & 15) || workspace_bytes < need)) return NEUS2B_E_INVALID;
	return with_half_type(desc->dtype, [&](auto t) {
		using T = decltype(t);
		const T* dz = (const T*)d_dL_dy;
		uint64_t dz_ld = dy_stride;
		if (desc->activation != NEUS2B_ACT_NONE) {
			slope_kernel<T><<<kSMs * 8, 256, 0, stream>>>(n, out, (int)desc->activation, (const T*)d_preact, preact_stride, dz, dz_ld, (T*)d_workspace);
			N2B_CHECK_LAUNCH();
			dz = (const T*)d_workspace;
			dz_ld = out;
		}
		if (d_wgrad) {
			Epilogue e{};
			e.out = d_wgrad, e.out_ld = in, e.out_f32 = 1, e.accumulate = grad_mode == NEUS2B_GRAD_ACCUMULATE;
			if (int rc = product<T>(out, in, n, dz, 1, dz_ld, (const T*)d_x, 1, x_stride, e, stream)) return rc;
		}
		if (d_bgrad) {
			column_sum_kernel<T><<<(out + 31) / 32, dim3(32, 32), 0, stream>>>(n, out, dz, dz_ld, d_bgrad, grad_mode == NEUS2B_GRAD_ACCUMULATE);
			N2B_CHECK_LAUNCH();
		}
		if (d_dL_dx) {
			Epilogue e{};
			e.out = d_dL_dx, e.out_ld = dx_stride, e.add = d_skip, e.add_ld = skip_stride;
			if (below_activation != NEUS2B_ACT_NONE) e.slope_z = d_below_preact, e.slope_ld = below_stride, e.act = (int)below_activation;
			if (int rc = product<T>(n, in, out, dz, dz_ld, 1, (const T*)d_w, 1, in, e, stream)) return rc;
		}
		return NEUS2B_OK;
	});
}
