// Layer norm over rows of any width, forward and backward.
#include "dense.cuh"

namespace n2b {

__device__ __forceinline__ float param_at(const void* p, uint32_t f32, uint32_t half_type, uint32_t c) {
	if (f32) return ((const float*)p)[c];
	return half_type == NEUS2B_F16 ? to_f(((const __half*)p)[c]) : to_f(((const __nv_bfloat16*)p)[c]);
}

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
__global__ void __launch_bounds__(256) norm_forward_kernel(neus2b_layer_norm_desc d, const T* x, uint64_t x_ld, const void* __restrict__ gamma,
                                                            const void* __restrict__ beta, T* y, uint64_t y_ld, float* __restrict__ mean_out,
                                                            float* __restrict__ rstd_out) {
	__shared__ float s[8];
	const uint32_t W = d.width, f32 = d.param_dtype == NEUS2B_F32;
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
			const float g = param_at(gamma, f32, d.param_dtype, c), b = beta ? param_at(beta, f32, d.param_dtype, c) : 0.f;
			y[r * y_ld + c] = from_f<T>(fmaf((to_f(xr[c]) - mean) * rstd, g, b));
		}
		if (mean_out && threadIdx.x == 0) mean_out[r] = mean, rstd_out[r] = rstd;
	}
}

template <typename T>
__global__ void __launch_bounds__(256) norm_backward_kernel(neus2b_layer_norm_desc d, const T* __restrict__ x, uint64_t x_ld,
                                                             const void* __restrict__ gamma, const float* __restrict__ mean,
                                                             const float* __restrict__ rstd, const T* dy, uint64_t dy_ld, const T* skip,
                                                             uint64_t skip_ld, T* dx, uint64_t dx_ld) {
	__shared__ float s[8];
	const uint32_t W = d.width, f32 = d.param_dtype == NEUS2B_F32;
	for (uint32_t r = blockIdx.x; r < d.n; r += gridDim.x) {
		const float mu = mean[r], rs = rstd[r];
		float s1 = 0.f, s2 = 0.f;
		for (uint32_t c = threadIdx.x; c < W; c += 256) {
			const float a = param_at(gamma, f32, d.param_dtype, c) * to_f(dy[r * dy_ld + c]);
			s1 += a;
			s2 = fmaf(a, (to_f(x[r * x_ld + c]) - mu) * rs, s2);
		}
		s1 = block_sum(s1, s) / (float)W;
		s2 = block_sum(s2, s) / (float)W;
		for (uint32_t c = threadIdx.x; c < W; c += 256) {
			const float a = param_at(gamma, f32, d.param_dtype, c) * to_f(dy[r * dy_ld + c]);
			const float xh = (to_f(x[r * x_ld + c]) - mu) * rs;
			dx[r * dx_ld + c] = from_f<T>(rs * (a - s1 - xh * s2) + (skip ? to_f(skip[r * skip_ld + c]) : 0.f));
		}
	}
}

// dgamma, dbeta of 32 columns
template <typename T>
__global__ void __launch_bounds__(1024) norm_params_kernel(uint32_t n, uint32_t width, const T* __restrict__ x, uint64_t x_ld,
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
		norm_forward_kernel<T><<<desc->n < 8u * kSMs ? desc->n : 8u * kSMs, 256, 0, stream>>>(*desc, (const T*)d_x, x_stride, d_gamma, d_beta, (T*)d_y,
		                                                                                 y_stride, d_mean, d_rstd);
		N2B_CHECK_LAUNCH();
		return NEUS2B_OK;
	});
}

extern "C" int neus2b_layer_norm_backward_workspace(const neus2b_layer_norm_desc* desc, uint64_t* bytes) {
	if (int rc = check_desc(desc)) return rc;
	if (!bytes) return NEUS2B_E_INVALID;
	*bytes = 0;
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
		if (d_dgamma || d_dbeta) {  // ahead of the input gradient, which may overwrite dL/dy
			norm_params_kernel<T><<<(width + 31) / 32, dim3(32, 32), 0, stream>>>(n, width, (const T*)d_x, x_stride, d_mean, d_rstd, (const T*)d_dL_dy,
			                                                                       dy_stride, d_dgamma, d_dbeta, grad_mode == NEUS2B_GRAD_ACCUMULATE);
			N2B_CHECK_LAUNCH();
		}
		if (d_dL_dx) {
			norm_backward_kernel<T><<<n < 8u * kSMs ? n : 8u * kSMs, 256, 0, stream>>>(*desc, (const T*)d_x, x_stride, d_gamma, d_mean, d_rstd,
			                                                                      (const T*)d_dL_dy, dy_stride, (const T*)d_skip, skip_stride,
			                                                                      (T*)d_dL_dx, dx_stride);
			N2B_CHECK_LAUNCH();
		}
		return NEUS2B_OK;
	});
}
