// Shared pieces of the layers of any width (linear.cu, layer_norm.cu, grad_norm.cu): element types, activations.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

namespace n2b {

inline size_t dtype_bytes(uint32_t t) { return t == NEUS2B_F32 ? 4 : 2; }
inline bool is_half_type(uint32_t t) { return t == NEUS2B_F16 || t == NEUS2B_BF16; }

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

constexpr float kGeluC = 0.79788456080286536f, kGeluA = 0.044715f;  // sqrt(2 / pi); the cubic term of the tanh form

// gelu(z) = z / (1 + e^(-2u)), silu(z) = z / (1 + e^(-z)): e^.. overflows to infinity on the far negative side, where the quotient is -0.
__device__ __forceinline__ float act_value(int act, float z) {
	if (act == NEUS2B_ACT_RELU) return z > 0.f ? z : (z != z ? z : 0.f);
	if (act == NEUS2B_ACT_GELU) return z / (1.f + __expf(-2.f * kGeluC * fmaf(kGeluA * z * z, z, z)));
	if (act == NEUS2B_ACT_SILU) return z / (1.f + __expf(-z));
	return z;
}
// d act / dz.  gelu: s + z s (1 - s) 2u'; behind |z| = 10 the second term is below 1e-35, and z is held there so that u' stays finite.
__device__ __forceinline__ float act_slope(int act, float z) {
	if (act == NEUS2B_ACT_RELU) return z > 0.f ? 1.f : 0.f;
	if (act == NEUS2B_ACT_GELU) {
		const float s = 1.f / (1.f + __expf(-2.f * kGeluC * fmaf(kGeluA * z * z, z, z)));
		const float zc = fminf(fmaxf(z, -10.f), 10.f);
		return fmaf(zc * s * (1.f - s), 2.f * kGeluC * fmaf(3.f * kGeluA * zc, zc, 1.f), s);
	}
	if (act == NEUS2B_ACT_SILU) {
		const float s = 1.f / (1.f + __expf(-z));
		const float zc = fminf(fmaxf(z, -100.f), 100.f);
		return fmaf(zc * s, 1.f - s, s);
	}
	return 1.f;
}

template <typename F>
int with_half_type(uint32_t dtype, F f) {
	if (dtype == NEUS2B_F16) return f(__half());
	if (dtype == NEUS2B_BF16) return f(__nv_bfloat16());
	return NEUS2B_E_UNSUPPORTED;
}
template <typename F>
int with_float_type(uint32_t dtype, F f) {
	if (dtype == NEUS2B_F32) return f(float());
	return with_half_type(dtype, f);
}

}  // namespace n2b
