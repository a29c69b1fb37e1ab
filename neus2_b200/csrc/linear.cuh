// Shared by the linear layer's translation units: the description of a product and of what happens to its sums on their way out.
#pragma once
#include "dense.cuh"

namespace n2b {

// forward: z = sum + bias, [z stored], act(z) + add; input gradient: sum * act'(slope_z) + add; weight gradient: fp32, optionally added
// to what is there.  All matrices are indexed (sample, feature) whatever the operands' roles in the product.
struct Epilogue {
	void* out;
	uint64_t out_ld;
	const void *bias, *add, *slope_z;
	uint64_t add_ld, slope_ld;
	void* preact;
	uint64_t preact_ld;
	int act, out_f32, accumulate;
	int vec;  // rows and bias start on 16-byte boundaries everywhere
};

// sum over k of a(m, k) b(n, k).  *_mn: the operand is stored with m (n) contiguous, [k][m], instead of [m][k].
struct Product {
	const void *a, *b;
	uint64_t a_ld, b_ld;
	uint32_t M, N, K;
	bool a_mn, b_mn, bf16;
	Epilogue e;
	float* column_sums;      // weight gradient: sum over k of a(m, k), or null
	void* workspace;         // weight gradient: partial sums
	uint64_t workspace_bytes;
};

// One 16-bit value: the two types share all code paths, the switch is uniform over the grid.
__device__ __forceinline__ float h2f(uint16_t v, bool bf) { return bf ? __uint_as_float((uint32_t)v << 16) : __half2float(__ushort_as_half(v)); }
__device__ __forceinline__ uint16_t f2h(float v, bool bf) {
	return bf ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}
__device__ __forceinline__ void unpack8(const uint4& p, bool bf, float (&v)[8]) {
	const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
	for (int i = 0; i < 4; ++i) {
		if (bf) {
			v[2 * i] = __uint_as_float(w[i] << 16);
			v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
		} else {
			const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
			v[2 * i] = f.x;
			v[2 * i + 1] = f.y;
		}
	}
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8], bool bf) {
	uint32_t w[4];
#pragma unroll
	for (int i = 0; i < 4; ++i) {
		if (bf) {
			const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
			w[i] = *reinterpret_cast<const uint32_t*>(&h);
		} else {
			const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
			w[i] = *reinterpret_cast<const uint32_t*>(&h);
		}
	}
	return make_uint4(w[0], w[1], w[2], w[3]);
}

// one sum, sample r, feature c
__device__ __forceinline__ void finish_one(const Epilogue& e, bool bf, uint64_t r, uint32_t c, float v) {
	if (e.out_f32) {
		float* o = (float*)e.out + r * e.out_ld + c;
		*o = e.accumulate ? *o + v : v;
		return;
	}
	if (e.bias) v += h2f(((const uint16_t*)e.bias)[c], bf);
	if (e.preact) ((uint16_t*)e.preact)[r * e.preact_ld + c] = f2h(v, bf);
	v = e.slope_z ? v * act_slope(e.act, h2f(((const uint16_t*)e.slope_z)[r * e.slope_ld + c], bf)) : act_value(e.act, v);
	if (e.add) v += h2f(((const uint16_t*)e.add)[r * e.add_ld + c], bf);
	((uint16_t*)e.out)[r * e.out_ld + c] = f2h(v, bf);
}

// eight sums, sample r, features c .. c + 7, all of them inside and on 16-byte boundaries
__device__ __forceinline__ void finish_eight(const Epilogue& e, bool bf, uint64_t r, uint32_t c, float (&v)[8]) {
	if (e.out_f32) {
		float4* o = reinterpret_cast<float4*>((float*)e.out + r * e.out_ld + c);
		if (e.accumulate) {
			const float4 a = o[0], b = o[1];
			v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w, v[4] += b.x, v[5] += b.y, v[6] += b.z, v[7] += b.w;
		}
		o[0] = make_float4(v[0], v[1], v[2], v[3]);
		o[1] = make_float4(v[4], v[5], v[6], v[7]);
		return;
	}
	float t[8];
	if (e.bias) {
		unpack8(__ldg(reinterpret_cast<const uint4*>((const uint16_t*)e.bias + c)), bf, t);
#pragma unroll
		for (int i = 0; i < 8; ++i) v[i] += t[i];
	}
	if (e.preact) *reinterpret_cast<uint4*>((uint16_t*)e.preact + r * e.preact_ld + c) = pack8(v, bf);
	if (e.slope_z) {
		unpack8(__ldg(reinterpret_cast<const uint4*>((const uint16_t*)e.slope_z + r * e.slope_ld + c)), bf, t);
		if (e.act == NEUS2B_ACT_RELU) {
#pragma unroll
			for (int i = 0; i < 8; ++i) v[i] *= act_slope(NEUS2B_ACT_RELU, t[i]);
		} else if (e.act == NEUS2B_ACT_GELU) {
#pragma unroll
			for (int i = 0; i < 8; ++i) v[i] *= act_slope(NEUS2B_ACT_GELU, t[i]);
		} else if (e.act == NEUS2B_ACT_SILU) {
#pragma unroll
			for (int i = 0; i < 8; ++i) v[i] *= act_slope(NEUS2B_ACT_SILU, t[i]);
		}
	} else if (e.act == NEUS2B_ACT_RELU) {
#pragma unroll
		for (int i = 0; i < 8; ++i) v[i] = act_value(NEUS2B_ACT_RELU, v[i]);
	} else if (e.act == NEUS2B_ACT_GELU) {
#pragma unroll
		for (int i = 0; i < 8; ++i) v[i] = act_value(NEUS2B_ACT_GELU, v[i]);
	} else if (e.act == NEUS2B_ACT_SILU) {
#pragma unroll
		for (int i = 0; i < 8; ++i) v[i] = act_value(NEUS2B_ACT_SILU, v[i]);
	}
	if (e.add) {
		unpack8(*reinterpret_cast<const uint4*>((const uint16_t*)e.add + r * e.add_ld + c), bf, t);  // may be the output itself
#pragma unroll
		for (int i = 0; i < 8; ++i) v[i] += t[i];
	}
	*reinterpret_cast<uint4*>((uint16_t*)e.out + r * e.out_ld + c) = pack8(v, bf);
}

// width of the product that carries the column sums where no weight gradient is wanted (it is not stored)
inline uint32_t sums_only_width(uint32_t out_width) { return out_width < 64u ? out_width : 64u; }
uint64_t wgrad_workspace(uint32_t out_width, uint32_t in_width, uint32_t n);
int run_product(const Product& p, cudaStream_t stream);         // forward and input gradient; p.M samples, p.N features
int run_weight_gradient(const Product& p, cudaStream_t stream);  // p.M = out_width, p.N = in_width, p.K = n

}  // namespace n2b
