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
	int vec;  // bytes of an access that every row and the bias allow: 16, 4 (16-bit matrices) or less
};

// sum over k of a(m, k) b(n, k).  b_mn: b is stored with n contiguous, [k][n], instead of [n][k] (the weight gradient: both are).
struct Product {
	const void *a, *b;
	uint64_t a_ld, b_ld;
	uint32_t M, N, K;
	bool b_mn, bf16;
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

// sum over the rows of a [rows][cols] matrix with rows on 16-byte boundaries
int run_column_sums(const void* a, uint64_t ld, uint32_t rows, uint32_t cols, bool bf16, float* out, int accumulate, cudaStream_t stream);
uint64_t wgrad_workspace(uint32_t out_width, uint32_t in_width, uint32_t n);
// sums of `splits` parts [M][N] (to out) and, behind all of them, of `splits` parts [M] (to sums, if not null)
int run_join(const float* partial, uint32_t splits, uint32_t M, uint32_t N, float* out, float* sums, int accumulate, cudaStream_t stream);
// Results of up to 64 columns (linear_narrow.cu).  forward or input gradient: `rows` the product for dL/dx or y, `weights` null or the
// weight gradient that shares its first operand.
bool narrow_fits(const Product& rows, bool backward, const Product* weights);
uint64_t narrow_workspace(uint32_t out_width, uint32_t in_width, uint32_t n);
int run_narrow(const Product& rows, bool backward, const Product* weights, cudaStream_t stream);
int read_narrow_error(uint32_t* flags);
int write_narrow_error(uint32_t flags);
// Rows on 16-byte boundaries, as the product kernels read them.
struct Operand {
	const void* from;
	uint64_t ld;
	uint32_t rows, cols;
	void* to;  // [rows][cols rounded up to 8]
};
bool operand_aligned(const void* p, uint64_t ld);
int run_realign(const Operand* ops, int count, cudaStream_t stream);  // three at most
int run_product(const Product& p, cudaStream_t stream);         // forward and input gradient; p.M samples, p.N features
int run_weight_gradient(const Product& p, cudaStream_t stream);  // p.M = out_width, p.N = in_width, p.K = n

}  // namespace n2b
