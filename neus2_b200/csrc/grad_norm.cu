// Global norm of a set of gradient tensors and clipping by it.
#include <stdlib.h>

#include "dense.cuh"

namespace n2b {

constexpr uint32_t kPiece = 8192;  // entries of one piece at most

struct Piece {
	const void* in;
	void* out;
	uint32_t n, dtype;
	uint64_t pad;
};

template <typename F>
__device__ __forceinline__ void each_entry(const Piece& p, F f) {
	if (p.dtype == NEUS2B_F32)
		for (uint32_t i = threadIdx.x; i < p.n; i += blockDim.x) f(i, (const float*)p.in, (float*)p.out);
	else if (p.dtype == NEUS2B_F16)
		for (uint32_t i = threadIdx.x; i < p.n; i += blockDim.x) f(i, (const __half*)p.in, (__half*)p.out);
	else
		for (uint32_t i = threadIdx.x; i < p.n; i += blockDim.x) f(i, (const __nv_bfloat16*)p.in, (__nv_bfloat16*)p.out);
}

__device__ __forceinline__ double block_sum(double v, double* s) {
#pragma unroll
	for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
	if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
	__syncthreads();
	v = 0.0;
	for (int w = 0; w < (int)(blockDim.x >> 5); ++w) v += s[w];
	return v;
}

__global__ void __launch_bounds__(256) norm_partial_kernel(const Piece* __restrict__ pieces, uint32_t n_pieces, uint32_t flags, double* __restrict__ partial,
                                                            uint32_t* __restrict__ nonfinite) {
	__shared__ double s[8];
	double v = 0.0;
	uint32_t bad = 0;
	for (uint32_t k = blockIdx.x; k < n_pieces; k += gridDim.x) {
		const Piece p = pieces[k];
		each_entry(p, [&](uint32_t i, auto in, auto) {
			const float g = to_f(in[i]);
			const bool odd = !(fabsf(g) <= 3.402823466e38f);
			bad += odd;
			if (!odd || !(flags & NEUS2B_NORM_SKIP_NONFINITE)) v = fma((double)g, (double)g, v);
		});
	}
	v = block_sum(v, s);
	if (threadIdx.x == 0) partial[blockIdx.x] = v;
	if (nonfinite && bad) atomicAdd(nonfinite, bad);
}

__global__ void __launch_bounds__(256) norm_final_kernel(const double* __restrict__ partial, uint32_t n, float scale, float max_norm, float* __restrict__ result) {
	__shared__ double s[8];
	double v = 0.0;
	for (uint32_t i = threadIdx.x; i < n; i += 256) v += partial[i];
	v = fabs((double)scale) * sqrt(block_sum(v, s));
	if (threadIdx.x == 0) {
		result[0] = (float)v;
		result[1] = (v > (double)max_norm && isfinite(v)) ? (float)((double)max_norm / v) : 1.f;
	}
}

__global__ void __launch_bounds__(256) clip_kernel(const Piece* __restrict__ pieces, uint32_t n_pieces, const float* __restrict__ result) {
	const float c = result[1];
	for (uint32_t k = blockIdx.x; k < n_pieces; k += gridDim.x) {
		const Piece p = pieces[k];
		if (!p.out || (p.out == p.in && c == 1.f)) continue;
		each_entry(p, [&](uint32_t i, auto in, auto out) {
			using T = typename std::remove_pointer<decltype(out)>::type;
			out[i] = from_f<T>(to_f(in[i]) * c);
		});
	}
}

struct Range {
	uintptr_t begin, end;
	bool written;
};
static int by_begin(const void* a, const void* b) {
	const uintptr_t x = ((const Range*)a)->begin, y = ((const Range*)b)->begin;
	return x < y ? -1 : x > y;
}
// An output that overlaps another output, or an input other than its own in place, would be read and written by different pieces.
static int check_ranges(const neus2b_grad_tensor* t, uint32_t n) {
	Range* r = (Range*)malloc(sizeof(Range) * 2 * ((size_t)n + 1));
	if (!r) return NEUS2B_E_TOO_LARGE;
	size_t count = 0;
	for (uint32_t i = 0; i < n; ++i) {
		if (!t[i].n) continue;
		const size_t bytes = t[i].n * dtype_bytes(t[i].dtype);
		const uintptr_t in = (uintptr_t)t[i].d_in, out = (uintptr_t)t[i].d_out;
		if (in != out) r[count++] = Range{in, in + bytes, false};
		if (out) r[count++] = Range{out, out + bytes, true};
	}
	qsort(r, count, sizeof(Range), by_begin);
	uintptr_t read_end = 0, written_end = 0;
	int rc = NEUS2B_OK;
	for (size_t i = 0; i < count; ++i) {
		if (r[i].begin < written_end || (r[i].written && r[i].begin < read_end)) rc = NEUS2B_E_INVALID;
		uintptr_t& end = r[i].written ? written_end : read_end;
		if (r[i].end > end) end = r[i].end;
	}
	free(r);
	return rc;
}

constexpr uint32_t kNormBlocks = 8u * kSMs;
static uint32_t blocks_for(uint32_t n_pieces) { return n_pieces < kNormBlocks ? n_pieces : kNormBlocks; }

static int run(const void* d_table, uint32_t n_pieces, float scale, float max_norm, uint32_t flags, float* d_result, uint32_t* d_nonfinite, void* d_workspace,
               uint64_t workspace_bytes, bool clip, cudaStream_t s) {
	if (!d_result || ((uintptr_t)d_result & 3) || ((uintptr_t)d_nonfinite & 3) || (flags & ~NEUS2B_NORM_SKIP_NONFINITE)) return NEUS2B_E_INVALID;
	if (!(max_norm > 0.f) || !isfinite(scale)) return NEUS2B_E_INVALID;
	if (!d_workspace || ((uintptr_t)d_workspace & 15) || workspace_bytes < neus2b_grad_norm_workspace(n_pieces)) return NEUS2B_E_INVALID;
	if (n_pieces && (!d_table || ((uintptr_t)d_table & 15))) return NEUS2B_E_INVALID;
	const uint32_t blocks = blocks_for(n_pieces);
	if (blocks) {
		norm_partial_kernel<<<blocks, 256, 0, s>>>((const Piece*)d_table, n_pieces, flags, (double*)d_workspace, d_nonfinite);
		N2B_CHECK_LAUNCH();
	}
	norm_final_kernel<<<1, 256, 0, s>>>((const double*)d_workspace, blocks, scale, max_norm, d_result);
	N2B_CHECK_LAUNCH();
	if (clip && blocks) {
		clip_kernel<<<blocks, 256, 0, s>>>((const Piece*)d_table, n_pieces, d_result);
		N2B_CHECK_LAUNCH();
	}
	return NEUS2B_OK;
}

}  // namespace n2b

using namespace n2b;

extern "C" int neus2b_grad_table(const neus2b_grad_tensor* h_tensors, uint32_t n_tensors, void* h_table, uint64_t* table_bytes, uint32_t* n_pieces) {
	if ((n_tensors && !h_tensors) || !table_bytes || !n_pieces) return NEUS2B_E_INVALID;
	uint64_t count = 0;
	Piece* p = (Piece*)h_table;
	for (uint32_t t = 0; t < n_tensors; ++t) {
		const neus2b_grad_tensor& g = h_tensors[t];
		if (g.dtype > NEUS2B_BF16) return NEUS2B_E_UNSUPPORTED;
		const size_t b = dtype_bytes(g.dtype);
		if (g.n && (!g.d_in || (((uintptr_t)g.d_in | (uintptr_t)g.d_out) & (b - 1)))) return NEUS2B_E_INVALID;
		if (g.n > (1ull << 60)) return NEUS2B_E_TOO_LARGE;
		const uint64_t pieces = (g.n + kPiece - 1) / kPiece;
		if (count + pieces > 0xffffffffull) return NEUS2B_E_TOO_LARGE;
		for (uint64_t k = 0; p && k < pieces; ++k) {
			const uint64_t at = k * kPiece;
			p[count + k] = Piece{(const char*)g.d_in + at * b, g.d_out ? (char*)g.d_out + at * b : nullptr, (uint32_t)(g.n - at < kPiece ? g.n - at : kPiece),
			                     g.dtype, 0};
		}
		count += pieces;
	}
	if (p)
		if (int rc = check_ranges(h_tensors, n_tensors)) return rc;
	*table_bytes = count * sizeof(Piece);
	*n_pieces = (uint32_t)count;
	return NEUS2B_OK;
}

extern "C" uint64_t neus2b_grad_norm_workspace(uint32_t n_pieces) { return (uint64_t)(n_pieces ? blocks_for(n_pieces) : 1u) * sizeof(double) + 16; }

extern "C" int neus2b_grad_norm(const void* d_table, uint32_t n_pieces, float scale, float max_norm, uint32_t flags, float* d_result,
                                uint32_t* d_nonfinite, void* d_workspace, uint64_t workspace_bytes, neus2b_stream_t stream) {
	return run(d_table, n_pieces, scale, max_norm, flags, d_result, d_nonfinite, d_workspace, workspace_bytes, false, stream);
}

extern "C" int neus2b_grad_clip(const void* d_table, uint32_t n_pieces, float scale, float max_norm, uint32_t flags, float* d_result,
                                uint32_t* d_nonfinite, void* d_workspace, uint64_t workspace_bytes, neus2b_stream_t stream) {
	return run(d_table, n_pieces, scale, max_norm, flags, d_result, d_nonfinite, d_workspace, workspace_bytes, true, stream);
}
