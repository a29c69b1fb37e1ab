// Global norm of a set of gradient tensors and clipping by it: norm = |scale| sqrt(sum of squares), factor = min(1, max_norm / norm).
//
// Bound by memory: two reads, of which the second finds what the L2 still holds, and one write.  12.6 M entries of three types 14.8 us, 400
// tensors of 40 M bf16 38 us (4.2 TB/s over one read and one write).  A grid's blocks share out pieces of 16 KB of one tensor each, so that
// many small tensors take no longer than one large one.
#include <stdlib.h>

#include <type_traits>

#include "dense.cuh"

namespace n2b {

// Bytes of one piece at most: 1024 accesses of 16 bytes, four for each of a block's threads, all of them in flight at one time.
constexpr uint32_t kPieceBytes = 16384;

struct Piece {
	const void* in;
	void* out;
	uint32_t n, dtype;
	uint64_t pad;
};

constexpr int kThreads = 256;

// Sum over the block in a fixed order, the same value in every thread.
__device__ __forceinline__ double block_sum(double v, double* s) {
#pragma unroll
	for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
	if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
	__syncthreads();
	v = 0.0;
#pragma unroll
	for (int w = 0; w < kThreads / 32; ++w) v += s[w];
	return v;
}

__device__ __forceinline__ void unpack(const uint4& p, float (&v)[4], const float*) {
	v[0] = __uint_as_float(p.x), v[1] = __uint_as_float(p.y), v[2] = __uint_as_float(p.z), v[3] = __uint_as_float(p.w);
}
__device__ __forceinline__ void unpack(const uint4& p, float (&v)[8], const __half*) {
	const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
	for (int i = 0; i < 4; ++i) {
		const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
		v[2 * i] = f.x, v[2 * i + 1] = f.y;
	}
}
__device__ __forceinline__ void unpack(const uint4& p, float (&v)[8], const __nv_bfloat16*) {
	const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
	for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
__device__ __forceinline__ uint4 pack(const float (&v)[4], const float*) {
	return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
__device__ __forceinline__ uint4 pack(const float (&v)[8], const __half*) {
	uint32_t w[4];
#pragma unroll
	for (int i = 0; i < 4; ++i) {
		const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
		w[i] = *reinterpret_cast<const uint32_t*>(&h);
	}
	return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 pack(const float (&v)[8], const __nv_bfloat16*) {
	uint32_t w[4];
#pragma unroll
	for (int i = 0; i < 4; ++i) {
		const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
		w[i] = *reinterpret_cast<const uint32_t*>(&h);
	}
	return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float square_sum(const float (&v)[4]) { return fmaf(v[0], v[0], v[1] * v[1]) + fmaf(v[2], v[2], v[3] * v[3]); }
__device__ __forceinline__ float square_sum(const float (&v)[8]) {
	return (fmaf(v[0], v[0], v[1] * v[1]) + fmaf(v[2], v[2], v[3] * v[3])) + (fmaf(v[4], v[4], v[5] * v[5]) + fmaf(v[6], v[6], v[7] * v[7]));
}

struct Sum {
	double v = 0.0;
	uint32_t bad = 0;
	bool skip;
	__device__ __forceinline__ void add(float g) {
		const bool odd = !(fabsf(g) <= 3.402823466e38f);
		bad += odd;
		const double d = (double)(odd && skip ? 0.f : g);
		v = fma(d, d, v);
	}
	// The squares of one access are summed in 32 bits, three roundings deep, where that neither overflows nor loses anything below
	// the normal numbers (a sum above 2^-70 is 2^56 times what can be lost), else one by one in 64 bits.  One conversion to 64 bits
	// per access: per entry they cost more than the entries' way from memory.
	template <typename T, int V>
	__device__ __forceinline__ void add(const uint4& raw, const float (&e)[V], const T*) {
		const float q = square_sum(e);
		if (q > 8.5e-22f && q <= 3.402823466e38f) {
			v += (double)q;
		} else if (((raw.x | raw.y | raw.z | raw.w) & (sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu)) != 0) {
#pragma unroll 1
			for (int i = 0; i < V; ++i) add(nth<T>(raw, i));
		}
	}
	template <typename T>
	static __device__ __forceinline__ float nth(const uint4& raw, int i) {
		const int per = 4 / (int)sizeof(T), word = i / per;
		const uint32_t w = word == 0 ? raw.x : word == 1 ? raw.y : word == 2 ? raw.z : raw.w;
		if (sizeof(T) == 4) return __uint_as_float(w);
		const uint16_t h = (uint16_t)(w >> (16 * (i & 1)));
		return to_f(*reinterpret_cast<const T*>(&h));
	}
};

// A piece, as a block's threads see it: what lies in front of the first 16-byte boundary and behind the last one goes entry by entry, the
// rest 16 bytes at a time.  `joint`: the output reaches a boundary at the same entry as the input; else everything goes entry by entry.
struct View {
	uint32_t head, vecs;
	template <typename T>
	__device__ __forceinline__ View(const Piece& p, const T*, bool joint) {
		const uint32_t lead = (uint32_t)((16u - ((uintptr_t)p.in & 15u)) & 15u) / (uint32_t)sizeof(T);
		head = !joint || lead > p.n ? p.n : lead;
		vecs = (p.n - head) / (16 / (uint32_t)sizeof(T));
	}
};
template <typename T>
__device__ __forceinline__ void load_piece(const Piece& p, const View& w, uint4 (&r)[4]) {
	const uint4* q = reinterpret_cast<const uint4*>((const T*)p.in + w.head);
#pragma unroll
	for (int k = 0; k < 4; ++k) r[k] = threadIdx.x + k * kThreads < w.vecs ? q[threadIdx.x + k * kThreads] : make_uint4(0, 0, 0, 0);
}
template <typename T>
__device__ __forceinline__ void sum_piece(const Piece& p, Sum& sum) {
	constexpr int V = 16 / sizeof(T);
	const View w(p, (const T*)nullptr, true);
	uint4 r[4];
	load_piece<T>(p, w, r);
	const T* in = (const T*)p.in;
	if (threadIdx.x < w.head) sum.add(to_f(in[threadIdx.x]));
	const uint32_t tail = w.head + w.vecs * V + threadIdx.x;
	if (tail < p.n) sum.add(to_f(in[tail]));
#pragma unroll
	for (int k = 0; k < 4; ++k) {
		float v[V];
		unpack(r[k], v, (const T*)nullptr);
		sum.add(r[k], v, (const T*)nullptr);
	}
}
template <typename T>
__device__ __forceinline__ void scale_piece(const Piece& p, const View& w, const uint4 (&r)[4], float c) {
	constexpr int V = 16 / sizeof(T);
	const T* in = (const T*)p.in;
	T* out = (T*)p.out;
	for (uint32_t i = threadIdx.x; i < w.head; i += kThreads) out[i] = from_f<T>(to_f(in[i]) * c);
	const uint32_t tail = w.head + w.vecs * V + threadIdx.x;
	if (tail < p.n) out[tail] = from_f<T>(to_f(in[tail]) * c);
	uint4* q = reinterpret_cast<uint4*>(out + w.head);
#pragma unroll
	for (int k = 0; k < 4; ++k) {
		float v[V];
		unpack(r[k], v, (const T*)nullptr);
#pragma unroll
		for (int e = 0; e < V; ++e) v[e] *= c;
		if (threadIdx.x + k * kThreads < w.vecs) q[threadIdx.x + k * kThreads] = pack(v, (const T*)nullptr);
	}
}
template <typename F>
__device__ __forceinline__ void by_type(uint32_t dtype, F f) {
	if (dtype == NEUS2B_F32) f((const float*)nullptr);
	else if (dtype == NEUS2B_F16) f((const __half*)nullptr);
	else f((const __nv_bfloat16*)nullptr);
}

__global__ void __launch_bounds__(kThreads, 6) norm_partial_kernel(const Piece* __restrict__ pieces, uint32_t n_pieces, uint32_t flags,
                                                                    double* __restrict__ partial, uint32_t* __restrict__ nonfinite) {
	__shared__ double s[kThreads / 32];
	wait_for_previous();
	let_next_start();  // the clipping kernel may start on what does not depend on the sums: the gradients, which are complete from here on
	Sum sum;
	sum.skip = flags & NEUS2B_NORM_SKIP_NONFINITE;
	Piece p{};
	if (blockIdx.x < n_pieces) p = pieces[blockIdx.x];
	for (uint32_t k = blockIdx.x; k < n_pieces; k += gridDim.x) {
		const Piece now = p;
		if (k + gridDim.x < n_pieces) p = pieces[k + gridDim.x];
		by_type(now.dtype, [&](auto t) { sum_piece<typename std::remove_const<typename std::remove_pointer<decltype(t)>::type>::type>(now, sum); });
	}
	const double v = block_sum(sum.v, s);
	if (threadIdx.x == 0) partial[blockIdx.x] = v;
	if (nonfinite && sum.bad) atomicAdd(nonfinite, sum.bad);
}

// Every block of the clipping kernel adds up the blocks' sums again, in the same order: cheaper than a launch in between.
__device__ __forceinline__ float2 norm_and_factor(const double* __restrict__ partial, uint32_t n, float scale, float max_norm) {
	__shared__ double s[kThreads / 32];
	double v = 0.0;
	for (uint32_t i = threadIdx.x; i < n; i += kThreads) v += partial[i];
	v = fabs((double)scale) * sqrt(block_sum(v, s));
	return make_float2((float)v, v > (double)max_norm && isfinite(v) ? (float)((double)max_norm / v) : 1.f);
}

__global__ void __launch_bounds__(kThreads) norm_final_kernel(const double* __restrict__ partial, uint32_t n, float scale, float max_norm, float* __restrict__ result) {
	wait_for_previous();
	const float2 r = norm_and_factor(partial, n, scale, max_norm);
	if (threadIdx.x == 0) result[0] = r.x, result[1] = r.y;
}

// Launched so that it may start while the sums are still being taken: each block fetches its first piece before it waits for them.
// The pieces are taken from the end: those that the norm read last are still in the L2 (40 M bf16 in 400 tensors: 38.3 us, from the
// beginning 40.5).
__global__ void __launch_bounds__(kThreads, 5) clip_kernel(const Piece* __restrict__ pieces, uint32_t n_pieces, const double* __restrict__ partial,
                                                            uint32_t n_partial, float scale, float max_norm, float* __restrict__ result) {
	uint4 r[4];
	Piece p = pieces[n_pieces - 1 - blockIdx.x];
	auto load = [&](const Piece& q) {
		by_type(q.dtype, [&](auto t) {
			using T = typename std::remove_const<typename std::remove_pointer<decltype(t)>::type>::type;
			if (q.out) load_piece<T>(q, View(q, t, (((uintptr_t)q.in ^ (uintptr_t)q.out) & 15u) == 0), r);
		});
	};
	load(p);
	wait_for_previous();
	const float2 f = norm_and_factor(partial, n_partial, scale, max_norm);
	if (blockIdx.x == 0 && threadIdx.x == 0) result[0] = f.x, result[1] = f.y;
	const float c = f.y;
	for (uint32_t k = blockIdx.x; k < n_pieces; k += gridDim.x) {
		if (p.out && !(p.out == p.in && c == 1.f))
			by_type(p.dtype, [&](auto t) {
				using T = typename std::remove_const<typename std::remove_pointer<decltype(t)>::type>::type;
				scale_piece<T>(p, View(p, t, (((uintptr_t)p.in ^ (uintptr_t)p.out) & 15u) == 0), r, c);
			});
		if (k + gridDim.x < n_pieces) {
			p = pieces[n_pieces - 1 - k - gridDim.x];
			if (!(p.out == p.in && c == 1.f)) load(p);
		}
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

constexpr uint32_t kNormBlocks = 6u * kSMs, kClipBlocks = 5u * kSMs;
static uint32_t blocks_for(uint32_t n_pieces) { return n_pieces < kNormBlocks ? n_pieces : kNormBlocks; }

static int run(const void* d_table, uint32_t n_pieces, float scale, float max_norm, uint32_t flags, float* d_result, uint32_t* d_nonfinite, void* d_workspace,
               uint64_t workspace_bytes, bool clip, cudaStream_t s) {
	if (!d_result || ((uintptr_t)d_result & 3) || ((uintptr_t)d_nonfinite & 3) || (flags & ~NEUS2B_NORM_SKIP_NONFINITE)) return NEUS2B_E_INVALID;
	if (!(max_norm > 0.f) || !isfinite(scale)) return NEUS2B_E_INVALID;
	if (n_pieces > 0x7fffffffu) return NEUS2B_E_TOO_LARGE;
	if (!d_workspace || ((uintptr_t)d_workspace & 15) || workspace_bytes < neus2b_grad_norm_workspace(n_pieces)) return NEUS2B_E_INVALID;
	if (n_pieces && (!d_table || ((uintptr_t)d_table & 15))) return NEUS2B_E_INVALID;
	const uint32_t blocks = blocks_for(n_pieces);
	if (blocks) {
		if (int rc = launch_behind(norm_partial_kernel, blocks, kThreads, 0, s, (const Piece*)d_table, n_pieces, flags, (double*)d_workspace, d_nonfinite)) return rc;
	}
	if (clip && blocks) {
		return launch_behind(clip_kernel, n_pieces < kClipBlocks ? n_pieces : kClipBlocks, kThreads, 0, s, (const Piece*)d_table, n_pieces,
		                     (const double*)d_workspace, blocks, scale, max_norm, d_result);
	}
	return launch_behind(norm_final_kernel, 1, kThreads, 0, s, (const double*)d_workspace, blocks, scale, max_norm, d_result);
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
		const uint64_t entries = kPieceBytes / b, pieces = (g.n + entries - 1) / entries;
		if (count + pieces > 0x7fffffffull) return NEUS2B_E_TOO_LARGE;
		for (uint64_t k = 0; p && k < pieces; ++k) {
			const uint64_t at = k * entries;
			p[count + k] = Piece{(const char*)g.d_in + at * b, g.d_out ? (char*)g.d_out + at * b : nullptr, (uint32_t)(g.n - at < entries ? g.n - at : entries),
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
