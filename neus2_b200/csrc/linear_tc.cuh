// What the linear layer's tcgen05 kernels share: barriers, TMA, tensor memory, descriptors, tensor maps, the epilogue's arithmetic.
#pragma once
#include <cuda.h>

#include "linear.cuh"
#include "tc05.cuh"

namespace n2b {
namespace lin {

constexpr int kBM = 128, kBK = 64;
constexpr int kMaxStages = 8, kSmemMost = 227 * 1024;

__device__ __forceinline__ uint32_t sptr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void arrive_expect(uint32_t bar, uint32_t bytes) {
	asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// x: first column (a multiple of 64), y: first row of a [rows][columns] matrix.  PAIR: the barrier may be the other CTA's.
template <bool PAIR>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
	if (PAIR)
		asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map),
		             "r"(x), "r"(y), "r"(bar)
		             : "memory");
	else
		asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map),
		             "r"(x), "r"(y), "r"(bar)
		             : "memory");
}
// At a barrier of the cluster, for what the arriving thread has read (its loads have returned): relaxed, since a release would wait for its stores
// too (a pair's epilogue, 26620 x 144 -> 912: 24 us, relaxed 18.4).
__device__ __forceinline__ void arrive_remote(uint32_t bar) {
	asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void tmem_alloc(uint32_t dst, uint32_t cols) {
	if (PAIR) {
		asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(cols) : "memory");
		asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
	} else {
		tc::tmem_alloc(dst, cols);
	}
}
template <bool PAIR>
__device__ __forceinline__ void tmem_dealloc(uint32_t addr, uint32_t cols) {
	if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
	else tc::tmem_dealloc(addr, cols);
}
template <bool PAIR>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t more) {
	if (PAIR)
		asm volatile(
		    "{\n\t.reg .pred p;\n\t"
		    "setp.ne.b32 p, %4, 0;\n\t"
		    "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
		    :
		    : "r"(d), "l"(a), "l"(b), "r"(id), "r"(more)
		    : "memory");
	else tc::mma_f16(d, a, b, id, more);
}
// PAIR: arrives at the barrier of this place in both CTAs.
template <bool PAIR>
__device__ __forceinline__ void commit(uint32_t bar) {
	if (PAIR)
		asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
	else tc::commit(bar);
}
// Matrix descriptors of the two 128-byte-swizzled layouts.  K-major: rows of 64 k, 8-row groups 1024 bytes apart.  MN-major: rows of
// 64 m (or n), one per k, 8-row groups 1024 bytes apart, slabs of 64 m 8192 bytes apart.
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) {
	return (uint64_t)((addr >> 4) & 0x3FFFu) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr) {
	return (uint64_t)((addr >> 4) & 0x3FFFu) | (512ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void tmem_ld16_raw(uint32_t taddr, uint32_t (&r)[16]) {
	asm volatile(
	    "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
	    : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
	      "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
	    : "r"(taddr)
	    : "memory");
}
__device__ __forceinline__ void tmem_wait16(uint32_t (&r)[16]) {
	asm volatile("tcgen05.wait::ld.sync.aligned;"
	             : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
	               "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}
__device__ __forceinline__ float2 unpack2(uint32_t w, bool bf) {
	return bf ? make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)) : __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, bool bf) {
	if (bf) {
		const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
		return *reinterpret_cast<const uint32_t*>(&h);
	}
	const __half2 h = __floats2half2_rn(a, b);
	return *reinterpret_cast<const uint32_t*>(&h);
}
template <int ACT>
__device__ __forceinline__ void apply_act(float (&v)[32]) {
#pragma unroll
	for (int i = 0; i < 32; ++i) v[i] = act_value(ACT, v[i]);
}
template <int ACT>
__device__ __forceinline__ void apply_slope(float (&v)[32], const uint32_t (&z)[16], bool bf) {
#pragma unroll
	for (int i = 0; i < 16; ++i) {
		const float2 f = unpack2(z[i], bf);
		v[2 * i] *= act_slope(ACT, f.x);
		v[2 * i + 1] *= act_slope(ACT, f.y);
	}
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                             CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static inline EncodeFn encode_fn() {
	static EncodeFn fn = [] {
		void* q = nullptr;
		cudaDriverEntryPointQueryResult res;
		if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &q, 12000, cudaEnableDefault, &res) != cudaSuccess) q = nullptr;
		return (EncodeFn)q;
	}();
	return fn;
}
// [rows][cols] matrix read in boxes of 64 columns and box_rows rows
static inline int make_map(CUtensorMap* map, const void* base, uint64_t ld, uint32_t rows, uint32_t cols, uint32_t box_rows, bool bf16) {
	const EncodeFn fn = encode_fn();
	if (!fn) return NEUS2B_E_NO_DEVICE;
	const cuuint64_t dims[2] = {cols, rows}, strides[1] = {ld * 2};
	const cuuint32_t box[2] = {64, box_rows}, unit[2] = {1, 1};
	const CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base), dims, strides, box, unit,
	                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
	return r == CUDA_SUCCESS ? NEUS2B_OK : NEUS2B_E_INVALID;
}
// TMA reads rows that start on 16-byte boundaries, less than 2^40 bytes apart
static inline bool tma_ok(const void* p, uint64_t ld) { return ((uintptr_t)p & 15u) == 0 && (ld & 7u) == 0 && ld < (1ull << 39); }

static inline uint32_t tiles_of(uint32_t n, uint32_t size) { return (n + size - 1) / size; }

}  // namespace lin
}  // namespace n2b
