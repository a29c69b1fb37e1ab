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

// The logistic function of -t ln 2, from the hardware's 2^x and 1/x (2 and 1 units of the last place off): results are rounded to 16
// bits.  2^t overflows to infinity on the far side, where the reciprocal is 0.
__device__ __forceinline__ float logistic2(float t) {
	float e, r;
	asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
	asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
	return r;
}
constexpr float kLog2e = 1.4426950408889634f;
// -2u log2(e), u = sqrt(2 / pi) (z + 0.044715 z^3)
__device__ __forceinline__ float gelu_argument(float z) {
	return z * fmaf(-2.f * kGeluC * kGeluA * kLog2e, z * z, -2.f * kGeluC * kLog2e);
}
__device__ __forceinline__ float act_value(int act, float z) {
	if (act == NEUS2B_ACT_RELU) return z > 0.f ? z : (z != z ? z : 0.f);
	if (act == NEUS2B_ACT_GELU) return z * logistic2(gelu_argument(z));
	if (act == NEUS2B_ACT_SILU) return z * logistic2(-kLog2e * z);
	return z;
}
// v held to +-most, NaN as it is
__device__ __forceinline__ float held(float v, float most) {
	float r;
	asm("min.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(most));
	return r;
}
// d act / dz.  gelu: s + z s (1 - s) 2u' with 2u' = 2 sqrt(2 / pi) (1 + 3 * 0.044715 z^2).  Where z is held, s is exactly 0 or 1 and s (1 - s)
// is 0: the slopes are 0 and 1 for infinite z, too (a preactivation beyond fp16's range is stored as one).
__device__ __forceinline__ float act_slope(int act, float z) {
	if (act == NEUS2B_ACT_RELU) return z > 0.f ? 1.f : 0.f;
	if (act == NEUS2B_ACT_GELU) {
		z = held(z, 1e15f);
		const float s = logistic2(gelu_argument(z));
		return fmaf(z * fmaf(-s, s, s), fmaf(6.f * kGeluC * kGeluA, z * z, 2.f * kGeluC), s);
	}
	if (act == NEUS2B_ACT_SILU) {
		z = held(z, 1e15f);
		const float s = logistic2(-kLog2e * z);
		return fmaf(z, fmaf(-s, s, s), s);
	}
	return 1.f;
}

// Programmatic launches: a kernel launched with `launch_behind` may start while the kernel ahead of it in the stream still runs, from
// where all blocks of that one have called `let_next_start` (or ended).  It has to call `wait_for_previous` in every block before it
// touches memory that others write or read; the call returns when everything ahead in the stream is complete and visible.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <typename... P, typename... A>
int launch_behind_in_clusters(uint32_t cluster, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A... args) {
	cudaLaunchConfig_t cfg{};
	cfg.gridDim = grid;
	cfg.blockDim = block;
	cfg.dynamicSmemBytes = smem;
	cfg.stream = stream;
	cudaLaunchAttribute attr[2];
	attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
	attr[0].val.programmaticStreamSerializationAllowed = 1;
	attr[1].id = cudaLaunchAttributeClusterDimension;
	attr[1].val.clusterDim.x = cluster;
	attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
	cfg.attrs = attr;
	cfg.numAttrs = cluster > 1 ? 2 : 1;
	N2B_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, (P)args...));
	N2B_CHECK_LAUNCH();
	return NEUS2B_OK;
}

template <typename... P, typename... A>
int launch_behind(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A... args) {
	return launch_behind_in_clusters(1, kernel, grid, block, smem, stream, args...);
}

__device__ __forceinline__ uint64_t now_ns() {
	uint64_t t;
	asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
	return t;
}
// Waits for a phase of a barrier in shared memory.  False when it has not completed after `limit`, four seconds, or when `hopeless()` says
// so: nothing that a kernel of these layers waits for takes a millisecond, and every copy that was issued has landed long before a wait
// is given up.
template <typename F>
__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t parity, F hopeless, uint64_t limit = 4000000000ull) {
	uint64_t start = 0;
	for (uint32_t it = 0;; ++it) {
		uint32_t ok;
		asm volatile(
		    "{\n\t.reg .pred p;\n\t"
		    "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
		    "selp.u32 %0, 1, 0, p;\n\t}"
		    : "=r"(ok)
		    : "r"(bar), "r"(parity)
		    : "memory");
		if (ok) return true;
		if ((it & 63u) == 63u) {
			const uint64_t t = now_ns();
			if (!start) start = t;
			else if (t - start > limit || hopeless()) return false;
		}
	}
}
__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t parity) {
	return wait_phase(bar, parity, [] { return false; });
}

// Blocks of a cluster and each other's shared memory
__device__ __forceinline__ uint32_t peer_address(uint32_t addr, uint32_t rank) {
	uint32_t p;
	asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(p) : "r"(addr), "r"(rank));
	return p;
}
__device__ __forceinline__ uint32_t cluster_rank() {
	uint32_t r;
	asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
	return r;
}
__device__ __forceinline__ void cluster_sync() {
	asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float load_peer(uint32_t addr, uint32_t rank) {
	float v;
	asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer_address(addr, rank)) : "memory");
	return v;
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
