// The bounded wait of the layers' kernels (neus2_b200/csrc/dense.cuh) on barriers that nothing completes: it ends by the clock, or as soon as
// there is no hope, and the barrier is as good as before.  One warp; the kernel ends by itself in a fraction of a second.
#include <stdio.h>

#include "../../neus2_b200/csrc/dense.cuh"

__global__ void wait_kernel(uint64_t limit, unsigned long long* out) {
	__shared__ uint64_t bar;
	const uint32_t b = (uint32_t)__cvta_generic_to_shared(&bar);
	if (threadIdx.x != 0) return;
	asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(b) : "memory");
	uint64_t t = n2b::now_ns();
	out[0] = n2b::wait_phase(b, 0, [] { return false; }, limit);  // nothing has arrived
	out[1] = n2b::now_ns() - t;
	asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(b) : "memory");
	t = n2b::now_ns();
	out[2] = n2b::wait_phase(b, 0);  // complete
	out[3] = n2b::now_ns() - t;
	t = n2b::now_ns();
	out[4] = n2b::wait_phase(b, 1, [] { return true; });  // the next phase, without hope
	out[5] = n2b::now_ns() - t;
}

int main() {
	const uint64_t limit = 100000000;  // a tenth of a second
	unsigned long long *d = nullptr, h[6] = {};
	cudaError_t e = cudaMalloc(&d, sizeof(h));
	if (e == cudaSuccess) {
		wait_kernel<<<1, 32>>>(limit, d);
		e = cudaMemcpy(h, d, sizeof(h), cudaMemcpyDeviceToHost);
		cudaFree(d);
	}
	if (e != cudaSuccess) {
		printf("CUDA: %s\n", cudaGetErrorString(e));
		return 1;
	}
	printf("ran out after %llu us, complete after %llu us, without hope after %llu us\n", h[1] / 1000, h[3] / 1000, h[5] / 1000);
	if (h[0] || h[1] < limit || h[1] > 3000000000ull) return 2;
	if (!h[2] || h[3] > limit) return 3;
	if (h[4] || h[5] > 2000000000ull) return 4;
	printf("bounded wait ok\n");
	return 0;
}
