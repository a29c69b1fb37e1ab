// "ResidualMLP" of the tiny-cuda-nn-shaped headers on an empty batch: its gradient is 0, so that Overwrite clears what an earlier batch left,
// and Accumulate and Ignore leave it.
#include <tiny-cuda-nn/common_device.h>
#include <tiny-cuda-nn/network.h>

#include <cstdio>

using namespace tcnn;
using T = __half;

static std::vector<float> gradients(const GPUMemory<T>& g) {
	std::vector<T> h(g.size());
	CUDA_CHECK_THROW(cudaMemcpy(h.data(), g.data(), h.size() * sizeof(T), cudaMemcpyDeviceToHost));
	std::vector<float> f;
	for (const T& v : h) f.push_back(__half2float(v));
	return f;
}

int main() {
	cudaStream_t stream;
	CUDA_CHECK_THROW(cudaStreamCreate(&stream));
	int failed = 0;
	{
		std::unique_ptr<Network<T>> network{
		    create_network<T>({{"otype", "ResidualMLP"}, {"n_input_dims", 32}, {"n_output_dims", 16}, {"n_neurons", 64}, {"n_hidden_layers", 1}, {"activation", "GELU"}})};
		const size_t count = network->n_params();
		GPUMemory<T> p(count), g(count);
		p.memset(0);
		network->set_params(p.data(), p.data(), nullptr, g.data());
		GPUMatrixDynamic<T> x{32, 0, stream}, y{16, 0, stream}, dy{16, 0, stream}, dx{32, 0, stream};
		auto ctx = network->forward(stream, x, &y, false, true);
		for (const auto mode : {EGradientMode::Accumulate, EGradientMode::Ignore, EGradientMode::Overwrite}) {
			CUDA_CHECK_THROW(cudaMemset(g.data(), 0x3c, count * sizeof(T)));  // 1.06 everywhere
			network->backward(stream, *ctx, x, y, dy, &dx, false, mode);
			CUDA_CHECK_THROW(cudaStreamSynchronize(stream));
			const float want = mode == EGradientMode::Overwrite ? 0.f : 1.05859375f;
			size_t off = 0;
			for (const float v : gradients(g)) off += v != want;
			if (off) {
				std::printf("FAILED: mode %d, %zu of %zu gradients\n", (int)mode, off, count);
				failed = 1;
			}
		}
	}
	CUDA_CHECK_THROW(cudaStreamDestroy(stream));
	std::printf(failed ? "empty batches FAILED\n" : "empty batches ok\n");
	return failed;
}
