// The "ResidualMLP" network of the tiny-cuda-nn-shaped headers: what its factory refuses, its forward pass and every gradient against a
// 64-bit restatement on the host, an encoding in front of it, and training steps.
#include <tiny-cuda-nn/common_device.h>
#include <tiny-cuda-nn/network_with_input_encoding.h>
#include <tiny-cuda-nn/trainer.h>

#include <cstdio>
#include <cstring>
#include <random>

using namespace tcnn;
using T = __half;

static int g_failed = 0;
#define EXPECT(c)                                                    \
	do {                                                             \
		if (!(c)) {                                                  \
			std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #c); \
			++g_failed;                                              \
		}                                                            \
	} while (0)
template <typename F>
static bool throws(F f) {
	try {
		f();
	} catch (const std::exception&) {
		return true;
	}
	return false;
}
template <typename V>
static std::vector<V> to_host(const V* p, size_t n) {
	std::vector<V> h(n);
	CUDA_CHECK_THROW(cudaMemcpy(h.data(), p, n * sizeof(V), cudaMemcpyDeviceToHost));
	return h;
}
static json net(uint32_t in, uint32_t out, uint32_t neurons, uint32_t blocks, const char* act) {
	return {{"otype", "ResidualMLP"}, {"n_input_dims", in}, {"n_output_dims", out}, {"n_neurons", neurons}, {"n_hidden_layers", blocks}, {"activation", act}};
}

// ---- the network in 64 bits: parameters in the block's order, x [n][in] -> y [n][out]
struct Plain {
	int in, out, W, L, act;
	size_t sq() const { return (size_t)W * W; }
	size_t w1(int l) const { return (size_t)W * in + 2 * l * sq(); }
	size_t w_out() const { return w1(L); }
	size_t b_in() const { return w_out() + (size_t)out * W; }
	size_t gamma(int l) const { return b_in() + W + (size_t)4 * l * W; }
	size_t b_out() const { return gamma(L) + 2 * (size_t)W; }
	size_t n_params() const { return b_out() + out; }
	double activate(double z) const {
		if (act == 1) return z > 0 ? z : 0;
		if (act == 2) return 0.5 * z * (1 + std::tanh(std::sqrt(2 / M_PI) * (z + 0.044715 * z * z * z)));
		if (act == 3) return z / (1 + std::exp(-z));
		return z;
	}
	void product(const double* p, size_t w, size_t b, const std::vector<double>& x, std::vector<double>& y, int rows) const {
		y.resize(rows);
		for (int r = 0; r < rows; ++r) {
			double s = p[b + r];
			for (size_t k = 0; k < x.size(); ++k) s += p[w + r * x.size() + k] * x[k];
			y[r] = s;
		}
	}
	void norm(const double* p, int l, const std::vector<double>& h, std::vector<double>& a) const {
		double m = 0, v = 0;
		for (double q : h) m += q / W;
		for (double q : h) v += (q - m) * (q - m) / W;
		a.resize(W);
		for (int c = 0; c < W; ++c) a[c] = p[gamma(l) + c] * (h[c] - m) / std::sqrt(v + 1e-5) + p[gamma(l) + W + c];
	}
	std::vector<double> run(const double* p, const double* x0) const {
		std::vector<double> x(x0, x0 + in), h, a, u, d;
		product(p, 0, b_in(), x, h, W);
		for (int l = 0; l < L; ++l) {
			norm(p, l, h, a);
			product(p, w1(l), gamma(l) + 2 * W, a, u, W);
			for (double& q : u) q = activate(q);
			product(p, w1(l) + sq(), gamma(l) + 3 * W, u, d, W);
			for (int c = 0; c < W; ++c) h[c] += d[c];
		}
		norm(p, L, h, a);
		product(p, w_out(), b_out(), a, d, out);
		return d;
	}
};

static void check_network(uint32_t in, uint32_t out, uint32_t W, uint32_t L, const char* act_name, int act, uint32_t n, cudaStream_t stream, std::mt19937& rng) {
	std::unique_ptr<Network<T>> network{create_network<T>(net(in, out, W, L, act_name))};
	const uint32_t padded = network->padded_output_width();
	Plain plain{(int)in, (int)padded, (int)W, (int)L, act};
	EXPECT(network->n_params() == plain.n_params() && padded == (out + 15) / 16 * 16);
	std::normal_distribution<float> nd(0.f, 1.f);
	std::vector<T> hp(plain.n_params()), hx((size_t)n * in), hdy((size_t)n * padded);
	for (size_t i = 0; i < hp.size(); ++i) hp[i] = __float2half(i < plain.b_in() ? nd(rng) * 1.2f / std::sqrt((float)W) : 0.2f * nd(rng));
	for (uint32_t l = 0; l <= L; ++l)
		for (uint32_t c = 0; c < W; ++c) hp[plain.gamma(l) + c] = __float2half(1.f + 0.2f * nd(rng));
	for (auto& v : hx) v = __float2half(nd(rng));
	for (auto& v : hdy) v = __float2half(nd(rng) / std::sqrt((float)n));
	GPUMemory<T> p, g(hp.size()), x, dy;
	p.resize_and_copy_from_host(hp);
	x.resize_and_copy_from_host(hx);
	dy.resize_and_copy_from_host(hdy);
	g.memset(0);
	network->set_params(p.data(), p.data(), nullptr, g.data());
	GPUMatrixDynamic<T> X(x.data(), in, n), dY(dy.data(), padded, n), Y{padded, n, stream}, dX{in, n, stream};
	auto ctx = network->forward(stream, X, &Y, false, true);
	network->backward(stream, *ctx, X, Y, dY, &dX, false, EGradientMode::Overwrite);
	CUDA_CHECK_THROW(cudaStreamSynchronize(stream));
	auto y = to_host(Y.data(), (size_t)n * padded), gp = to_host(g.data(), hp.size()), dx = to_host(dX.data(), (size_t)n * in);

	std::vector<double> dp(hp.size()), xs(hx.size());
	for (size_t i = 0; i < dp.size(); ++i) dp[i] = __half2float(hp[i]);
	for (size_t i = 0; i < xs.size(); ++i) xs[i] = __half2float(hx[i]);
	// outputs: 3 L + 3 roundings to 11 bits on the way, each spread over the row by products of norm about one
	double err = 0, ref = 0;
	for (uint32_t i = 0; i < n; ++i) {
		const auto want = plain.run(dp.data(), &xs[(size_t)i * in]);
		for (uint32_t c = 0; c < padded; ++c) {
			const double d = __half2float(y[(size_t)i * padded + c]) - want[c];
			err += d * d, ref += want[c] * want[c];
		}
	}
	const double steps = std::sqrt(3.0 * L + 3) * std::ldexp(1.0, -11);
	EXPECT(std::sqrt(err / ref) < 4 * steps);

	// gradients of sum(dy * y): central differences in 64 bits at a few entries of every tensor
	auto loss_row = [&](const double* q, const double* row, uint32_t i) {
		const auto o = plain.run(q, row);
		double s = 0;
		for (uint32_t c = 0; c < padded; ++c) s += o[c] * __half2float(hdy[(size_t)i * padded + c]);
		return s;
	};
	struct Span {
		size_t at, n;
	};
	std::vector<Span> spans{{0, (size_t)W * in}, {plain.w_out(), (size_t)padded * W}, {plain.b_in(), W}, {plain.b_out(), padded}};
	for (uint32_t l = 0; l < L; ++l) {
		spans.push_back({plain.w1(l), plain.sq()});
		spans.push_back({plain.w1(l) + plain.sq(), plain.sq()});
		for (int k = 0; k < 4; ++k) spans.push_back({plain.gamma(l) + (size_t)k * W, W});
	}
	for (int k = 0; k < 2; ++k) spans.push_back({plain.gamma(L) + (size_t)k * W, W});
	for (const Span& s : spans) {
		double rms = 0;
		for (size_t i = 0; i < s.n; ++i) rms += std::pow((double)__half2float(gp[s.at + i]), 2);
		rms = std::sqrt(rms / s.n);
		EXPECT(rms > 0);
		for (int k = 0; k < 3; ++k) {
			const size_t e = s.at + rng() % s.n;
			double v[2];
			for (int sign = 0; sign < 2; ++sign) {
				auto q = dp;
				q[e] += sign ? -1e-5 : 1e-5;
				v[sign] = 0;
				for (uint32_t i = 0; i < n; ++i) v[sign] += loss_row(q.data(), &xs[(size_t)i * in], i);
			}
			const double want = (v[0] - v[1]) / 2e-5;
			// both passes' roundings, about 6 L + 6 of 11 bits, in a sum whose terms are as large as the tensor's entries; ReLU: a few
			// of the n W units lie within a rounding of their corner
			EXPECT(std::fabs(__half2float(gp[e]) - want) <= (act == 1 ? 12 : 6) * 2 * steps * (rms + std::fabs(want)));
		}
	}
	double rms = 0;
	for (const T& v : dx) rms += std::pow((double)__half2float(v), 2);
	rms = std::sqrt(rms / dx.size());
	for (int k = 0; k < 6; ++k) {
		const size_t e = rng() % xs.size();
		const uint32_t i = (uint32_t)(e / in);
		auto row = std::vector<double>(&xs[(size_t)i * in], &xs[(size_t)i * in] + in);
		row[e % in] += 1e-5;
		const double hi = loss_row(dp.data(), row.data(), i);
		row[e % in] -= 2e-5;
		const double want = (hi - loss_row(dp.data(), row.data(), i)) / 2e-5;
		EXPECT(std::fabs(__half2float(dx[e]) - want) <= (act == 1 ? 12 : 6) * 2 * steps * (rms + std::fabs(want)));
	}
	{  // accumulation doubles the gradient, ignoring leaves it; strided and row-major operands give the same
		network->backward(stream, *ctx, X, Y, dY, nullptr, false, EGradientMode::Accumulate);
		auto twice = to_host(g.data(), 64);
		network->backward(stream, *ctx, X, Y, dY, &dX, false, EGradientMode::Ignore);
		auto still = to_host(g.data(), 64);
		for (int i = 0; i < 64; ++i) EXPECT(std::fabs(__half2float(twice[i]) - 2 * __half2float(gp[i])) <= 2e-3 * std::fabs(2 * __half2float(gp[i])) + 1e-6);
		EXPECT(!std::memcmp(twice.data(), still.data(), 64 * sizeof(T)));
		GPUMatrixDynamic<T> wide{in + 24, n, stream};
		GPUMatrixDynamic<T> slice = wide.slice_rows(8, in);
		CUDA_CHECK_THROW(cudaMemcpy2DAsync(slice.data(), (in + 24) * sizeof(T), x.data(), in * sizeof(T), in * sizeof(T), n, cudaMemcpyDeviceToDevice, stream));
		GPUMatrixDynamic<T> Y2{padded, n, stream};
		network->inference_mixed_precision(stream, slice, Y2, false);
		GPUMatrix<T, RM> rm{padded, n, stream};
		network->inference_mixed_precision(stream, X, rm, false);
		CUDA_CHECK_THROW(cudaStreamSynchronize(stream));
		auto a = to_host(Y2.data(), (size_t)n * padded), b = to_host(rm.data(), (size_t)n * padded);
		bool same = true;
		for (uint32_t i = 0; i < n; ++i)
			for (uint32_t c = 0; c < padded; ++c) same = same && __half2float(a[(size_t)i * padded + c]) == __half2float(y[(size_t)i * padded + c]) &&
			                                             __half2float(b[(size_t)c * n + i]) == __half2float(y[(size_t)i * padded + c]);
		EXPECT(same);
	}
}

int main(int argc, char** argv) {
	{
		std::unique_ptr<Network<T>> a{create_network<T>(net(48, 3, 256, 2, "SiLU"))};
		EXPECT(a->input_width() == 48 && a->output_width() == 3 && a->padded_output_width() == 16 && a->num_forward_activations() == 2 && a->width(0) == 256);
		EXPECT(a->layer_sizes().size() == 6 && a->layer_sizes()[5] == std::make_pair(16u, 256u) && a->required_input_alignment() == 16);
		EXPECT(a->n_params() == 256 * 48 + 4 * 256 * 256 + 16 * 256 + 256 + 2 * 4 * 256 + 2 * 256 + 16);
		EXPECT(a->hyperparams()["otype"] == "ResidualMLP" && a->hyperparams()["n_neurons"] == 256);
		EXPECT(minimum_alignment(net(48, 3, 256, 2, "SiLU")) == 16);
		EXPECT(throws([] { delete create_network<T>(net(40, 3, 256, 2, "SiLU")); }));
		EXPECT(throws([] { delete create_network<T>(net(48, 3, 100, 2, "SiLU")); }));
		EXPECT(throws([] { delete create_network<T>(net(48, 0, 256, 2, "SiLU")); }));
		EXPECT(throws([] { delete create_network<T>(net(48, 3, 256, 0, "SiLU")); }));
		EXPECT(throws([] { delete create_network<T>(net(48, 3, 256, 2, "Sine")); }));
		EXPECT(throws([] { json j = net(48, 3, 256, 2, "SiLU"); j["output_activation"] = "Sigmoid"; delete create_network<T>(j); }));
	}
	if (argc > 1 && std::strcmp(argv[1], "--check-only") == 0) {
		std::printf(g_failed ? "host checks FAILED\n" : "host checks ok\n");
		return g_failed ? 1 : 0;
	}
	cudaStream_t stream;
	CUDA_CHECK_THROW(cudaStreamCreate(&stream));
	{
		std::mt19937 rng(11);
		check_network(32, 16, 64, 1, "GELU", 2, 200, stream, rng);
		check_network(48, 3, 96, 2, "SiLU", 3, 37, stream, rng);
		check_network(16, 20, 32, 2, "ReLU", 1, 300, stream, rng);
		check_network(32, 5, 48, 1, "None", 0, 1, stream, rng);
		{  // behind the hash grid, with the optimizer, for a few steps: everything stays finite and every parameter group moves
			const json grid = {{"otype", "HashGrid"}, {"n_levels", 8}, {"n_features_per_level", 2}, {"log2_hashmap_size", 14}, {"base_resolution", 8}, {"per_level_scale", 1.5f}};
			json n = net(0, 4, 128, 2, "GELU");
			n.erase("n_input_dims");
			n.erase("n_output_dims");
			auto model = std::make_shared<NetworkWithInputEncoding<T>>(3, 4, grid, n);
			std::shared_ptr<Optimizer<T>> opt{create_optimizer<T>({{"otype", "Adam"}, {"learning_rate", 1e-3f}})};
			std::shared_ptr<Loss<T>> loss{create_loss<T>({{"otype", "L2"}})};
			auto trainer = std::make_shared<Trainer<float, T, T>>(model, opt, loss, 1337);
			const uint32_t batch = 1 << 12;
			std::uniform_real_distribution<float> u01(0.f, 1.f);
			std::vector<float> hx((size_t)batch * 3), ht((size_t)batch * 4);
			for (auto& v : hx) v = u01(rng);
			for (size_t i = 0; i < batch; ++i)
				for (int c = 0; c < 4; ++c) ht[i * 4 + c] = std::sin(6.f * hx[i * 3 + c % 3] + c);
			GPUMemory<float> x, t;
			x.resize_and_copy_from_host(hx);
			t.resize_and_copy_from_host(ht);
			auto before = to_host(trainer->params_full_precision(), trainer->n_params());
			for (int s = 0; s < 5; ++s) trainer->training_step(stream, GPUMatrix<float>(x.data(), 3, batch), GPUMatrix<float>(t.data(), 4, batch));
			CUDA_CHECK_THROW(cudaStreamSynchronize(stream));
			auto after = to_host(trainer->params_full_precision(), trainer->n_params());
			size_t moved = 0;
			bool finite = true;
			for (size_t i = 0; i < after.size(); ++i) finite = finite && std::isfinite(after[i]), moved += after[i] != before[i];
			EXPECT(finite && moved > after.size() / 8);
		}
	}
	uint32_t flags = 1;
	EXPECT(neus2b_device_error_flags(&flags) == 0 && flags == 0);
	CUDA_CHECK_THROW(cudaStreamDestroy(stream));
	std::printf(g_failed ? "residual network FAILED\n" : "residual network ok\n");
	return g_failed ? 1 : 0;
}
