/* tiny-cuda-nn/networks/residual_mlp.h of the B200-native stand-in: "ResidualMLP", a network of any width beside the fused 64-neuron
 * one.  No counterpart in the reference, whose networks are all 64 neurons wide.
 *
 *   h_0 = W_in x + b_in,   h_(l+1) = h_l + W2_l act(W1_l LN_l(h_l) + b1_l) + b2_l,   y = W_out LN(h_L) + b_out
 *
 * over the C interface's linear layers and layer norms: bias, activation and the skip connection are part of the products, the
 * backward pass of a product carries the activation's slope, that of a norm the skip connection's gradient.
 * Keys: "n_neurons" (a multiple of 16), "n_hidden_layers" (blocks), "activation" ("ReLU", "GELU", "SiLU" or "None"), no output activation.
 * Included by network.h. */
#pragma once

TCNN_NAMESPACE_BEGIN

#if defined(__CUDACC__)
template <typename T>
__global__ void fill_parameter_kernel(const uint32_t n, float* __restrict__ out, const float value) {
	const uint32_t i = threadIdx.x + blockIdx.x * blockDim.x;
	if (i < n) out[i] = value;
}
#endif

template <typename T>
class ResidualMLP : public Network<T> {
	static_assert(std::is_same<T, __half>::value, "parameters and activations of this library's networks are fp16");

public:
	struct ForwardContext : public Context {
		GPUMemoryArena::Allocation saved;
		T *h = nullptr, *a = nullptr, *z = nullptr, *u = nullptr; /* [blocks + 1], [blocks + 1], [blocks], [blocks] times [n][width] */
		float *mean = nullptr, *rstd = nullptr;                   /* [blocks + 1][n] */
	};

	ResidualMLP(uint32_t input_width, uint32_t output_width, uint32_t n_neurons, uint32_t n_blocks, const std::string& activation, Activation output_activation)
	    : m_input_width{input_width}, m_output_width{output_width}, m_padded_output{next_multiple(output_width, 16u)}, m_width{n_neurons}, m_blocks{n_blocks} {
		if (input_width == 0 || input_width % 16) throw std::runtime_error("ResidualMLP: input widths are multiples of 16, got " + std::to_string(input_width));
		if (n_neurons == 0 || n_neurons % 16) throw std::runtime_error("ResidualMLP: n_neurons is a multiple of 16, got " + std::to_string(n_neurons));
		if (output_width == 0) throw std::runtime_error("ResidualMLP: at least one output");
		if (n_blocks == 0) throw std::runtime_error("ResidualMLP: at least one hidden layer (residual block)");
		if (output_activation != Activation::None) throw std::runtime_error("ResidualMLP: no output activation");
		const std::string act = to_lower(activation);
		if (act == "relu") m_act = NEUS2B_ACT_RELU;
		else if (act == "gelu") m_act = NEUS2B_ACT_GELU;
		else if (act == "silu") m_act = NEUS2B_ACT_SILU;
		else if (act == "none") m_act = NEUS2B_ACT_NONE;
		else throw std::runtime_error("ResidualMLP: activation \"" + activation + "\" is not ReLU, GELU, SiLU or None");
		m_activation = activation;
	}

	void inference_mixed_precision_impl(cudaStream_t stream, const GPUMatrixDynamic<T>& input, GPUMatrixDynamic<T>& output, bool use_inference_params = true) override {
		forward_impl(stream, input, &output, use_inference_params, false);
	}

	std::unique_ptr<Context> forward_impl(cudaStream_t stream, const GPUMatrixDynamic<T>& input, GPUMatrixDynamic<T>* output = nullptr, bool use_inference_params = false,
	                                      bool prepare_input_gradients = false) override {
		(void)prepare_input_gradients;
		auto ctx = std::make_unique<ForwardContext>();
		const uint32_t n = input.n();
		if (!n) return ctx;
#if defined(__CUDACC__)
		const T* p = use_inference_params ? m_inference_params : m_params;
		const size_t each = (size_t)n * m_width, values = each * (4 * (size_t)m_blocks + 2), stats = (size_t)n * (m_blocks + 1);
		ctx->saved = allocate_workspace(stream, values * sizeof(T) + 2 * stats * sizeof(float));
		ctx->h = (T*)ctx->saved.data();
		ctx->a = ctx->h + each * (m_blocks + 1);
		ctx->z = ctx->a + each * (m_blocks + 1);
		ctx->u = ctx->z + each * m_blocks;
		ctx->mean = (float*)(ctx->u + each * m_blocks);
		ctx->rstd = ctx->mean + stats;
		DenseColumns<T> x{stream, input, true, true};
		linear(stream, n, m_input_width, m_width, NEUS2B_ACT_NONE, x.data(), x.copied() ? m_input_width : input.stride(), p + w_in(), p + b_in(), nullptr, ctx->h, m_width, nullptr);
		for (uint32_t l = 0; l <= m_blocks; ++l) {
			T *h = ctx->h + l * each, *a = ctx->a + l * each;
			const neus2b_layer_norm_desc d{n, m_width, NEUS2B_F16, NEUS2B_F16, 1e-5f};
			check(neus2b_layer_norm_forward(&d, h, m_width, p + gamma(l), p + beta(l), a, m_width, ctx->mean + (size_t)l * n, ctx->rstd + (size_t)l * n, stream), "layer norm");
			if (l == m_blocks) break;
			T *z = ctx->z + l * each, *u = ctx->u + l * each;
			linear(stream, n, m_width, m_width, m_act, a, m_width, p + w1(l), p + b1(l), nullptr, u, m_width, m_act == NEUS2B_ACT_NONE ? nullptr : z);
			linear(stream, n, m_width, m_width, NEUS2B_ACT_NONE, u, m_width, p + w2(l), p + b2(l), h, h + each, m_width, nullptr);
		}
		if (output) {
			DenseColumns<T> y{stream, *output, false, true};
			linear(stream, n, m_width, m_padded_output, NEUS2B_ACT_NONE, ctx->a + m_blocks * each, m_width, p + w_out(), p + b_out(), nullptr, y.data(),
			       y.copied() ? m_padded_output : output->stride(), nullptr);
			y.scatter();
		}
#else
		throw std::runtime_error("ResidualMLP: needs a CUDA translation unit");
#endif
		return ctx;
	}

	void backward_impl(cudaStream_t stream, const Context& ctx, const GPUMatrixDynamic<T>& input, const GPUMatrixDynamic<T>& output, const GPUMatrixDynamic<T>& dL_doutput,
	                   GPUMatrixDynamic<T>* dL_dinput = nullptr, bool use_inference_params = false, EGradientMode param_gradients_mode = EGradientMode::Overwrite) override {
		(void)output;
		const uint32_t n = input.n();
		if (!n) { /* the gradient of nothing is 0 */
			if (param_gradients_mode == EGradientMode::Overwrite) CUDA_CHECK_THROW(cudaMemsetAsync(m_gradients, 0, n_params() * sizeof(T), stream));
			return;
		}
#if defined(__CUDACC__)
		const auto& f = dynamic_cast<const ForwardContext&>(ctx);
		const T* p = use_inference_params ? m_inference_params : m_params;
		const bool params = param_gradients_mode != EGradientMode::Ignore;
		if (params) m_grad_scratch.enlarge(n_params());
		float* g = params ? m_grad_scratch.data() : nullptr;
		const int mode = params ? NEUS2B_GRAD_OVERWRITE : NEUS2B_GRAD_IGNORE;
		const size_t each = (size_t)n * m_width;
		auto scratch = allocate_workspace(stream, 3 * each * sizeof(T));
		T *dh = (T*)scratch.data(), *da = dh + each, *dz = da + each;
		DenseColumns<T> x{stream, input, true, true}, dy{stream, dL_doutput, true, true};
		auto norm_back = [&](uint32_t l, const T* skip) {
			const neus2b_layer_norm_desc d{n, m_width, NEUS2B_F16, NEUS2B_F16, 1e-5f};
			uint64_t bytes = 0;
			check(neus2b_layer_norm_backward_workspace(&d, &bytes), "layer norm");
			auto ws = allocate_workspace(stream, (size_t)bytes + 16);
			check(neus2b_layer_norm_backward(&d, f.h + l * each, m_width, p + gamma(l), f.mean + (size_t)l * n, f.rstd + (size_t)l * n, da, m_width, skip, m_width, dh, m_width,
			                                 g ? g + gamma(l) : nullptr, g ? g + beta(l) : nullptr, mode, ws.data(), bytes, stream),
			      "layer norm backward");
		};
		back(stream, n, m_width, m_padded_output, f.a + m_blocks * each, m_width, p + w_out(), dy.data(), dy.copied() ? m_padded_output : dL_doutput.stride(), NEUS2B_ACT_NONE, nullptr,
		     da, m_width, g ? g + w_out() : nullptr, g ? g + b_out() : nullptr, mode);
		norm_back(m_blocks, nullptr);
		for (uint32_t l = m_blocks; l-- > 0;) {
			back(stream, n, m_width, m_width, f.u + l * each, m_width, p + w2(l), dh, m_width, m_act, m_act == NEUS2B_ACT_NONE ? nullptr : f.z + l * each, dz, m_width,
			     g ? g + w2(l) : nullptr, g ? g + b2(l) : nullptr, mode);
			back(stream, n, m_width, m_width, f.a + l * each, m_width, p + w1(l), dz, m_width, NEUS2B_ACT_NONE, nullptr, da, m_width, g ? g + w1(l) : nullptr, g ? g + b1(l) : nullptr, mode);
			norm_back(l, dh);
		}
		std::unique_ptr<DenseColumns<T>> dx;
		if (dL_dinput) dx = std::make_unique<DenseColumns<T>>(stream, *dL_dinput, false, true);
		if (dx || g)
			back(stream, n, m_input_width, m_width, x.data(), x.copied() ? m_input_width : input.stride(), p + w_in(), dh, m_width, NEUS2B_ACT_NONE, nullptr, dx ? dx->data() : nullptr,
			     dx ? (dx->copied() ? m_input_width : dL_dinput->stride()) : 0u, g ? g + w_in() : nullptr, g ? g + b_in() : nullptr, mode);
		if (dx) dx->scatter();
		if (params) {
			const uint32_t count = (uint32_t)n_params();
			gradient_from_float_kernel<T>
			    <<<n_blocks_linear(count), n_threads_linear, 0, stream>>>(count, m_grad_scratch.data(), m_gradients, param_gradients_mode == EGradientMode::Accumulate);
		}
#else
		throw std::runtime_error("ResidualMLP: needs a CUDA translation unit");
#endif
	}

	void backward_backward_input_impl(cudaStream_t, const Context&, const GPUMatrixDynamic<T>&, const GPUMatrixDynamic<T>&, const GPUMatrixDynamic<T>&, GPUMatrixDynamic<T>* = nullptr,
	                                  GPUMatrixDynamic<T>* = nullptr, bool = false, EGradientMode = EGradientMode::Overwrite) override {
		throw std::runtime_error("ResidualMLP: second-order gradients are not part of this network");
	}

	void set_params(T* params, T* inference_params, T* backward_params, T* gradients) override {
		(void)backward_params;
		m_params = params;
		m_inference_params = inference_params;
		m_gradients = gradients;
	}
	/* matrices uniform in +-sqrt(6 / (fan_in + fan_out)) * scale, norms 1 and 0, biases 0 */
	void initialize_params(pcg32& rnd, float* params_full_precision, T* params, T* inference_params, T* backward_params, T* gradients, float scale = 1) override {
		set_params(params, inference_params, backward_params, gradients);
#if defined(__CUDACC__)
		size_t offset = 0;
		for (const auto& layer : layer_sizes()) {
			const float bound = std::sqrt(6.0f / (float)(layer.first + layer.second)) * scale;
			generate_random_uniform<float>(rnd, (size_t)layer.first * layer.second, params_full_precision + offset, -bound, bound);
			offset += (size_t)layer.first * layer.second;
		}
		CUDA_CHECK_THROW(cudaMemset(params_full_precision + offset, 0, (n_params() - offset) * sizeof(float)));
		for (uint32_t l = 0; l <= m_blocks; ++l)
			fill_parameter_kernel<T><<<n_blocks_linear(m_width), n_threads_linear>>>(m_width, params_full_precision + gamma(l), 1.0f);
#else
		throw std::runtime_error("ResidualMLP: needs a CUDA translation unit");
#endif
	}
	/* matrices first (what the optimizer's weight decay covers), then biases and norms */
	size_t n_params() const override { return b_out() + m_padded_output; }
	std::vector<std::pair<uint32_t, uint32_t>> layer_sizes() const override {
		std::vector<std::pair<uint32_t, uint32_t>> r{{m_width, m_input_width}};
		for (uint32_t l = 0; l < 2 * m_blocks; ++l) r.push_back({m_width, m_width});
		r.push_back({m_padded_output, m_width});
		return r;
	}
	uint32_t input_width() const override { return m_input_width; }
	uint32_t padded_output_width() const override { return m_padded_output; }
	uint32_t output_width() const override { return m_output_width; }
	uint32_t required_input_alignment() const override { return 16; }
	uint32_t width(uint32_t layer) const override {
		(void)layer;
		return m_width;
	}
	uint32_t num_forward_activations() const override { return m_blocks; }
	/* the state behind block `layer` */
	std::pair<const T*, MatrixLayout> forward_activations(const Context& ctx, uint32_t layer) const override {
		const auto& f = dynamic_cast<const ForwardContext&>(ctx);
		const size_t n = f.mean ? (size_t)(f.rstd - f.mean) / (m_blocks + 1) : 0;
		return {f.h + (size_t)(layer + 1) * n * m_width, CM};
	}
	T* params() const { return m_params; }
	T* inference_params() const { return m_inference_params; }
	T* gradients() const { return m_gradients; }
	json hyperparams() const override {
		return {{"otype", "ResidualMLP"}, {"activation", m_activation}, {"output_activation", "None"}, {"n_neurons", m_width}, {"n_hidden_layers", m_blocks}};
	}

private:
	static void check(int rc, const char* what) {
		if (rc) throw std::runtime_error(std::string("ResidualMLP: ") + what + ": " + neus2b_error_string(rc));
	}
	/* offsets into the parameter block */
	size_t square() const { return (size_t)m_width * m_width; }
	size_t w_in() const { return 0; }
	size_t w1(uint32_t l) const { return (size_t)m_width * m_input_width + 2 * l * square(); }
	size_t w2(uint32_t l) const { return w1(l) + square(); }
	size_t w_out() const { return w1(m_blocks); }
	size_t b_in() const { return w_out() + (size_t)m_padded_output * m_width; }
	size_t gamma(uint32_t l) const { return b_in() + m_width + (size_t)4 * l * m_width; } /* of a block: gamma, beta, b1, b2 */
	size_t beta(uint32_t l) const { return gamma(l) + m_width; }
	size_t b1(uint32_t l) const { return gamma(l) + 2 * (size_t)m_width; }
	size_t b2(uint32_t l) const { return gamma(l) + 3 * (size_t)m_width; }
	size_t b_out() const { return gamma(m_blocks) + 2 * (size_t)m_width; }

#if defined(__CUDACC__)
	static int off16(const void* p, uint64_t stride) { return ((size_t)p | (stride * sizeof(T))) & 15 ? 1 : 0; }
	static void linear(cudaStream_t stream, uint32_t n, uint32_t in, uint32_t out, uint32_t act, const T* x, uint64_t x_stride, const T* w, const T* bias, const T* residual, T* y,
	                   uint64_t y_stride, T* z) {
		const neus2b_linear_desc d{n, in, out, NEUS2B_F16, act};
		uint64_t bytes = 0;
		check(neus2b_linear_forward_workspace(&d, off16(x, x_stride) | off16(w, in), &bytes), "linear");
		GPUMemoryArena::Allocation ws;
		if (bytes) ws = allocate_workspace(stream, (size_t)bytes);
		check(neus2b_linear_forward(&d, x, x_stride, w, bias, residual, out, y, y_stride, z, out, bytes ? ws.data() : nullptr, bytes, stream), "linear");
	}
	/* dy is the gradient of the product itself; below_z: the activation that made x */
	static void back(cudaStream_t stream, uint32_t n, uint32_t in, uint32_t out, const T* x, uint64_t x_stride, const T* w, const T* dy, uint64_t dy_stride, uint32_t below,
	                 const T* below_z, T* dx, uint64_t dx_stride, float* wgrad, float* bgrad, int mode) {
		const neus2b_linear_desc d{n, in, out, NEUS2B_F16, NEUS2B_ACT_NONE};
		uint64_t bytes = 0;
		check(neus2b_linear_backward_workspace(&d, off16(x, x_stride) | off16(w, in) | off16(dy, dy_stride), &bytes), "linear backward");
		GPUMemoryArena::Allocation ws;
		if (bytes) ws = allocate_workspace(stream, (size_t)bytes);
		check(neus2b_linear_backward(&d, x, x_stride, w, nullptr, 0, dy, dy_stride, below, below_z, in, nullptr, 0, dx, dx_stride, wgrad, bgrad, mode, bytes ? ws.data() : nullptr, bytes,
		                             stream),
		      "linear backward");
	}
#endif

	uint32_t m_input_width, m_output_width, m_padded_output, m_width, m_blocks, m_act = NEUS2B_ACT_NONE;
	std::string m_activation;
	T *m_params = nullptr, *m_inference_params = nullptr, *m_gradients = nullptr;
	GPUMemory<float> m_grad_scratch;
};

TCNN_NAMESPACE_END
