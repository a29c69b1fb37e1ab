// Linear layers of any width: y = act(x W^T + b) + r, and the two products of the backward pass.
#include "linear.cuh"

namespace n2b {

// dz = dy * act'(z), eight columns a thread; rows of dz start on 16-byte boundaries and hold whole units of eight.  VEC: rows of z and dy start
// there, too.  Bound by memory: 8192 x 4096 fp16 in 35 us, 5.8 TB/s; entry by entry with a division each it took 100.
template <typename T, int ACT, bool VEC>
__global__ void __launch_bounds__(256) slope_kernel(uint32_t n, uint32_t width, const T* __restrict__ z, uint64_t z_ld, const T* __restrict__ dy, uint64_t dy_ld,
                                                     T* __restrict__ dz) {
	wait_for_previous();
	let_next_start();
	const uint32_t per = (width + 7) / 8;
	const uint64_t units = (uint64_t)n * per, step = gridDim.x * 256ull;
	const uint32_t step_row = (uint32_t)(step / per), step_col = (uint32_t)(step - (uint64_t)step_row * per);
	uint64_t u = blockIdx.x * 256ull + threadIdx.x;
	uint32_t row = (uint32_t)(u / per), col = (uint32_t)(u - (uint64_t)row * per);
	for (; u < units; u += step) {
		const T *zp = z + row * z_ld + col * 8u, *dp = dy + row * dy_ld + col * 8u;
		const uint32_t count = width - col * 8u;  // 8 at least, but for the last ones of a row
		union Eight {
			uint4 q;
			T v[8];
		} a{}, b{};
		if (VEC && count >= 8) {
			a.q = *reinterpret_cast<const uint4*>(zp);
			b.q = *reinterpret_cast<const uint4*>(dp);
		} else {
#pragma unroll
			for (uint32_t k = 0; k < 8; ++k)
				if (k < count) a.v[k] = zp[k], b.v[k] = dp[k];
		}
#pragma unroll
		for (int k = 0; k < 8; ++k) b.v[k] = from_f<T>(to_f(b.v[k]) * act_slope(ACT, to_f(a.v[k])));
		reinterpret_cast<uint4*>(dz)[u] = b.q;
		row += step_row, col += step_col;
		if (col >= per) col -= per, ++row;
	}
}
template <typename T>
static int run_slope(uint32_t n, uint32_t width, int act, const void* z, uint64_t z_ld, const void* dy, uint64_t dy_ld, void* dz, cudaStream_t stream) {
	const bool vec = operand_aligned(z, z_ld) && operand_aligned(dy, dy_ld);
	const uint64_t blocks = ((uint64_t)n * ((width + 7) / 8) + 255) / 256;
	auto go = [&](auto kernel) {
		return launch_behind(kernel, (uint32_t)(blocks < 8ull * kSMs ? blocks : 8 * kSMs), 256, 0, stream, n, width, (const T*)z, z_ld, (const T*)dy, dy_ld, (T*)dz);
	};
	if (act == NEUS2B_ACT_RELU) return vec ? go(slope_kernel<T, NEUS2B_ACT_RELU, true>) : go(slope_kernel<T, NEUS2B_ACT_RELU, false>);
	if (act == NEUS2B_ACT_GELU) return vec ? go(slope_kernel<T, NEUS2B_ACT_GELU, true>) : go(slope_kernel<T, NEUS2B_ACT_GELU, false>);
	return vec ? go(slope_kernel<T, NEUS2B_ACT_SILU, true>) : go(slope_kernel<T, NEUS2B_ACT_SILU, false>);
}

static bool bad_desc(const neus2b_linear_desc* d) {
	return !d || d->in_width == 0 || d->out_width == 0 || d->activation > NEUS2B_ACT_SILU;
}
constexpr uint32_t kMost = 1u << 30;  // samples and widths: tile coordinates are signed 32-bit numbers
static bool too_large(const neus2b_linear_desc* d) { return d->n > kMost || d->in_width > kMost || d->out_width > kMost; }
// An output that is an input, other than as the interface allows it: the same rows, read by the thread that writes them.
static bool clash(const void* out, const void* in) { return out && out == in; }
static bool clash(const void* out, uint64_t out_stride, const void* in, uint64_t in_stride, uint32_t n) { return out && out == in && n > 1 && out_stride != in_stride; }
static bool bad_matrix(const void* p, uint64_t stride, uint32_t width, size_t align) { return !p || stride < width || ((uintptr_t)p & (align - 1)); }
static bool bad_optional(const void* p, uint64_t stride, uint32_t width, size_t align) { return p && bad_matrix(p, stride, width, align); }

static bool starts_on(uint32_t at, const void* p, uint64_t ld, size_t bytes) { return !p || (((uintptr_t)p | (ld * bytes)) & (at - 1)) == 0; }
// Bytes that the epilogue may move at a time: every row that it touches starts on such a boundary, and rows of 16-bit values are whole numbers
// of accesses (an fp32 row's end is handled apart).
static int widest_access(const Epilogue& e, uint32_t width) {
	auto fits = [&](uint32_t at) {
		return (e.out_f32 || width % (at / 2) == 0) && starts_on(at, e.out, e.out_ld, e.out_f32 ? 4 : 2) && starts_on(at, e.bias, 0, 2) &&
		       starts_on(at, e.add, e.add_ld, 2) && starts_on(at, e.slope_z, e.slope_ld, 2) && starts_on(at, e.preact, e.preact_ld, 2);
	};
	return fits(16) ? 16 : fits(4) ? 4 : 2;
}

}  // namespace n2b

using namespace n2b;

// A copy of a matrix with rows on 16-byte boundaries
static uint64_t copy_bytes(uint64_t rows, uint32_t cols) { return (rows * ((cols + 7) / 8) * 16 + 255) / 256 * 256; }
// Takes the place of a product's operand by its copy, where it needs one; `at` moves on behind it.
static void realigned(const void*& p, uint64_t& ld, uint32_t rows, uint32_t cols, char*& at, Operand* ops, int& count) {
	if (operand_aligned(p, ld)) return;
	ops[count++] = Operand{p, ld, rows, cols, at};
	p = at, ld = (cols + 7) / 8 * 8;
	at += copy_bytes(rows, cols);
}

extern "C" int neus2b_linear_forward_workspace(const neus2b_linear_desc* desc, int unaligned, uint64_t* bytes) {
	if (bad_desc(desc) || !bytes) return NEUS2B_E_INVALID;
	if (!is_half_type(desc->dtype)) return NEUS2B_E_UNSUPPORTED;
	if (too_large(desc)) return NEUS2B_E_TOO_LARGE;
	*bytes = unaligned ? copy_bytes(desc->n, desc->in_width) + copy_bytes(desc->out_width, desc->in_width) : 0;
	return NEUS2B_OK;
}

extern "C" int neus2b_linear_forward(const neus2b_linear_desc* desc, const void* d_x, uint64_t x_stride, const void* d_w, const void* d_bias,
                                     const void* d_residual, uint64_t residual_stride, void* d_y, uint64_t y_stride, void* d_preact,
                                     uint64_t preact_stride, void* d_workspace, uint64_t workspace_bytes, neus2b_stream_t stream) {
	uint64_t need = 0;
	if (int rc = neus2b_linear_forward_workspace(desc, 1, &need)) return rc;
	const uint32_t in = desc->in_width, out = desc->out_width;
	if (bad_matrix(d_w, in, in, 2) || ((uintptr_t)d_bias & 1)) return NEUS2B_E_INVALID;
	if (desc->n == 0) return NEUS2B_OK;
	if (bad_matrix(d_x, x_stride, in, 2) || bad_matrix(d_y, y_stride, out, 2) || bad_optional(d_residual, residual_stride, out, 2) ||
	    bad_optional(d_preact, preact_stride, out, 2))
		return NEUS2B_E_INVALID;
	if (clash(d_y, d_x) || clash(d_y, d_w) || clash(d_y, d_preact) || clash(d_preact, d_x) || clash(d_preact, d_w) || clash(d_preact, d_residual) ||
	    clash(d_y, y_stride, d_residual, residual_stride, desc->n))
		return NEUS2B_E_INVALID;
	Product p{};
	p.a = d_x, p.a_ld = x_stride, p.b = d_w, p.b_ld = in;
	p.M = desc->n, p.N = out, p.K = in, p.bf16 = desc->dtype == NEUS2B_BF16;
	if (!(operand_aligned(p.a, p.a_ld) && operand_aligned(p.b, p.b_ld))) {
		if (!d_workspace || ((uintptr_t)d_workspace & 15) || workspace_bytes < need) return NEUS2B_E_INVALID;
		Operand ops[2];
		int count = 0;
		char* at = (char*)d_workspace;
		realigned(p.a, p.a_ld, desc->n, in, at, ops, count);
		realigned(p.b, p.b_ld, out, in, at, ops, count);
		if (int rc = run_realign(ops, count, stream)) return rc;
	}
	Epilogue& e = p.e;
	e.out = d_y, e.out_ld = y_stride, e.bias = d_bias, e.add = d_residual, e.add_ld = residual_stride;
	e.preact = d_preact, e.preact_ld = preact_stride, e.act = (int)desc->activation;
	e.vec = widest_access(e, out);
	if (narrow_fits(p, false, nullptr)) return run_narrow(p, false, nullptr, stream);
	return run_product(p, stream);
}

// Workspace of the backward pass: dz where the layer has an activation, copies of unaligned operands, what the weight gradient needs.
static uint64_t dz_bytes(const neus2b_linear_desc* d) { return d->activation == NEUS2B_ACT_NONE ? 0 : copy_bytes(d->n, d->out_width); }
static uint64_t copies_bytes(const neus2b_linear_desc* d) {
	return copy_bytes(d->n, d->out_width) + copy_bytes(d->n, d->in_width) + copy_bytes(d->out_width, d->in_width);
}

extern "C" int neus2b_linear_backward_workspace(const neus2b_linear_desc* desc, int unaligned, uint64_t* bytes) {
	if (bad_desc(desc) || !bytes) return NEUS2B_E_INVALID;
	if (!is_half_type(desc->dtype)) return NEUS2B_E_UNSUPPORTED;
	if (too_large(desc)) return NEUS2B_E_TOO_LARGE;
	uint64_t parts = 0;
	if (desc->n) {
		const uint64_t narrow = narrow_workspace(desc->out_width, desc->in_width, desc->n);
		parts = wgrad_workspace(desc->out_width, desc->in_width, desc->n);
		if (narrow > parts) parts = narrow;
	}
	*bytes = dz_bytes(desc) + (unaligned ? copies_bytes(desc) : 0) + parts;
	return NEUS2B_OK;
}

extern "C" int neus2b_linear_backward(const neus2b_linear_desc* desc, const void* d_x, uint64_t x_stride, const void* d_w, const void* d_preact,
                                      uint64_t preact_stride, const void* d_dL_dy, uint64_t dy_stride, uint32_t below_activation,
                                      const void* d_below_preact, uint64_t below_stride, const void* d_skip, uint64_t skip_stride, void* d_dL_dx,
                                      uint64_t dx_stride, float* d_wgrad, float* d_bgrad, int grad_mode, void* d_workspace,
                                      uint64_t workspace_bytes, neus2b_stream_t stream) {
	uint64_t need = 0;
	if (int rc = neus2b_linear_backward_workspace(desc, 0, &need)) return rc;
	if (below_activation > NEUS2B_ACT_SILU || grad_mode < NEUS2B_GRAD_IGNORE || grad_mode > NEUS2B_GRAD_ACCUMULATE) return NEUS2B_E_INVALID;
	const uint32_t n = desc->n, in = desc->in_width, out = desc->out_width;
	if (grad_mode == NEUS2B_GRAD_IGNORE) d_wgrad = d_bgrad = nullptr;
	if (!d_wgrad && !d_bgrad) need = dz_bytes(desc);
	if (((uintptr_t)d_wgrad | (uintptr_t)d_bgrad) & 3) return NEUS2B_E_INVALID;
	if (n == 0) {
		if (grad_mode == NEUS2B_GRAD_OVERWRITE) {
			if (d_wgrad) N2B_CHECK_CUDA(cudaMemsetAsync(d_wgrad, 0, (size_t)in * out * 4, stream));
			if (d_bgrad) N2B_CHECK_CUDA(cudaMemsetAsync(d_bgrad, 0, (size_t)out * 4, stream));
		}
		return NEUS2B_OK;
	}
	if (bad_matrix(d_dL_dy, dy_stride, out, 2) || (d_wgrad && bad_matrix(d_x, x_stride, in, 2)) || (d_dL_dx && bad_matrix(d_w, in, in, 2)) ||
	    bad_optional(d_dL_dx, dx_stride, in, 2) || bad_optional(d_skip, skip_stride, in, 2))
		return NEUS2B_E_INVALID;
	if (desc->activation != NEUS2B_ACT_NONE && bad_matrix(d_preact, preact_stride, out, 2)) return NEUS2B_E_INVALID;
	if (d_dL_dx && below_activation != NEUS2B_ACT_NONE && bad_matrix(d_below_preact, below_stride, in, 2)) return NEUS2B_E_INVALID;
	if (need && (!d_workspace || ((uintptr_t)d_workspace & 15) || workspace_bytes < need)) return NEUS2B_E_INVALID;
	if (clash(d_dL_dx, d_x) || clash(d_dL_dx, d_w) || clash(d_dL_dx, d_dL_dy) || clash(d_dL_dx, d_preact) || clash(d_dL_dx, d_below_preact) ||
	    clash(d_dL_dx, dx_stride, d_skip, skip_stride, n))
		return NEUS2B_E_INVALID;
	const void *dz = d_dL_dy, *xs = d_x, *ws = d_w;
	uint64_t dz_ld = dy_stride, xs_ld = x_stride, ws_ld = in;
	char* at = (char*)d_workspace;
	if (desc->activation != NEUS2B_ACT_NONE) {
		const uint64_t ld = (out + 7) / 8 * 8;
		const int rc = with_half_type(desc->dtype, [&](auto t) {
			using T = decltype(t);
			return run_slope<T>(n, out, (int)desc->activation, d_preact, preact_stride, d_dL_dy, dy_stride, d_workspace, stream);
		});
		if (rc) return rc;
		dz = d_workspace, dz_ld = ld;
		at += dz_bytes(desc);
	}
	const bool params = d_wgrad || d_bgrad;
	const bool copy_dz = !operand_aligned(dz, dz_ld) && (params || d_dL_dx), copy_x = d_wgrad && !operand_aligned(xs, xs_ld),
	           copy_w = d_dL_dx && !operand_aligned(ws, ws_ld);
	if (copy_dz || copy_x || copy_w) {
		if (!d_workspace || ((uintptr_t)d_workspace & 15) || workspace_bytes < need + copies_bytes(desc)) return NEUS2B_E_INVALID;
		Operand ops[3];
		int count = 0;
		if (copy_dz) realigned(dz, dz_ld, n, out, at, ops, count);
		if (copy_x) realigned(xs, xs_ld, n, in, at, ops, count);
		if (copy_w) realigned(ws, ws_ld, out, in, at, ops, count);
		if (int rc = run_realign(ops, count, stream)) return rc;
	}
	Product w{}, x{};  // the weight gradient, the input gradient
	w.bf16 = x.bf16 = desc->dtype == NEUS2B_BF16;
	w.a = x.a = dz, w.a_ld = x.a_ld = dz_ld;
	if (d_wgrad) {
		w.b = xs, w.b_ld = xs_ld;
		w.M = out, w.N = in, w.K = n;
		w.e.out = d_wgrad, w.e.out_ld = in, w.e.out_f32 = 1, w.e.accumulate = grad_mode == NEUS2B_GRAD_ACCUMULATE;
		w.e.vec = widest_access(w.e, in);
		w.column_sums = d_bgrad;
		w.workspace = at, w.workspace_bytes = workspace_bytes - (uint64_t)(at - (char*)d_workspace);
	}
	x.b = ws, x.b_ld = ws_ld;
	x.M = n, x.N = in, x.K = out;
	x.b_mn = true;
	x.e.out = d_dL_dx, x.e.out_ld = dx_stride, x.e.add = d_skip, x.e.add_ld = skip_stride;
	if (d_dL_dx && below_activation != NEUS2B_ACT_NONE) x.e.slope_z = d_below_preact, x.e.slope_ld = below_stride, x.e.act = (int)below_activation;
	x.e.vec = widest_access(x.e, in);
	if (d_bgrad && !d_wgrad)
		if (int rc = run_column_sums(dz, dz_ld, n, out, w.bf16, d_bgrad, grad_mode == NEUS2B_GRAD_ACCUMULATE, stream)) return rc;
	if ((d_wgrad || d_dL_dx) && narrow_fits(x, true, d_wgrad ? &w : nullptr)) return run_narrow(x, true, d_wgrad ? &w : nullptr, stream);
	if (d_wgrad)
		if (int rc = run_weight_gradient(w, stream)) return rc;
	if (d_dL_dx)
		if (int rc = run_product(x, stream)) return rc;
	return NEUS2B_OK;
}
