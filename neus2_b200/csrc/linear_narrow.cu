// Linear layers with results of at most 64 columns from at most 128: the widths of the framework's own networks.  These products are
// bound by the samples' way through memory, so that every operand of a tile of 128 samples travels by TMA, ahead of its turn, and
// nothing is read twice.
//
// A persistent CTA keeps the weights in shared memory.  forward: y = act(x W^T + b) + r for a tile.  backward: dL/dx and the weight
// gradient in one pass over dz and x: the tile of dz is the K-major operand of dL/dx = dz W and, the same bytes, the MN-major operand of
// dz^T x.  The weight gradient's sums stay in tensor memory for four tiles (512 samples), then in registers, and leave the CTA
// once; the bias gradient is the product of dz^T with a tile of ones.
//
// 262144 samples, fp16: 48 -> 64 with ReLU 13.2 us (4.5 TB/s over what has to move), backward of 64 <- 64 with slopes, skip connection
// and bias 36 us with its join (4.6 TB/s).  A tile's operands are 16 KB each, so that two to eight stages fit; one CTA on an SM.
#include "linear_tc.cuh"

namespace n2b {
namespace lin {

static __device__ uint32_t g_narrow_error;  // bit 0: a bounded wait ran out

constexpr int kTile = 128 * 128;  // bytes of 128 rows of 64 values
constexpr int kRound = 4;         // tiles whose weight gradient is summed in tensor memory

struct alignas(64) NarrowArgs {
	CUtensorMap ta, tx, tw, tslope, tadd, tout, tpre;
	uint32_t n, N, K, bf16;
	const uint16_t* bias;
	int act;
	uint32_t slope, add, pre, out, params;  // what there is
	uint32_t stages, stage_bytes;
	float* partial;  // [gridDim.x][K][N], then [gridDim.x][K]
};

template <bool BACKWARD>
struct Narrow {
	static constexpr int kGroups = BACKWARD ? 2 : 4;  // groups of four epilogue warps take tiles in turn
	static constexpr int kEpiWarps = 4 * kGroups, kDrain = kEpiWarps, kMma = kEpiWarps + (BACKWARD ? 4 : 0), kLoad = kMma + 1;
	static constexpr int kThreads = (kLoad + 1) * 32;
	static constexpr int kBufs = 4, kTmem = BACKWARD ? 512 : 256;
};

__device__ __forceinline__ void tma_store(const CUtensorMap* map, uint32_t src, int x, int y) {
	asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(src) : "memory");
}
__device__ __forceinline__ uint64_t desc_mn_slabs(uint32_t addr, uint32_t slab_bytes) {
	return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(slab_bytes >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// 16-byte unit u of row r of a 128-byte-swizzled tile
__device__ __forceinline__ uint32_t unit128(int r, int u) { return (uint32_t)(r * 128 + ((u ^ (r & 7)) << 4)); }
__device__ __forceinline__ void tile_units(uint32_t (&w)[16], const unsigned char* tile, int r, int u0) {
#pragma unroll
	for (int u = 0; u < 4; ++u) {
		const uint4 v = *reinterpret_cast<const uint4*>(tile + unit128(r, u0 + u));
		w[4 * u] = v.x, w[4 * u + 1] = v.y, w[4 * u + 2] = v.z, w[4 * u + 3] = v.w;
	}
}
__device__ __forceinline__ void put_units(const uint32_t (&w)[16], unsigned char* tile, int r, int u0) {
#pragma unroll
	for (int u = 0; u < 4; ++u) *reinterpret_cast<uint4*>(tile + unit128(r, u0 + u)) = make_uint4(w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
}

template <bool BACKWARD>
__global__ void __launch_bounds__(Narrow<BACKWARD>::kThreads, 1) narrow_kernel(const __grid_constant__ NarrowArgs p) {
	using S = Narrow<BACKWARD>;
	extern __shared__ unsigned char smem_raw[];
	unsigned char* smem = smem_raw + ((1024u - (sptr(smem_raw) & 1023u)) & 1023u);
	const uint32_t slabs = p.K > 64 ? 2u : 1u;
	unsigned char* const weights = smem;                                   // forward: [slab][64 rows][64 k]; backward: [slab of 64 k][64 n]
	unsigned char* const misc = smem + slabs * 8192;                       // 512 bytes of ones, bias, barriers
	float* const bias = reinterpret_cast<float*>(misc + 512);              // [64]
	uint64_t* const bars = reinterpret_cast<uint64_t*>(misc + 1024);       // 1024 bytes
	uint32_t* const tmem_ptr = reinterpret_cast<uint32_t*>(misc + 2048 - 16);
	unsigned char* const stages = misc + 2048;
	const bool in_place = p.slope || p.add;  // the result takes the place of the last input in its stage
	unsigned char* const outs = stages + p.stages * p.stage_bytes;  // [group][result, preactivation]: the result only where it has no place
	const uint32_t out_bytes = (in_place ? 0u : (uint32_t)kTile) + (p.pre ? (uint32_t)kTile : 0u);
	const uint32_t full = sptr(bars), empty = full + 8 * kMaxStages, tfull = empty + 8 * kMaxStages, tempty = tfull + 8 * S::kBufs, wfull = tempty + 8 * S::kBufs,
	               wempty = wfull + 16, wload = wempty + 16;
	const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
	const bool bf = p.bf16 != 0;

	if (tid == 0) {
		for (uint32_t i = 0; i < p.stages; ++i) {
			tc::mbar_init(full + 8 * i, 1);
			tc::mbar_init(empty + 8 * i, 1 + (p.out ? 1 : 0));  // the MMAs, and the epilogue group's last reader
		}
		for (int i = 0; i < S::kBufs; ++i) tc::mbar_init(tfull + 8 * i, 1), tc::mbar_init(tempty + 8 * i, 4);
		for (int i = 0; i < 2; ++i) tc::mbar_init(wfull + 8 * i, 1), tc::mbar_init(wempty + 8 * i, 4);
		tc::mbar_init(wload, 1);
		asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
	}
	for (int i = tid; i < 256; i += S::kThreads) reinterpret_cast<uint16_t*>(misc)[i] = bf ? 0x3f80u : 0x3c00u;
	tc::fence_async_smem();
	if (warp == 0) tc::tmem_alloc(sptr(tmem_ptr), S::kTmem);
	wait_for_previous();
	for (int i = tid; i < 64; i += S::kThreads) bias[i] = p.bias && (uint32_t)i < p.N ? h2f(p.bias[i], bf) : 0.f;
	tc::fence_before_sync();
	__syncthreads();
	tc::fence_after_sync();
	const uint32_t tmem = *tmem_ptr;
	let_next_start();  // (the next kernel's blocks may take tensor memory: only now that this one has its own)
	const uint32_t tiles = (p.n + 127u) / 128u;
	const uint32_t x_at = slabs * kTile, slope_at = x_at + (p.params ? kTile : 0), add_at = slope_at + (p.slope ? kTile : 0);
	bool ok = true;

	if (warp == S::kLoad) {
		if (lane == 0) {
			if (p.out) arrive_expect(wload, slabs * 8192);
			for (uint32_t s = 0; p.out && s < slabs; ++s) {
				if (BACKWARD) tma_load<false>(sptr(weights) + s * 8192, &p.tw, 0, s * 64, wload);
				else tma_load<false>(sptr(weights) + s * 8192, &p.tw, s * 64, 0, wload);
			}
			uint32_t stage = 0, phase = 0;
			for (uint32_t t = blockIdx.x; t < tiles; t += gridDim.x) {
				ok = wait_phase(empty + 8 * stage, phase ^ 1u);
				if (!ok) break;
				const uint32_t at = sptr(stages + stage * p.stage_bytes), bar = full + 8 * stage, row = t * 128;
				arrive_expect(bar, p.stage_bytes);
				for (uint32_t s = 0; s < slabs; ++s) tma_load<false>(at + s * kTile, &p.ta, s * 64, row, bar);
				if (p.params) tma_load<false>(at + x_at, &p.tx, 0, row, bar);
				if (p.slope) tma_load<false>(at + slope_at, &p.tslope, 0, row, bar);
				if (p.add) tma_load<false>(at + add_at, &p.tadd, 0, row, bar);
				if (++stage == p.stages) stage = 0, phase ^= 1u;
			}
		}
		__syncwarp();
	} else if (warp == S::kMma) {
		if (lane == 0) {
			const uint32_t type = bf ? (1u << 7) | (1u << 10) : 0u;
			const uint32_t id = tc::idesc_f16(128, 64, 0, BACKWARD) | type, id_w = tc::idesc_f16(128, 64, 1, 1) | type, id_ones = tc::idesc_f16(128, 16, 1, 0) | type;
			const uint64_t ones = tc::smem_desc(sptr(misc), 128, 256);
			const uint32_t sw = sptr(weights);
			uint32_t stage = 0, phase = 0, buf = 0, buf_phase = 0, wbuf = 0, wphase = 0, i = 0;
			if (p.out) ok = wait_phase(wload, 0);
			for (uint32_t t = blockIdx.x; t < tiles && ok; t += gridDim.x, ++i) {
				ok = wait_phase(full + 8 * stage, phase);
				if (!ok) break;
				tc::fence_after_sync();
				const uint32_t sa = sptr(stages + stage * p.stage_bytes);
				if (p.out) {
					ok = wait_phase(tempty + 8 * buf, buf_phase ^ 1u);
					if (!ok) break;
					tc::fence_after_sync();
					for (uint32_t s = 0; s < slabs; ++s) {
						const int steps = min(4, (int)((p.K - s * 64 + 15) / 16));
						const uint64_t da = desc_k(sa + s * kTile), db = BACKWARD ? desc_mn(sw + s * 8192) : desc_k(sw + s * 8192);
						for (int k = 0; k < steps; ++k) tc::mma_f16(tmem + buf * 64, da + k * 2, db + k * (BACKWARD ? 128 : 2), id, s > 0 || k > 0);
					}
					tc::commit(tfull + 8 * buf);
					if (++buf == S::kBufs) buf = 0, buf_phase ^= 1u;
				}
				if (BACKWARD && p.params) {
					const bool first = i % kRound == 0, last = i % kRound == kRound - 1 || t + gridDim.x >= tiles;
					if (first) {
						ok = wait_phase(wempty + 8 * wbuf, wphase ^ 1u);
						if (!ok) break;
						tc::fence_after_sync();
					}
					// dz as [128 samples][64 columns] slabs: columns are rows of the gradient (a second slab only where there is one)
					const uint64_t da = desc_mn_slabs(sa, slabs > 1 ? kTile : 0), db = desc_mn_slabs(sa + x_at, 0);
#pragma unroll
					for (int k = 0; k < 8; ++k) {
						tc::mma_f16(tmem + 256 + wbuf * 64, da + k * 128, db + k * 128, id_w, !first || k > 0);
						tc::mma_f16(tmem + 384 + wbuf * 16, da + k * 128, ones, id_ones, !first || k > 0);
					}
					if (last) {
						tc::commit(wfull + 8 * wbuf);
						if (++wbuf == 2) wbuf = 0, wphase ^= 1u;
					}
				}
				tc::commit(empty + 8 * stage);
				if (++stage == p.stages) stage = 0, phase ^= 1u;
			}
		}
		__syncwarp();
	} else if (BACKWARD && warp >= S::kDrain) {
		// ---------------------------------------------------------------- weight gradient: thread = row of the gradient
		if (p.params) {
			const uint32_t q = warp & 3, lanes = tmem + ((q * 32u) << 16), m = q * 32 + lane;
			float acc[64], sum = 0.f;
#pragma unroll
			for (int c = 0; c < 64; ++c) acc[c] = 0.f;
			uint32_t wbuf = 0, wphase = 0;
			for (uint32_t t = blockIdx.x; t < tiles; t += gridDim.x * kRound) {
				ok = wait_phase(wfull + 8 * wbuf, wphase);
				if (!ok) break;
				tc::fence_after_sync();
#pragma unroll
				for (int c = 0; c < 64; c += 32) {
					uint32_t r0[16], r1[16];
					tmem_ld16_raw(lanes + 256 + wbuf * 64 + c, r0);
					tmem_ld16_raw(lanes + 256 + wbuf * 64 + c + 16, r1);
					tmem_wait16(r0);
					tmem_wait16(r1);
#pragma unroll
					for (int i = 0; i < 16; ++i) acc[c + i] += __uint_as_float(r0[i]), acc[c + 16 + i] += __uint_as_float(r1[i]);
				}
				uint32_t r[16];
				tmem_ld16_raw(lanes + 384 + wbuf * 16, r);
				tmem_wait16(r);
				sum += __uint_as_float(r[0]);
				tc::fence_before_sync();
				__syncwarp();
				if (lane == 0) arrive(wempty + 8 * wbuf);
				if (++wbuf == 2) wbuf = 0, wphase ^= 1u;
			}
			if (ok && m < p.K) {
				float* o = p.partial + ((uint64_t)blockIdx.x * p.K + m) * p.N;
#pragma unroll
				for (int c = 0; c < 64; ++c)
					if ((uint32_t)c < p.N) o[c] = acc[c];
				p.partial[(uint64_t)gridDim.x * p.K * p.N + (uint64_t)blockIdx.x * p.K + m] = sum;
			}
		}
	} else if (p.out) {
		// ---------------------------------------------------------------- epilogue: thread = row of the tile
		const uint32_t q = warp & 3, group = warp >> 2, lanes = tmem + ((q * 32u) << 16);
		const int row = q * 32 + lane;
		const bool issuer = (tid & 127) == 0;
		unsigned char* const own = outs + group * out_bytes;
		unsigned char* const pre = own + (in_place ? 0 : kTile);
		uint32_t stage = 0, phase = 0, buf = 0, buf_phase = 0, turn = 0;
		for (uint32_t t = blockIdx.x; t < tiles; t += gridDim.x) {
			const bool mine = turn == group;
			if (++turn == S::kGroups) turn = 0;
			const uint32_t now = stage, now_phase = phase, b = buf, b_phase = buf_phase;
			if (++stage == p.stages) stage = 0, phase ^= 1u;
			if (++buf == S::kBufs) buf = 0, buf_phase ^= 1u;
			if (!mine) continue;
			unsigned char* const at = stages + now * p.stage_bytes;
			unsigned char* const result = p.add ? at + add_at : p.slope ? at + slope_at : own;
			ok = wait_phase(tfull + 8 * b, b_phase);
			if (ok && in_place) ok = wait_phase(full + 8 * now, now_phase);  // (complete: the MMAs have read the stage; now this thread may)
			if (!ok) break;
			tc::fence_after_sync();
			if (!in_place || p.pre) {  // the group's own tiles are free when the stores of its last turn have read them
				if (issuer) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
				asm volatile("bar.sync %0, 128;" ::"r"(group + 1) : "memory");
			}
#pragma unroll
			for (int c = 0; c < 2; ++c) {
				uint32_t r0[16], r1[16], other[16];
				tmem_ld16_raw(lanes + b * 64 + c * 32, r0);
				tmem_ld16_raw(lanes + b * 64 + c * 32 + 16, r1);
				tmem_wait16(r0);
				tmem_wait16(r1);
				float v[32];
#pragma unroll
				for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r0[i]), v[16 + i] = __uint_as_float(r1[i]);
				if (c == 1) {
					tc::fence_before_sync();
					__syncwarp();
					if (lane == 0) arrive(tempty + 8 * b);
				}
				if (p.bias) {
#pragma unroll
					for (int i = 0; i < 8; ++i) {
						const float4 f = *reinterpret_cast<const float4*>(bias + c * 32 + 4 * i);
						v[4 * i] += f.x, v[4 * i + 1] += f.y, v[4 * i + 2] += f.z, v[4 * i + 3] += f.w;
					}
				}
				if (p.pre) {
#pragma unroll
					for (int i = 0; i < 16; ++i) other[i] = pack2(v[2 * i], v[2 * i + 1], bf);
					put_units(other, pre, row, c * 4);
				}
				if (p.slope) {
					tile_units(other, at + slope_at, row, c * 4);
					if (p.act == NEUS2B_ACT_RELU) apply_slope<NEUS2B_ACT_RELU>(v, other, bf);
					else if (p.act == NEUS2B_ACT_GELU) apply_slope<NEUS2B_ACT_GELU>(v, other, bf);
					else apply_slope<NEUS2B_ACT_SILU>(v, other, bf);
				} else if (p.act == NEUS2B_ACT_RELU) {
					apply_act<NEUS2B_ACT_RELU>(v);
				} else if (p.act == NEUS2B_ACT_GELU) {
					apply_act<NEUS2B_ACT_GELU>(v);
				} else if (p.act == NEUS2B_ACT_SILU) {
					apply_act<NEUS2B_ACT_SILU>(v);
				}
				if (p.add) {
					tile_units(other, at + add_at, row, c * 4);
#pragma unroll
					for (int i = 0; i < 16; ++i) {
						const float2 f = unpack2(other[i], bf);
						v[2 * i] += f.x;
						v[2 * i + 1] += f.y;
					}
				}
#pragma unroll
				for (int i = 0; i < 16; ++i) other[i] = pack2(v[2 * i], v[2 * i + 1], bf);
				put_units(other, result, row, c * 4);
			}
			tc::fence_async_smem();
			asm volatile("bar.sync %0, 128;" ::"r"(group + 1) : "memory");
			if (issuer) {
				tma_store(&p.tout, sptr(result), 0, t * 128);
				if (p.pre) tma_store(&p.tpre, sptr(pre), 0, t * 128);
				asm volatile("cp.async.bulk.commit_group;" ::: "memory");
				if (in_place) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // before the stage is filled again
				arrive(empty + 8 * now);
			}
		}
		if (issuer) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
	}
	if (!ok) atomicOr(&g_narrow_error, 1u);
	tc::fence_before_sync();
	__syncthreads();
	if (warp == 0) tc::tmem_dealloc(tmem, S::kTmem);
}

static uint32_t narrow_ctas(uint32_t n) { return tiles_of(n, 128) < (uint32_t)kSMs ? tiles_of(n, 128) : (uint32_t)kSMs; }

template <bool BACKWARD>
static int launch_narrow(const Product& r, const Product* w, cudaStream_t stream) {
	NarrowArgs a{};
	const Epilogue& e = r.e;
	a.n = r.M, a.N = r.N, a.K = r.K, a.bf16 = r.bf16;
	a.bias = (const uint16_t*)e.bias;
	a.act = e.act;
	a.out = e.out != nullptr, a.slope = a.out && e.slope_z, a.add = a.out && e.add, a.pre = a.out && e.preact, a.params = w != nullptr;
	auto map = [&](CUtensorMap* m, const void* base, uint64_t ld, uint32_t rows, uint32_t cols, uint32_t box) { return make_map(m, base, ld, rows, cols, box, r.bf16); };
	if (int rc = map(&a.ta, r.a, r.a_ld, r.M, r.K, 128)) return rc;
	if (a.out) {
		if (int rc = BACKWARD ? map(&a.tw, r.b, r.b_ld, r.K, r.N, 64) : map(&a.tw, r.b, r.b_ld, r.N, r.K, 64)) return rc;
		if (int rc = map(&a.tout, e.out, e.out_ld, r.M, r.N, 128)) return rc;
	}
	if (a.params)
		if (int rc = map(&a.tx, w->b, w->b_ld, r.M, w->N, 128)) return rc;
	if (a.slope)
		if (int rc = map(&a.tslope, e.slope_z, e.slope_ld, r.M, r.N, 128)) return rc;
	if (a.add)
		if (int rc = map(&a.tadd, e.add, e.add_ld, r.M, r.N, 128)) return rc;
	if (a.pre)
		if (int rc = map(&a.tpre, e.preact, e.preact_ld, r.M, r.N, 128)) return rc;
	using S = Narrow<BACKWARD>;
	const uint32_t slabs = r.K > 64 ? 2u : 1u;
	const uint32_t outs = a.out ? S::kGroups * ((a.slope || a.add ? 0u : (uint32_t)kTile) + (a.pre ? (uint32_t)kTile : 0u)) : 0u;
	const uint32_t fixed = slabs * 8192 + 2048 + 1024 + outs;
	a.stage_bytes = (slabs + a.params + a.slope + a.add) * kTile;
	a.stages = (kSmemMost - fixed) / a.stage_bytes;
	if (a.stages > (uint32_t)kMaxStages) a.stages = kMaxStages;
	if (a.stages < 2) return NEUS2B_E_UNSUPPORTED;
	a.partial = w ? (float*)w->workspace : nullptr;
	const uint32_t smem = fixed + a.stages * a.stage_bytes;
	N2B_CHECK_CUDA(cudaFuncSetAttribute(narrow_kernel<BACKWARD>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost));
	return launch_behind(narrow_kernel<BACKWARD>, narrow_ctas(r.M), S::kThreads, smem, stream, a);
}

}  // namespace lin

using namespace lin;

// More than two tiles of samples (below, spreading a tile's work over several SMs is faster), and every matrix readable by TMA.  Results
// leave by TMA stores, which write whole 16-byte units of a row: their width has to be a multiple of 8, or the units would reach into
// what the caller keeps behind the row.
bool narrow_fits(const Product& r, bool backward, const Product* w) {
	const Epilogue& e = r.e;
	if (r.M <= 256 || r.N > 64 || r.K > 128 || (e.out && r.N % 8)) return false;
	auto fine = [](const void* p, uint64_t ld) { return !p || tma_ok(p, ld); };
	if (!tma_ok(r.a, r.a_ld)) return false;
	if (e.out && !(tma_ok(r.b, r.b_ld) && tma_ok(e.out, e.out_ld) && fine(e.slope_z, e.slope_ld) && fine(e.add, e.add_ld) && fine(e.preact, e.preact_ld))) return false;
	if (w && !tma_ok(w->b, w->b_ld)) return false;
	return backward || !w;
}
uint64_t narrow_workspace(uint32_t out_width, uint32_t in_width, uint32_t n) {
	return in_width <= 64 && out_width <= 128 ? (uint64_t)narrow_ctas(n) * ((uint64_t)out_width * in_width + out_width) * 4 : 0;
}

int run_narrow(const Product& r, bool backward, const Product* w, cudaStream_t stream) {
	if (!backward) return launch_narrow<false>(r, nullptr, stream);
	if (w && w->workspace_bytes < narrow_workspace(w->M, w->N, w->K)) return NEUS2B_E_INVALID;
	if (int rc = launch_narrow<true>(r, w, stream)) return rc;
	if (!w) return NEUS2B_OK;
	return run_join((const float*)w->workspace, narrow_ctas(r.M), w->M, w->N, (float*)w->e.out, w->column_sums, w->e.accumulate, stream);
}

int read_narrow_error(uint32_t* flags) {
	const cudaError_t e = cudaMemcpyFromSymbol(flags, g_narrow_error, sizeof(*flags));
	return e == cudaSuccess ? NEUS2B_OK : (int)e;
}
int write_narrow_error(uint32_t flags) {
	const cudaError_t e = cudaMemcpyToSymbol(g_narrow_error, &flags, sizeof(flags));
	return e == cudaSuccess ? NEUS2B_OK : (int)e;
}

}  // namespace n2b
