// The products of the linear layer on tcgen05: operands in 128-byte-swizzled shared-memory tiles, sums in tensor memory.
//
// A CTA computes 128 x BN tiles of sum_k a(m, k) b(n, k), 64 k at a time.  Warps 0-7 take finished sums out of tensor memory and run
// the epilogue while the MMA warp fills the other accumulator; one warp issues the MMAs; operand tiles are brought in by TMA, or,
// where rows do not start on 16-byte boundaries, by warps that shift them into place (GATHER).  Both layouts of an operand are
// read as they lie in memory: [m][k] is a K-major tile (128 rows of 64 k), [k][m] an MN-major one (slabs of 64 k x 64 m), so neither
// backward product transposes anything.
#include <cuda.h>

#include "linear.cuh"
#include "tc05.cuh"

namespace n2b {
namespace lin {

static __device__ uint32_t g_error;  // bit 0: a bounded wait ran out

constexpr int kBM = 128, kBK = 64;
constexpr int kEpiWarps = 8, kMmaWarp = 8, kLoadWarp = 9;
constexpr int kGatherWarps = 7;  // warps 9..15
constexpr int kMaxStages = 8, kSmemBudget = 200 * 1024;
constexpr int kChunk = 8;  // weight gradient: k blocks (512 samples) summed in tensor memory before the sum moves to registers

struct alignas(64) Args {
	CUtensorMap ta, tb;
	const uint16_t *a, *b;
	uint64_t a_ld, b_ld;
	uint32_t M, N, K;
	uint32_t tiles_m, tiles_n, splits, cluster;  // cluster: CTAs that share one tile's k range and join through each other's shared memory
	uint32_t bf16;
	float *partial, *column_sums;  // splits > 1: [splits][M][N] and [splits][M]
	uint32_t want_sums;
	Epilogue e;
};

__device__ __forceinline__ uint32_t sptr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint64_t now_ns() {
	uint64_t t;
	asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
	return t;
}
// False when the phase has not completed after four seconds: nothing that a tile waits for takes a millisecond, and every copy that
// was issued has landed long before a role gives up and the CTA ends.
__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t parity) {
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
			else if (t - start > 4000000000ull) return false;
		}
	}
}
__device__ __forceinline__ void arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void arrive_expect(uint32_t bar, uint32_t bytes) {
	asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// x: first column (a multiple of 64), y: first row of a [rows][columns] matrix
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
	asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map),
	             "r"(x), "r"(y), "r"(bar)
	             : "memory");
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
__device__ __forceinline__ uint32_t cluster_rank() {
	uint32_t r;
	asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
	return r;
}
__device__ __forceinline__ void cluster_sync() {
	asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float load_peer(uint32_t addr, uint32_t rank) {
	uint32_t p;
	float v;
	asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(p) : "r"(addr), "r"(rank));
	asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(p) : "memory");
	return v;
}

// Eight 16-bit values that start at any even address, as two aligned 16-byte loads and a shift.
__device__ __forceinline__ uint4 shifted_load(const char* p) {
	const uint32_t s = (uint32_t)(uintptr_t)p & 15u;
	const uint4* q = reinterpret_cast<const uint4*>(p - s);
	const uint4 lo = __ldg(q);
	if (s == 0) return lo;
	const uint4 hi = __ldg(q + 1);
	uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
	if (s & 8u) {
#pragma unroll
		for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
	}
	if (s & 4u) {
#pragma unroll
		for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
	}
	const uint32_t b = (s & 2u) * 8u;
	return make_uint4(__funnelshift_r(w[0], w[1], b), __funnelshift_r(w[1], w[2], b), __funnelshift_r(w[2], w[3], b), __funnelshift_r(w[3], w[4], b));
}
// `count` rows of 64 columns from (row0, col0) of a [rows][cols] matrix of any alignment into a swizzled tile; zeros outside.
// The two aligned loads of a piece may reach up to 14 bytes around it: they are used only where that stays inside the matrix's
// extent in memory, which is the caller's.
__device__ __forceinline__ void gather_box(unsigned char* dst, const uint16_t* base, uint64_t ld, uint32_t rows, uint32_t cols, uint32_t row0, uint32_t col0,
                                           int count, int tid) {
	const char* begin = reinterpret_cast<const char*>(base);
	const char* end = begin + ((uint64_t)(rows - 1) * ld + cols) * 2;
	for (int u = tid; u < count * 8; u += kGatherWarps * 32) {
		const int r = u >> 3, c8 = u & 7;
		const uint32_t row = row0 + r, col = col0 + c8 * 8;
		uint4 v = make_uint4(0, 0, 0, 0);
		if (row < rows && col < cols) {
			const uint16_t* p = base + (uint64_t)row * ld + col;
			const char* q = reinterpret_cast<const char*>(p);
			const char* lo = q - ((uintptr_t)q & 15u);
			if (col + 8 <= cols && lo >= begin && lo + 32 <= end) {
				v = shifted_load(q);
			} else {
				uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
				for (int i = 0; i < 8; ++i)
					if (col + i < cols) w[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
				v = make_uint4(w[0], w[1], w[2], w[3]);
			}
		}
		*reinterpret_cast<uint4*>(dst + r * 128 + ((c8 ^ (r & 7)) << 4)) = v;
	}
}

template <int BN, bool AMN, bool BMN, bool SWAP, bool WGRAD, bool GATHER>
struct Shape {
	static constexpr int kABytes = kBM * 128;
	static constexpr int kBBytes = (BMN && BN < 64 ? 64 : BN) * 128;
	static constexpr int kStage = kABytes + kBBytes;
	static constexpr int kStages = kSmemBudget / kStage < kMaxStages ? kSmemBudget / kStage : kMaxStages;
	static constexpr int kSmem = kStages * kStage + 2048 + 1024;  // ones tile and barriers; alignment of the base
	static constexpr int kTmem = WGRAD ? 512 : (2 * BN < 32 ? 32 : 2 * BN);
	static constexpr int kThreads = (GATHER ? kLoadWarp + kGatherWarps : kLoadWarp + 1) * 32;
};

template <int BN, bool AMN, bool BMN, bool SWAP, bool WGRAD, bool GATHER>
__global__ void __launch_bounds__(Shape<BN, AMN, BMN, SWAP, WGRAD, GATHER>::kThreads, 1) product_kernel(const __grid_constant__ Args p) {
	using S = Shape<BN, AMN, BMN, SWAP, WGRAD, GATHER>;
	extern __shared__ unsigned char smem_raw[];
	unsigned char* smem = smem_raw + ((1024u - (sptr(smem_raw) & 1023u)) & 1023u);
	unsigned char* ones = smem + S::kStages * S::kStage;  // 512 bytes: a [16][16] tile of 1.0
	uint64_t* bars = reinterpret_cast<uint64_t*>(ones + 1024);
	uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(ones + 2048 - 16);
	const uint32_t full = sptr(bars), empty = full + 8 * kMaxStages, tfull = empty + 8 * kMaxStages, tempty = tfull + 16;
	const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
	const bool bf = p.bf16 != 0;

	if (tid == 0) {
		for (int i = 0; i < S::kStages; ++i) {
			tc::mbar_init(full + 8 * i, GATHER ? kGatherWarps * 32 : 1);
			tc::mbar_init(empty + 8 * i, 1);
		}
		for (int i = 0; i < 2; ++i) {
			tc::mbar_init(tfull + 8 * i, 1);
			tc::mbar_init(tempty + 8 * i, kEpiWarps);
		}
		asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
	}
	if (WGRAD)
		for (int i = tid; i < 256; i += S::kThreads) reinterpret_cast<uint16_t*>(ones)[i] = bf ? 0x3f80u : 0x3c00u;
	tc::fence_async_smem();
	if (warp == 0) tc::tmem_alloc(sptr(tmem_ptr), S::kTmem);
	tc::fence_before_sync();
	__syncthreads();
	tc::fence_after_sync();
	const uint32_t tmem = *tmem_ptr;

	const uint32_t tiles = p.tiles_m * p.tiles_n, kblocks = (p.K + kBK - 1) / kBK;
	const uint32_t rank = p.cluster > 1 ? cluster_rank() : 0u;
	const uint32_t first = p.cluster > 1 ? (blockIdx.x / p.cluster) + rank * tiles : blockIdx.x;
	const uint32_t step = p.cluster > 1 ? tiles * p.splits : gridDim.x;  // a cluster computes one tile
	const uint32_t units = tiles * p.splits;
	bool ok = true;
	uint32_t last_m = 0, last_n = 0;

	// unit -> tile and k range.  Tiles go down 16 rows of tiles before they move to the next column: what runs at one time shares operands.
	auto locate = [&](uint32_t u, uint32_t& mt, uint32_t& nt, uint32_t& split, uint32_t& kb0, uint32_t& kb1) {
		split = u / tiles;
		const uint32_t t = u - split * tiles, width = 16u * p.tiles_n, g = t / width, in = t - g * width;
		const uint32_t rows = min(16u, p.tiles_m - g * 16u);
		nt = in / rows;
		mt = g * 16u + (in - nt * rows);
		kb0 = (uint32_t)((uint64_t)split * kblocks / p.splits);
		kb1 = (uint32_t)((uint64_t)(split + 1) * kblocks / p.splits);
	};

	if (warp >= kLoadWarp) {
		// ---------------------------------------------------------------- operand tiles
		uint32_t stage = 0, phase = 0;
		for (uint32_t u = first; u < units && ok; u += step) {
			uint32_t mt, nt, split, kb0, kb1;
			locate(u, mt, nt, split, kb0, kb1);
			for (uint32_t kb = kb0; kb < kb1; ++kb) {
				if (GATHER || lane == 0) ok = wait_phase(empty + 8 * stage, phase ^ 1u);
				if (!ok) break;
				unsigned char* sa = smem + stage * S::kStage;
				unsigned char* sb = sa + S::kABytes;
				if (GATHER) {
					const int t = tid - kLoadWarp * 32;
					if (AMN) {
						for (int s = 0; s < 2; ++s) gather_box(sa + s * 8192, p.a, p.a_ld, p.K, p.M, kb * kBK, mt * kBM + s * 64, 64, t);
					} else {
						gather_box(sa, p.a, p.a_ld, p.M, p.K, mt * kBM, kb * kBK, kBM, t);
					}
					if (BMN) {
						for (int s = 0; s < (BN + 63) / 64; ++s) gather_box(sb + s * 8192, p.b, p.b_ld, p.K, p.N, kb * kBK, nt * BN + s * 64, 64, t);
					} else {
						gather_box(sb, p.b, p.b_ld, p.N, p.K, nt * BN, kb * kBK, BN, t);
					}
					tc::fence_async_smem();
					arrive(full + 8 * stage);
				} else if (lane == 0) {
					const uint32_t bar = full + 8 * stage;
					// slabs that lie outside of the matrix are not loaded: what the tile holds there reaches only sums that are not used
					const int slabs_a = AMN ? min(2, (int)((p.M - mt * kBM + 63) / 64)) : 1;
					const int slabs_b = BMN ? min((BN + 63) / 64, (int)((p.N - nt * BN + 63) / 64)) : 1;
					arrive_expect(bar, (AMN ? slabs_a * 8192 : S::kABytes) + (BMN ? slabs_b * 8192 : S::kBBytes));
					if (AMN) {
						for (int s = 0; s < slabs_a; ++s) tma_load(sptr(sa) + s * 8192, &p.ta, mt * kBM + s * 64, kb * kBK, bar);
					} else {
						tma_load(sptr(sa), &p.ta, kb * kBK, mt * kBM, bar);
					}
					if (BMN) {
						for (int s = 0; s < slabs_b; ++s) tma_load(sptr(sb) + s * 8192, &p.tb, nt * BN + s * 64, kb * kBK, bar);
					} else {
						tma_load(sptr(sb), &p.tb, kb * kBK, nt * BN, bar);
					}
				}
				if (++stage == S::kStages) stage = 0, phase ^= 1u;
			}
			ok = __shfl_sync(~0u, (int)ok, 0) != 0;
		}
	} else if (warp == kMmaWarp) {
		// ---------------------------------------------------------------- MMAs, one thread
		if (lane == 0) {
			const uint32_t type = bf ? (1u << 7) | (1u << 10) : 0u;
			const uint32_t id = tc::idesc_f16(kBM, BN, AMN, BMN) | type, id_ones = tc::idesc_f16(kBM, 16, AMN, 0) | type;
			uint32_t stage = 0, phase = 0, buf = 0, buf_phase = 0;
			for (uint32_t u = first; u < units && ok; u += step) {
				uint32_t mt, nt, split, kb0, kb1;
				locate(u, mt, nt, split, kb0, kb1);
				const bool sums = WGRAD && p.want_sums && nt == 0;
				for (uint32_t c0 = kb0; c0 < kb1 && ok; c0 += WGRAD ? kChunk : kb1 - kb0) {
					const uint32_t c1 = WGRAD ? min(c0 + kChunk, kb1) : kb1;
					ok = wait_phase(tempty + 8 * buf, buf_phase ^ 1u);
					if (!ok) break;
					tc::fence_after_sync();
					for (uint32_t kb = c0; kb < c1; ++kb) {
						ok = wait_phase(full + 8 * stage, phase);
						if (!ok) break;
						tc::fence_after_sync();
						const uint32_t sa = sptr(smem + stage * S::kStage), sb = sa + S::kABytes;
						const int steps = min(4, (int)((p.K - kb * kBK + 15) / 16));
						for (int k = 0; k < steps; ++k) {
							const uint64_t da = AMN ? desc_mn(sa + k * 2048) : desc_k(sa + k * 32);
							const uint64_t db = BMN ? desc_mn(sb + k * 2048) : desc_k(sb + k * 32);
							const uint32_t more = kb > c0 || k > 0;
							tc::mma_f16(tmem + buf * BN, da, db, id, more);
							if (sums) tc::mma_f16(tmem + 2 * BN + buf * 16, da, tc::smem_desc(sptr(ones), 128, 256), id_ones, more);
						}
						tc::commit(empty + 8 * stage);
						if (++stage == S::kStages) stage = 0, phase ^= 1u;
					}
					if (!ok) break;
					tc::commit(tfull + 8 * buf);
					if (++buf == 2) buf = 0, buf_phase ^= 1u;
				}
			}
		}
		__syncwarp();
	} else {
		// ---------------------------------------------------------------- epilogue: warp w owns rows 32 (w % 4) .. and columns (w / 4) BN / 2 ..
		const uint32_t q = warp & 3, half = warp >> 2;
		const uint32_t lanes = tmem + ((q * 32u) << 16);
		constexpr int kCols = BN / 2;
		uint32_t buf = 0, buf_phase = 0;
		for (uint32_t u = first; u < units && ok; u += step) {
			uint32_t mt, nt, split, kb0, kb1;
			locate(u, mt, nt, split, kb0, kb1);
			last_m = mt, last_n = nt;
			const uint32_t m = mt * kBM + q * 32 + lane, n0 = nt * BN + half * kCols;
			if (WGRAD) {
				float acc[kCols], sum = 0.f;
#pragma unroll
				for (int i = 0; i < kCols; ++i) acc[i] = 0.f;
				const bool sums = p.want_sums && nt == 0 && half == 0;
				for (uint32_t c0 = kb0; c0 < kb1 && ok; c0 += kChunk) {
					ok = wait_phase(tfull + 8 * buf, buf_phase);
					if (!ok) break;
					tc::fence_after_sync();
#pragma unroll
					for (int c = 0; c < kCols; c += 16) {
						uint32_t r[16];
						tmem_ld16_raw(lanes + buf * BN + half * kCols + c, r);
						tmem_wait16(r);
#pragma unroll
						for (int i = 0; i < 16; ++i) acc[c + i] += __uint_as_float(r[i]);
					}
					if (sums) {
						uint32_t r[16];
						tmem_ld16_raw(lanes + 2 * BN + buf * 16, r);
						tmem_wait16(r);
						sum += __uint_as_float(r[0]);
					}
					tc::fence_before_sync();
					__syncwarp();
					if (lane == 0) arrive(tempty + 8 * buf);
					if (++buf == 2) buf = 0, buf_phase ^= 1u;
				}
				if (!ok) break;
				if (m < p.M) {
					Epilogue e = p.e;
					if (p.splits > 1) {
						e.out = p.partial + (uint64_t)split * p.M * p.N;
						e.out_ld = p.N;
						e.accumulate = 0;
						e.vec = (p.N & 3u) == 0;
					}
#pragma unroll
					for (int c = 0; c < kCols; c += 8) {
						if (!p.e.out) break;
						float v[8];
#pragma unroll
						for (int i = 0; i < 8; ++i) v[i] = acc[c + i];
						if (e.vec && n0 + c + 8 <= p.N) {
							finish_eight(e, bf, m, n0 + c, v);
						} else {
#pragma unroll
							for (int i = 0; i < 8; ++i)
								if (n0 + c + i < p.N) finish_one(e, bf, m, n0 + c + i, v[i]);
						}
					}
					if (sums) {
						if (p.splits > 1) p.partial[(uint64_t)p.splits * p.M * p.N + (uint64_t)split * p.M + m] = sum;
						else p.column_sums[m] = p.e.accumulate ? p.column_sums[m] + sum : sum;
					}
				}
			} else {
				ok = wait_phase(tfull + 8 * buf, buf_phase);
				if (!ok) break;
				tc::fence_after_sync();
				float* joined = reinterpret_cast<float*>(smem);  // cluster: [BN][129]; every tile of this CTA's only unit has been consumed
#pragma unroll 1
				for (int c = 0; c < kCols; c += 16) {
					uint32_t r[16];
					tmem_ld16_raw(lanes + buf * BN + half * kCols + c, r);
					tmem_wait16(r);
					if (p.cluster > 1) {
#pragma unroll
						for (int i = 0; i < 16; ++i) joined[(half * kCols + c + i) * 129 + q * 32 + lane] = __uint_as_float(r[i]);
					} else if (SWAP) {
						// m is the feature, the tile's columns are samples
#pragma unroll
						for (int i = 0; i < 16; ++i)
							if (m < p.M && n0 + c + i < p.N) finish_one(p.e, bf, n0 + c + i, m, __uint_as_float(r[i]));
					} else if (m < p.M) {
#pragma unroll
						for (int k = 0; k < 16; k += 8) {
							float v[8];
#pragma unroll
							for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[k + i]);
							if (p.e.vec && n0 + c + k + 8 <= p.N) {
								finish_eight(p.e, bf, m, n0 + c + k, v);
							} else {
#pragma unroll
								for (int i = 0; i < 8; ++i)
									if (n0 + c + k + i < p.N) finish_one(p.e, bf, m, n0 + c + k + i, v[i]);
							}
						}
					}
				}
				tc::fence_before_sync();
				__syncwarp();
				if (lane == 0) arrive(tempty + 8 * buf);
				if (++buf == 2) buf = 0, buf_phase ^= 1u;
			}
		}
	}
	if (!ok) atomicOr(&g_error, 1u);
	if (!WGRAD && p.cluster > 1) {
		// every CTA adds up its share of the tile over the cluster's partial sums, in rank order, and finishes it
		__syncwarp();
		cluster_sync();
		uint32_t mt, nt, split, kb0, kb1;
		locate(first, mt, nt, split, kb0, kb1);
		const uint32_t joined = sptr(smem), count = kBM * BN / p.cluster;
		for (uint32_t i = tid; i < count; i += S::kThreads) {
			const uint32_t idx = rank * count + i;
			const uint32_t m = SWAP ? idx % kBM : idx / BN, n = SWAP ? idx / kBM : idx % BN;
			if (mt * kBM + m >= p.M || nt * BN + n >= p.N) continue;
			float v = 0.f;
			for (uint32_t s = 0; s < p.cluster; ++s) v += load_peer(joined + (n * 129 + m) * 4, s);
			if (SWAP) finish_one(p.e, bf, nt * BN + n, mt * kBM + m, v);
			else finish_one(p.e, bf, mt * kBM + m, nt * BN + n, v);
		}
		__syncwarp();
		cluster_sync();
	}
	tc::fence_before_sync();
	__syncthreads();
	if (warp == 0) tc::tmem_dealloc(tmem, S::kTmem);
}

// partial sums of the splits, in order
__global__ void __launch_bounds__(256) join_kernel(const float* __restrict__ partial, uint32_t splits, uint32_t M, uint32_t N, float* __restrict__ out,
                                                    float* __restrict__ sums, int accumulate) {
	const uint64_t n = (uint64_t)M * N, total = n + (sums ? M : 0);
	for (uint64_t i = (out ? 0 : n) + blockIdx.x * 256ull + threadIdx.x; i < total; i += gridDim.x * 256ull) {
		const bool is_sum = i >= n;
		const float* q = is_sum ? partial + splits * n + (i - n) : partial + i;
		const uint64_t pitch = is_sum ? M : n;
		float v = 0.f;
		for (uint32_t s = 0; s < splits; ++s) v += q[s * pitch];
		float* o = is_sum ? sums + (i - n) : out + i;
		*o = accumulate ? *o + v : v;
	}
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                             CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeFn encode_fn() {
	static EncodeFn fn = [] {
		void* q = nullptr;
		cudaDriverEntryPointQueryResult res;
		if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &q, 12000, cudaEnableDefault, &res) != cudaSuccess) q = nullptr;
		return (EncodeFn)q;
	}();
	return fn;
}
// [rows][cols] matrix read in boxes of 64 columns and box_rows rows
static int make_map(CUtensorMap* map, const void* base, uint64_t ld, uint32_t rows, uint32_t cols, uint32_t box_rows, bool bf16) {
	const EncodeFn fn = encode_fn();
	if (!fn) return NEUS2B_E_NO_DEVICE;
	const cuuint64_t dims[2] = {cols, rows}, strides[1] = {ld * 2};
	const cuuint32_t box[2] = {64, box_rows}, unit[2] = {1, 1};
	const CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base), dims, strides, box, unit,
	                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
	return r == CUDA_SUCCESS ? NEUS2B_OK : NEUS2B_E_INVALID;
}
// TMA reads rows that start on 16-byte boundaries, less than 2^40 bytes apart
static bool tma_ok(const void* p, uint64_t ld) { return ((uintptr_t)p & 15u) == 0 && (ld & 7u) == 0 && ld < (1ull << 39); }

template <int BN, bool AMN, bool BMN, bool SWAP, bool WGRAD, bool GATHER>
static int launch(Args& a, uint32_t ctas, cudaStream_t stream) {
	using S = Shape<BN, AMN, BMN, SWAP, WGRAD, GATHER>;
	auto kernel = product_kernel<BN, AMN, BMN, SWAP, WGRAD, GATHER>;
	if (!GATHER) {
		if (int rc = AMN ? make_map(&a.ta, a.a, a.a_ld, a.K, a.M, 64, a.bf16) : make_map(&a.ta, a.a, a.a_ld, a.M, a.K, kBM, a.bf16)) return rc;
		if (int rc = BMN ? make_map(&a.tb, a.b, a.b_ld, a.K, a.N, 64, a.bf16) : make_map(&a.tb, a.b, a.b_ld, a.N, a.K, BN, a.bf16)) return rc;
	}
	N2B_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
	cudaLaunchConfig_t cfg{};
	cfg.gridDim = dim3(ctas);
	cfg.blockDim = dim3(S::kThreads);
	cfg.dynamicSmemBytes = S::kSmem;
	cfg.stream = stream;
	cudaLaunchAttribute attr[1];
	attr[0].id = cudaLaunchAttributeClusterDimension;
	attr[0].val.clusterDim.x = a.cluster;
	attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
	cfg.attrs = attr;
	cfg.numAttrs = a.cluster > 1 ? 1 : 0;
	const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, (const Args)a);
	if (e != cudaSuccess) return (int)e;
	N2B_CHECK_LAUNCH();
	return NEUS2B_OK;
}

template <int BN, bool AMN, bool BMN, bool SWAP, bool WGRAD>
static int launch_any(Args& a, uint32_t ctas, cudaStream_t stream) {
	if (tma_ok(a.a, a.a_ld) && tma_ok(a.b, a.b_ld)) return launch<BN, AMN, BMN, SWAP, WGRAD, false>(a, ctas, stream);
	return launch<BN, AMN, BMN, SWAP, WGRAD, true>(a, ctas, stream);
}

// Tile width, and over how many CTAs of a cluster a tile's sum is split, for `tiles_of(BN)` tiles and `kblocks` steps of 64.
struct Plan {
	uint32_t bn, cluster;
};
static uint32_t cluster_for(uint64_t tiles, uint32_t kblocks) {
	uint32_t c = 1;
	while (c < 8 && tiles * c * 2 <= (uint64_t)kSMs && kblocks >= c * 2 * 4) c *= 2;  // at least four steps stay for every CTA
	return c;
}

template <bool BMN_FORWARD>
static int product_of(const Product& p, cudaStream_t stream) {
	Args a{};
	a.bf16 = p.bf16;
	a.K = p.K;
	a.e = p.e;
	a.splits = a.cluster = 1;
	const uint32_t kblocks = (p.K + kBK - 1) / kBK;
	auto go = [&](auto launcher, uint32_t bn) {
		a.tiles_m = (a.M + kBM - 1) / kBM;
		a.tiles_n = (a.N + bn - 1) / bn;
		const uint64_t tiles = (uint64_t)a.tiles_m * a.tiles_n;
		if (tiles >= (1ull << 31)) return NEUS2B_E_TOO_LARGE;
		a.cluster = bn <= 128 ? cluster_for(tiles, kblocks) : 1u;
		a.splits = a.cluster;
		return launcher(a, (uint32_t)(a.cluster > 1 ? tiles * a.cluster : (tiles < (uint64_t)kSMs ? tiles : (uint64_t)kSMs)), stream);
	};
	if (p.M <= 64) {
		// few samples: the weights are the 128-row operand, the samples its columns
		a.a = (const uint16_t*)p.b, a.a_ld = p.b_ld, a.M = p.N;
		a.b = (const uint16_t*)p.a, a.b_ld = p.a_ld, a.N = p.M;
		if (p.M <= 32) return go(launch_any<32, BMN_FORWARD, false, true, false>, 32);
		return go(launch_any<64, BMN_FORWARD, false, true, false>, 64);
	}
	a.a = (const uint16_t*)p.a, a.a_ld = p.a_ld, a.M = p.M;
	a.b = (const uint16_t*)p.b, a.b_ld = p.b_ld, a.N = p.N;
	const uint64_t rows = (p.M + kBM - 1) / kBM;
	if (p.N > 128 && rows * ((p.N + 255) / 256) >= (uint64_t)kSMs) return go(launch_any<256, false, BMN_FORWARD, false, false>, 256);
	if (p.N > 64 && rows * ((p.N + 127) / 128) >= (uint64_t)kSMs) return go(launch_any<128, false, BMN_FORWARD, false, false>, 128);
	return go(launch_any<64, false, BMN_FORWARD, false, false>, 64);
}

constexpr uint32_t kWgradBN = 128;
static uint32_t wgrad_splits(uint32_t M, uint32_t N, uint32_t K) {
	const uint64_t tiles = (uint64_t)((M + kBM - 1) / kBM) * ((N + kWgradBN - 1) / kWgradBN);
	const uint32_t kblocks = (K + kBK - 1) / kBK;
	const uint64_t fill = (uint64_t)kSMs / tiles, most = kblocks / kChunk;
	const uint64_t s = fill < most ? fill : most;
	return s > 1 ? (uint32_t)s : 1u;
}

}  // namespace lin

using namespace lin;

int read_linear_error(uint32_t* flags) {
	const cudaError_t e = cudaMemcpyFromSymbol(flags, g_error, sizeof(*flags));
	return e == cudaSuccess ? NEUS2B_OK : (int)e;
}
int write_linear_error(uint32_t flags) {
	const cudaError_t e = cudaMemcpyToSymbol(g_error, &flags, sizeof(flags));
	return e == cudaSuccess ? NEUS2B_OK : (int)e;
}

int run_product(const Product& p, cudaStream_t stream) { return p.b_mn ? product_of<true>(p, stream) : product_of<false>(p, stream); }

static uint64_t partial_bytes(uint32_t M, uint32_t N, uint32_t K) {
	const uint64_t s = wgrad_splits(M, N, K);
	return s > 1 ? s * ((uint64_t)M * N + M) * 4 : 0;
}
uint64_t wgrad_workspace(uint32_t out_width, uint32_t in_width, uint32_t n) {
	const uint64_t a = partial_bytes(out_width, in_width, n), b = partial_bytes(out_width, sums_only_width(out_width), n);
	return a > b ? a : b;
}

int run_weight_gradient(const Product& p, cudaStream_t stream) {
	Args a{};
	a.bf16 = p.bf16;
	a.M = p.M, a.N = p.N, a.K = p.K;
	a.a = (const uint16_t*)p.a, a.a_ld = p.a_ld, a.b = (const uint16_t*)p.b, a.b_ld = p.b_ld;
	a.e = p.e;
	a.tiles_m = (p.M + kBM - 1) / kBM;
	a.tiles_n = (p.N + kWgradBN - 1) / kWgradBN;
	a.splits = wgrad_splits(p.M, p.N, p.K);
	a.cluster = 1;
	a.column_sums = p.column_sums;
	a.want_sums = p.column_sums != nullptr;
	a.partial = (float*)p.workspace;
	if (a.splits > 1 && p.workspace_bytes < partial_bytes(p.M, p.N, p.K)) return NEUS2B_E_INVALID;
	const uint64_t units = (uint64_t)a.tiles_m * a.tiles_n * a.splits;
	if (units >= (1ull << 31)) return NEUS2B_E_TOO_LARGE;
	if (int rc = launch_any<kWgradBN, true, true, false, true>(a, (uint32_t)(units < (uint64_t)kSMs ? units : kSMs), stream)) return rc;
	if (a.splits > 1) {
		const uint64_t total = (uint64_t)p.M * p.N + p.M;
		join_kernel<<<(uint32_t)(total < 256ull * 8 * kSMs ? (total + 255) / 256 : 8 * kSMs), 256, 0, stream>>>(a.partial, a.splits, p.M, p.N, (float*)p.e.out, p.column_sums, p.e.accumulate);
		N2B_CHECK_LAUNCH();
	}
	return NEUS2B_OK;
}

}  // namespace n2b
