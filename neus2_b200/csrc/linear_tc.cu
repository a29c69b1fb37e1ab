// The products of the linear layer on tcgen05: operands in 128-byte-swizzled shared-memory tiles, sums in tensor memory.
//
// A CTA computes 128 x BN tiles of sum_k a(m, k) b(n, k), 64 k at a time.  One warp brings in operand tiles by TMA, one issues the MMAs,
// 8 or 16 warps take finished sums out of tensor memory and run the epilogue while the MMA warp fills another accumulator.  Both
// layouts of an operand are read as they lie in memory: [m][k] is a K-major tile (128 rows of 64 k), [k][m] an MN-major one (slabs of
// 64 k x 64 m), so neither backward product transposes anything.  Operands whose rows do not start on 16-byte boundaries, which TMA
// cannot read, are copied once ahead of the product (realign_kernel).
#include <algorithm>

#include "linear_tc.cuh"

namespace n2b {
namespace lin {

static __device__ uint32_t g_error;  // bit 0: a bounded wait ran out

constexpr int kChunkBytes = 32 * 64;  // 32 x 32 values on their way between the epilogue and global memory
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
	uint32_t stages, chunks;
	Epilogue e;
};

// Copies of up to three matrices with rows on 16-byte boundaries, for operands that have none.  A thread's unit is 16 bytes of a copy, eight
// values that start at any even address: two aligned 16-byte reads and a shift, zeros behind the row's end.  The reads may reach up to
// 14 bytes around the values: they are used only where that stays inside the matrix's extent in memory, which is the caller's.
struct Realign {
	const uint16_t* from[3];
	uint64_t from_ld[3];
	uint16_t* to[3];
	uint32_t rows[3], cols[3];
	uint32_t blocks[4];  // first block of each, and behind the last
};
__device__ __noinline__ uint4 unit_by_entries(const uint16_t* p, uint32_t n) {  // at the matrix's two ends
	uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
	for (uint32_t i = 0; i < 8; ++i)
		if (i < n) w[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
	return make_uint4(w[0], w[1], w[2], w[3]);
}
// the 16 bytes from byte `shift` (even, below 16) of two neighbouring units on, the first n values of them
__device__ __forceinline__ uint4 shifted(const uint4& lo, const uint4& hi, uint32_t shift, uint32_t n) {
	uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
	if (shift & 8u) {
#pragma unroll
		for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
	}
	if (shift & 4u) {
#pragma unroll
		for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
	}
	const uint32_t b = (shift & 2u) * 8u;
	uint32_t y[4];
#pragma unroll
	for (int i = 0; i < 4; ++i) {
		y[i] = __funnelshift_r(w[i], w[i + 1], b);
		if (2 * i + 1 >= (int)n) y[i] = 2 * i < (int)n ? y[i] & 0xffffu : 0u;
	}
	return make_uint4(y[0], y[1], y[2], y[3]);
}
// A thread has kAhead units on their way in shared memory: registers for them would leave too few threads to fill the memory's latency.
constexpr int kAhead = 8, kRealignSmem = kAhead * 2 * 256 * 16, kRealignBlocks = 3 * kSMs;
__global__ void __launch_bounds__(256, 3) realign_kernel(const Realign r) {
	extern __shared__ uint4 ring[];  // [kAhead][2][256]
	let_next_start();
	const int k = blockIdx.x >= r.blocks[2] ? 2 : blockIdx.x >= r.blocks[1] ? 1 : 0;
	const uint32_t per = (r.cols[k] + 7) / 8, cols = r.cols[k];
	const uint64_t units = (uint64_t)r.rows[k] * per, width = (uint64_t)(r.blocks[k + 1] - r.blocks[k]) * 256;
	// a thread's units lie `width` apart: (row, column) moves on by one division's worth, taken once
	struct Place {
		uint64_t u;
		uint32_t row, col;
	};
	Place ahead;
	ahead.u = (uint64_t)(blockIdx.x - r.blocks[k]) * 256 + threadIdx.x;
	ahead.row = (uint32_t)(ahead.u / per), ahead.col = (uint32_t)(ahead.u - (uint64_t)ahead.row * per);
	Place now = ahead;
	const uint32_t step_row = (uint32_t)(width / per), step_col = (uint32_t)(width - (uint64_t)step_row * per);
	auto next = [&](Place& p) {
		p.u += width, p.row += step_row, p.col += step_col;
		if (p.col >= per) p.col -= per, ++p.row;
	};
	const char *begin = reinterpret_cast<const char*>(r.from[k]), *end = begin + ((uint64_t)(r.rows[k] - 1) * r.from_ld[k] + cols) * 2;
	auto address = [&](const Place& p, const char*& down) {
		const char* q = begin + ((uint64_t)p.row * r.from_ld[k] + p.col * 8u) * 2;
		down = q - ((uintptr_t)q & 15u);
		return q;
	};
	auto fetch = [&](uint32_t slot) {
		const char* down;
		address(ahead, down);
		if (ahead.u < units && down >= begin && down + 32 <= end) {
			const uint32_t s = sptr(ring + slot * 512 + threadIdx.x);
			asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(s), "l"(down) : "memory");
			asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(s + 256 * 16), "l"(down + 16) : "memory");
		}
		asm volatile("cp.async.commit_group;" ::: "memory");
		next(ahead);
	};
	wait_for_previous();
#pragma unroll 1
	for (int i = 0; i < kAhead; ++i) fetch(i);
#pragma unroll 1
	for (uint32_t slot = 0; now.u < units; slot = slot + 1 == kAhead ? 0 : slot + 1) {
		asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
		const char *down, *q = address(now, down);
		const uint32_t n = min(8u, cols - now.col * 8);
		uint4 v;
		if (down >= begin && down + 32 <= end) v = shifted(ring[slot * 512 + threadIdx.x], ring[slot * 512 + 256 + threadIdx.x], (uint32_t)(q - down), n);
		else v = unit_by_entries(reinterpret_cast<const uint16_t*>(q), n);
		reinterpret_cast<uint4*>(r.to[k])[now.u] = v;
		next(now);
		fetch(slot);
	}
	asm volatile("cp.async.wait_all;" ::: "memory");
}

// What a block of one variant is made of.  Large products are bound by the MMAs and the power they draw: 8192 x 4096 -> 4096 with bias, GELU and
// residual takes 210 us in a burst, 1310 TFLOP/s of the 1679 that a library product reaches in one, and 236 to 247 us over seconds, 1110 to
// 1165 of 1403 (the product alone 193 and 226, a library product of the shape 183 and 217); short k by the epilogue (8192 x 1024 -> 4096
// with the slopes of a GELU 69 us, 59 without; its chain of loads, MUFU and stores of 16 warps at 96 registers), small products by latency
// (100 x 256 -> 256 6.6 us, one row through 4096 -> 4096 10.4 us where its weights alone take 5.1).  Tiles of 128 x 64 and 128 x 128 take
// their operands out of the L2 at about 45 bytes a cycle and SM.  PAIR: two CTAs of a cluster compute a 256 x BN tile together, each with 128 of its rows in its
// tensor memory and half of B's tile in its shared memory.  The epilogue is a long chain of dependent steps, so that it takes 16 warps to
// keep up with the MMAs: on wide tiles they share the columns, narrow ones (BN 64) go to four groups in turn, each with an accumulator.
template <int BN, bool AMN, bool BMN, bool SWAP, bool WGRAD, bool PAIR>
struct Shape {
	static constexpr int kBRows = PAIR ? BN / 2 : BN;  // of B's tile in this CTA
	static constexpr int kABytes = kBM * 128;
	static constexpr int kBBytes = (BMN && kBRows < 64 ? 64 : kBRows) * 128;
	static constexpr int kStage = kABytes + kBBytes;
	static constexpr bool kTurns = BN == 64 && !SWAP && !WGRAD, kMany = !SWAP && !WGRAD && (PAIR || BN <= 128);
	static constexpr int kHalves = kTurns ? 1 : kMany ? 4 : 2, kGroups = kTurns ? 4 : 1, kBufs = kTurns ? 4 : 2;
	static constexpr int kEpiWarps = 4 * kHalves * kGroups, kMmaWarp = kEpiWarps, kLoadWarp = kEpiWarps + 1;
	static constexpr int kThreads = (kLoadWarp + 1) * 32;
	// Shared memory behind the operand stages: chunks of the epilogue (`chunks` for every warp), ones tile and barriers; alignment of the base.
	static constexpr int fixed(int chunks) { return (SWAP ? 0 : kEpiWarps * (WGRAD ? 4096 : chunks * kChunkBytes)) + 2048 + 1024; }
	static constexpr int stages(int chunks) {
		// few samples: room for a second CTA on the SM
		const int room = ((SWAP ? kSmemMost / 2 - 1024 : kSmemMost) - fixed(chunks)) / kStage;
		return room < kMaxStages ? room : kMaxStages;
	}
	static constexpr int kCols = kBufs * BN + (WGRAD && !PAIR ? 32 : 0);
	static constexpr int kTmem = kCols <= 64 ? 64 : kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
};

// ---- 32 x 32 values of a matrix between global memory and registers, through 2 KB of shared memory of a warp.  Global memory is read
// (asynchronously) and written in whole row segments (64 bytes), a thread computes on one row.  Where rows do not start on 16-byte
// boundaries a thread moves two of its entries (rows on 4-byte boundaries) or one: still whole segments of rows per instruction.  The
// 16-byte units of a row are permuted so that neither side's accesses collide.
__device__ __forceinline__ uint32_t unit_at(int row, int unit) { return (uint32_t)(row * 64 + ((unit ^ ((row >> 1) & 3)) << 4)); }
__device__ __forceinline__ void chunk_fetch(uint32_t chunk, const void* base, uint64_t ld, uint32_t row0, uint32_t rows, uint32_t col0, uint32_t cols, int vec, int lane) {
	const uint16_t* p = (const uint16_t*)base;
	if (vec == 16) {
		const uint32_t r0 = row0 + (lane >> 2), c = col0 + (lane & 3) * 8;
		const uint16_t* q = p + (uint64_t)r0 * ld + c;
#pragma unroll
		for (int i = 0; i < 4; ++i, q += 8 * ld)
			if (r0 + 8 * i < rows && c < cols)
				asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(chunk + unit_at(i * 8 + (lane >> 2), lane & 3)), "l"(q) : "memory");
	} else if (vec == 4) {  // two rows an instruction
		const uint32_t c = col0 + (lane & 15) * 2;
		uint32_t r = lane >> 4;
		const uint16_t* q = p + (uint64_t)(row0 + r) * ld + c;
#pragma unroll 4
		for (; r < 32; r += 2, q += 2 * ld)
			if (row0 + r < rows && c < cols)
				asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(chunk + unit_at(r, (lane & 15) >> 2) + (lane & 3) * 4), "l"(q) : "memory");
	} else {
		const uint16_t* q = p + (uint64_t)row0 * ld + col0 + lane;
#pragma unroll
		for (int h = 0; h < 32; h += 16) {  // 16 on their way together
			uint16_t v[16];
#pragma unroll
			for (int i = 0; i < 16; ++i, q += ld) v[i] = row0 + h + i < rows && col0 + lane < cols ? *q : (uint16_t)0;
#pragma unroll
			for (int i = 0; i < 16; ++i) asm volatile("st.shared.u16 [%0], %1;" ::"r"(chunk + unit_at(h + i, lane >> 3) + (lane & 7) * 2), "h"(v[i]) : "memory");
		}
	}
}
// The thread's own row of a chunk that has arrived.
__device__ __forceinline__ void chunk_row(uint32_t (&row)[16], const unsigned char* chunk, int lane) {
#pragma unroll
	for (int u = 0; u < 4; ++u) {
		const uint4 v = *reinterpret_cast<const uint4*>(chunk + unit_at(lane, u));
		row[4 * u] = v.x, row[4 * u + 1] = v.y, row[4 * u + 2] = v.z, row[4 * u + 3] = v.w;
	}
}
__device__ __forceinline__ void chunk_store(const uint32_t (&row)[16], void* base, uint64_t ld, uint32_t row0, uint32_t rows, uint32_t col0, uint32_t cols,
                                            unsigned char* chunk, int vec, int lane) {
	uint16_t* p = (uint16_t*)base;
	__syncwarp();  // what was here before has been read
#pragma unroll
	for (int u = 0; u < 4; ++u)
		*reinterpret_cast<uint4*>(chunk + unit_at(lane, u)) = make_uint4(row[4 * u], row[4 * u + 1], row[4 * u + 2], row[4 * u + 3]);
	__syncwarp();
	if (vec == 16) {
		const uint32_t r0 = row0 + (lane >> 2), c = col0 + (lane & 3) * 8;
		uint16_t* q = p + (uint64_t)r0 * ld + c;
#pragma unroll
		for (int i = 0; i < 4; ++i, q += 8 * ld) {
			const uint4 v = *reinterpret_cast<const uint4*>(chunk + unit_at(i * 8 + (lane >> 2), lane & 3));
			if (r0 + 8 * i < rows && c < cols) *reinterpret_cast<uint4*>(q) = v;
		}
	} else if (vec == 4) {
		const uint32_t c = col0 + (lane & 15) * 2;
		uint32_t r = lane >> 4;
		uint16_t* q = p + (uint64_t)(row0 + r) * ld + c;
#pragma unroll 4
		for (; r < 32; r += 2, q += 2 * ld) {
			const uint32_t v = *reinterpret_cast<const uint32_t*>(chunk + unit_at(r, (lane & 15) >> 2) + (lane & 3) * 4);
			if (row0 + r < rows && c < cols) *reinterpret_cast<uint32_t*>(q) = v;
		}
	} else {
		uint16_t* q = p + (uint64_t)row0 * ld + col0 + lane;
#pragma unroll 8
		for (int i = 0; i < 32; ++i, q += ld) {
			const uint16_t v = *reinterpret_cast<const uint16_t*>(chunk + unit_at(i, lane >> 3) + (lane & 7) * 2);
			if (row0 + i < rows && col0 + lane < cols) *q = v;
		}
	}
}
// 32 x 32 fp32 sums of a weight gradient, a row a thread, to global memory in row segments (128 bytes) through 4 KB of a warp: written
// a row a thread they would take 32 accesses of a few bytes an instruction (8 us a tile where rows are unaligned).
__device__ __forceinline__ void sums_store(const float (&v)[32], const Epilogue& e, uint32_t row0, uint32_t rows, uint32_t col0, uint32_t cols, unsigned char* chunk,
                                           int lane) {
	__syncwarp();  // what was here before has been read
#pragma unroll
	for (int u = 0; u < 8; ++u)
		*reinterpret_cast<float4*>(chunk + lane * 128 + ((u ^ (lane & 7)) << 4)) = make_float4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
	__syncwarp();
	if (e.vec == 16 && col0 + 32 <= cols) {
		float* o = (float*)e.out + (uint64_t)(row0 + (lane >> 3)) * e.out_ld + col0 + (lane & 7) * 4;
#pragma unroll 4
		for (int r = lane >> 3; r < 32; r += 4, o += 4 * e.out_ld) {
			float4 s = *reinterpret_cast<const float4*>(chunk + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
			if (row0 + r >= rows) continue;
			if (e.accumulate) {
				const float4 a = *reinterpret_cast<const float4*>(o);
				s.x += a.x, s.y += a.y, s.z += a.z, s.w += a.w;
			}
			*reinterpret_cast<float4*>(o) = s;
		}
	} else {
		float* o = (float*)e.out + (uint64_t)row0 * e.out_ld + col0 + lane;
#pragma unroll 8
		for (int r = 0; r < 32; ++r, o += e.out_ld) {
			const float s = *reinterpret_cast<const float*>(chunk + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
			if (row0 + r < rows && col0 + lane < cols) *o = e.accumulate ? *o + s : s;
		}
	}
}

// Place of sum (m, n) of a tile in shared memory.  Features are contiguous, as they are in the result: what a warp reads of another
// CTA's tile has to be (spread over 32 lines it takes 8 us instead of 1.5).
template <int BN, bool SWAP>
__device__ __forceinline__ uint32_t joined_at(uint32_t m, uint32_t n) {
	return SWAP ? n * (kBM + 1) + m : m * (BN + 1) + n;
}

template <int BN, bool AMN, bool BMN, bool SWAP, bool WGRAD, bool PAIR>
__global__ void __launch_bounds__(Shape<BN, AMN, BMN, SWAP, WGRAD, PAIR>::kThreads, SWAP ? 2 : 1) product_kernel(const __grid_constant__ Args p) {
	using S = Shape<BN, AMN, BMN, SWAP, WGRAD, PAIR>;
	extern __shared__ unsigned char smem_raw[];
	unsigned char* smem = smem_raw + ((1024u - (sptr(smem_raw) & 1023u)) & 1023u);
	const uint32_t stages = p.stages;
	unsigned char* ones = smem + stages * S::kStage;  // 512 bytes: a [16][16] tile of 1.0
	unsigned char* chunks = ones + 2048;              // p.chunks for every epilogue warp
	uint64_t* bars = reinterpret_cast<uint64_t*>(ones + 1024);
	uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(ones + 2048 - 16);
	const uint32_t full = sptr(bars), empty = full + 8 * kMaxStages, tfull = empty + 8 * kMaxStages, tempty = tfull + 8 * 4;
	const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
	const bool bf = p.bf16 != 0;
	const uint32_t rank = PAIR || p.cluster > 1 ? cluster_rank() : 0u;

	if (tid == 0) {
		for (uint32_t i = 0; i < stages; ++i) {
			tc::mbar_init(full + 8 * i, 1);
			tc::mbar_init(empty + 8 * i, 1);
		}
		for (int i = 0; i < S::kBufs; ++i) {
			tc::mbar_init(tfull + 8 * i, 1);
			tc::mbar_init(tempty + 8 * i, 4 * S::kHalves * (PAIR ? 2 : 1));
		}
		asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
	}
	if (WGRAD)
		for (int i = tid; i < 256; i += S::kThreads) reinterpret_cast<uint16_t*>(ones)[i] = bf ? 0x3f80u : 0x3c00u;
	tc::fence_async_smem();
	if (warp == 0) tmem_alloc<PAIR>(sptr(tmem_ptr), S::kTmem);
	tc::fence_before_sync();
	if (PAIR) cluster_sync();
	else __syncthreads();
	tc::fence_after_sync();
	const uint32_t tmem = *tmem_ptr;
	let_next_start();     // (the next kernel's blocks may take tensor memory: only now that this one has its own)
	wait_for_previous();  // the set-up above runs beside the end of the kernel ahead

	// With few samples, or where a cluster splits k, a CTA computes one tile; otherwise a pair, or a CTA by itself, takes every `step`-th.
	const uint32_t tiles = p.tiles_m * p.tiles_n, kblocks = (p.K + kBK - 1) / kBK;
	const uint32_t first = PAIR ? blockIdx.x / 2 : p.cluster > 1 ? (blockIdx.x / p.cluster) + rank * tiles : blockIdx.x;
	const uint32_t units = tiles * p.splits;
	const bool single = !PAIR && (SWAP || p.cluster > 1);
	const uint32_t step = PAIR ? gridDim.x / 2 : single ? units : gridDim.x;
	const uint32_t row_offset = PAIR ? rank * kBM : 0u;
	constexpr int kTileM = PAIR ? 2 * kBM : kBM;
	bool ok = true;

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

	if (warp >= S::kLoadWarp) {
		// ---------------------------------------------------------------- operand tiles by TMA, one thread
		uint32_t stage = 0, phase = 0;
		const uint32_t full_lead = PAIR ? peer_address(full, 0) : full;  // a pair's tiles are counted in by the first CTA
		for (uint32_t u = first; lane == 0 && u < units && ok; u += step) {
			uint32_t mt, nt, split, kb0, kb1;
			locate(u, mt, nt, split, kb0, kb1);
			const uint32_t m0 = mt * kTileM + row_offset, n0 = nt * BN + (PAIR ? rank * S::kBRows : 0u);
			// slabs that lie outside of the matrix are not loaded: what the tile holds there reaches only sums that are not used
			const int slabs_a = AMN ? (PAIR ? 2 : min(2, (int)((p.M - m0 + 63) / 64))) : 1;
			const int slabs_b = BMN ? (PAIR ? S::kBRows / 64 : min((BN + 63) / 64, (int)((p.N - n0 + 63) / 64))) : 1;
			const uint32_t bytes = (AMN ? slabs_a * 8192 : S::kABytes) + (BMN ? slabs_b * 8192 : S::kBBytes);
			for (uint32_t kb = kb0; kb < kb1; ++kb) {
				ok = wait_phase(empty + 8 * stage, phase ^ 1u);
				if (!ok) break;
				const uint32_t sa = sptr(smem + stage * S::kStage), sb = sa + S::kABytes, bar = full_lead + 8 * stage;
				if (!PAIR) arrive_expect(full + 8 * stage, bytes);
				else if (rank == 0) arrive_expect(full + 8 * stage, 2 * bytes);
				if (AMN) {
					for (int s = 0; s < slabs_a; ++s) tma_load<PAIR>(sa + s * 8192, &p.ta, m0 + s * 64, kb * kBK, bar);
				} else {
					tma_load<PAIR>(sa, &p.ta, kb * kBK, m0, bar);
				}
				if (BMN) {
					for (int s = 0; s < slabs_b; ++s) tma_load<PAIR>(sb + s * 8192, &p.tb, n0 + s * 64, kb * kBK, bar);
				} else {
					tma_load<PAIR>(sb, &p.tb, kb * kBK, n0, bar);
				}
				if (++stage == stages) stage = 0, phase ^= 1u;
			}
		}
		__syncwarp();
	} else if (warp == S::kMmaWarp) {
		// ---------------------------------------------------------------- MMAs, one thread (of a pair's first CTA)
		if (lane == 0 && (!PAIR || rank == 0)) {
			const uint32_t type = bf ? (1u << 7) | (1u << 10) : 0u;
			const uint32_t id = tc::idesc_f16(kTileM, BN, AMN, BMN) | type, id_ones = tc::idesc_f16(kBM, 16, AMN, 0) | type;
			uint32_t stage = 0, phase = 0, buf = 0, buf_phase = 0;
			for (uint32_t u = first; u < units && ok; u += step) {
				uint32_t mt, nt, split, kb0, kb1;
				locate(u, mt, nt, split, kb0, kb1);
				const bool sums = WGRAD && !PAIR && p.want_sums && nt == 0;
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
						const uint64_t da = AMN ? desc_mn(sa) : desc_k(sa), db = BMN ? desc_mn(sb) : desc_k(sb);
						constexpr uint64_t kStepA = (AMN ? 2048 : 32) / 16, kStepB = (BMN ? 2048 : 32) / 16;  // 16 k further
						const uint32_t d = tmem + buf * BN;
						if (p.K - kb * kBK >= kBK) {
							// one thread issues all MMAs of the SM: nothing but the two descriptors' sums between them
							mma<PAIR>(d, da, db, id, kb > c0);
#pragma unroll
							for (int k = 1; k < 4; ++k) mma<PAIR>(d, da + k * kStepA, db + k * kStepB, id, 1u);
						} else {
							const int steps = (int)((p.K - kb * kBK + 15) / 16);
							for (int k = 0; k < steps; ++k) mma<PAIR>(d, da + k * kStepA, db + k * kStepB, id, kb > c0 || k > 0);
						}
						if (sums) {
							const int steps = min(4, (int)((p.K - kb * kBK + 15) / 16));
							for (int k = 0; k < steps; ++k)
								tc::mma_f16(tmem + S::kBufs * BN + buf * 16, da + k * kStepA, tc::smem_desc(sptr(ones), 128, 256), id_ones, kb > c0 || k > 0);
						}
						commit<PAIR>(empty + 8 * stage);
						if (++stage == stages) stage = 0, phase ^= 1u;
					}
					if (!ok) break;
					commit<PAIR>(tfull + 8 * buf);
					if (++buf == S::kBufs) buf = 0, buf_phase ^= 1u;
				}
			}
		}
		__syncwarp();
	} else {
		// ---------------------------------------------------------------- epilogue: warp w owns rows 32 (w % 4) ..
		const uint32_t q = warp & 3, half = (warp >> 2) % S::kHalves, group = (warp >> 2) / S::kHalves;
		const uint32_t lanes = tmem + ((q * 32u) << 16);
		constexpr int kCols = BN / S::kHalves;  // columns half * kCols .. of the tile
		// the result of 32 columns goes out through the place that its last input came in by
		unsigned char* const slope = chunks + warp * p.chunks * kChunkBytes;
		unsigned char* const addend = slope + (p.chunks - 1) * kChunkBytes;
		unsigned char* const result = addend;
		uint32_t turn = 0, buf = 0, buf_phase = 0;
		auto next_buf = [&] {
			if (++buf == S::kBufs) buf = 0, buf_phase ^= 1u;
		};
		auto release = [&] {
			tc::fence_before_sync();
			__syncwarp();
			if (lane == 0) {
				if (PAIR) arrive_remote(peer_address(tempty + 8 * buf, 0));
				else arrive(tempty + 8 * buf);
			}
		};
		for (uint32_t u = first; u < units && ok; u += step) {
			if (S::kGroups > 1) {
				const bool mine = turn == group;
				if (++turn == S::kGroups) turn = 0;
				if (!mine) {
					next_buf();
					continue;
				}
			}
			uint32_t mt, nt, split, kb0, kb1;
			locate(u, mt, nt, split, kb0, kb1);
			const uint32_t row0 = mt * kTileM + row_offset + q * 32, m = row0 + lane, n0 = nt * BN + half * kCols;
			if (WGRAD) {
				float acc[kCols], sum = 0.f;
#pragma unroll
				for (int i = 0; i < kCols; ++i) acc[i] = 0.f;
				const bool sums = !PAIR && p.want_sums && nt == 0 && half == 0;
				for (uint32_t c0 = kb0; c0 < kb1 && ok; c0 += kChunk) {
					ok = wait_phase(tfull + 8 * buf, buf_phase);
					if (!ok) break;
					tc::fence_after_sync();
#pragma unroll
					for (int c = 0; c < kCols; c += 32) {
						uint32_t r0[16], r1[16];
						tmem_ld16_raw(lanes + buf * BN + half * kCols + c, r0);
						tmem_ld16_raw(lanes + buf * BN + half * kCols + c + 16, r1);
						tmem_wait16(r0);
						tmem_wait16(r1);
#pragma unroll
						for (int i = 0; i < 16; ++i) acc[c + i] += __uint_as_float(r0[i]), acc[c + 16 + i] += __uint_as_float(r1[i]);
					}
					if (sums) {
						uint32_t r[16];
						tmem_ld16_raw(lanes + S::kBufs * BN + buf * 16, r);
						tmem_wait16(r);
						sum += __uint_as_float(r[0]);
					}
					release();
					next_buf();
				}
				if (!ok) break;
				if (p.cluster > 1) {  // (every operand tile of this CTA's only unit has been consumed)
					float* const joined = reinterpret_cast<float*>(smem);
#pragma unroll
					for (int i = 0; i < kCols; ++i) joined[joined_at<BN, SWAP>(q * 32 + lane, half * kCols + i)] = acc[i];
					if (sums) joined[kBM * (BN + 1) + q * 32 + lane] = sum;
					continue;
				}
				Epilogue e = p.e;
				if (p.splits > 1) {
					e.out = p.partial + (uint64_t)split * p.M * p.N;
					e.out_ld = p.N;
					e.accumulate = 0;
					e.vec = (p.N & 3u) == 0 ? 16 : 4;
				}
#pragma unroll
				for (int c = 0; c < kCols; c += 32) {
					if (n0 + c >= p.N) break;
					float v[32];
#pragma unroll
					for (int i = 0; i < 32; ++i) v[i] = acc[c + i];
					sums_store(v, e, row0, p.M, n0 + c, p.N, chunks + warp * 4096, lane);
				}
				if (sums && m < p.M) {
					if (p.splits > 1) p.partial[(uint64_t)p.splits * p.M * p.N + (uint64_t)split * p.M + m] = sum;
					else p.column_sums[m] = p.e.accumulate ? p.column_sums[m] + sum : sum;
				}
			} else if (single) {
				ok = wait_phase(tfull + 8 * buf, buf_phase);
				if (!ok) break;
				tc::fence_after_sync();
				float* joined = reinterpret_cast<float*>(smem);  // every operand tile of this CTA's only unit has been consumed
#pragma unroll 1
				for (uint32_t c = half * kCols; c < (half + 1) * kCols && nt * BN + c < p.N; c += 16) {
					uint32_t r[16];
					tmem_ld16_raw(lanes + buf * BN + c, r);
					tmem_wait16(r);
#pragma unroll
					for (int i = 0; i < 16; ++i) joined[joined_at<BN, SWAP>(q * 32 + lane, c + i)] = __uint_as_float(r[i]);
				}
			} else {
				const Epilogue& e = p.e;
				// the inputs' next 32 columns are on their way while the sums are still being computed
				auto fetch = [&](uint32_t col) {
					if (e.slope_z) chunk_fetch(sptr(slope), e.slope_z, e.slope_ld, row0, p.M, col, p.N, e.vec, lane);
					if (e.add) chunk_fetch(sptr(addend), e.add, e.add_ld, row0, p.M, col, p.N, e.vec, lane);
					asm volatile("cp.async.commit_group;" ::: "memory");
				};
				const bool inputs = e.slope_z || e.add;
				if (inputs) fetch(n0);
				ok = wait_phase(tfull + 8 * buf, buf_phase);
				if (!ok) break;
				tc::fence_after_sync();
#pragma unroll 1
				for (int c = 0; c < kCols; c += 32) {
					const uint32_t col = n0 + c;
					uint32_t r0[16], r1[16], other[16];
					tmem_ld16_raw(lanes + buf * BN + half * kCols + c, r0);
					tmem_ld16_raw(lanes + buf * BN + half * kCols + c + 16, r1);
					tmem_wait16(r0);
					tmem_wait16(r1);
					float v[32];
#pragma unroll
					for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r0[i]), v[16 + i] = __uint_as_float(r1[i]);
					if (c + 32 >= kCols) release();
					if (e.bias) {
						const uint16_t* b = (const uint16_t*)e.bias;
						if (e.vec == 16 && col + 32 <= p.N) {
#pragma unroll
							for (int i = 0; i < 4; ++i) {
								const uint4 w = __ldg(reinterpret_cast<const uint4*>(b + col) + i);
								const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
								for (int j = 0; j < 4; ++j) {
									const float2 f = unpack2(ws[j], bf);
									v[8 * i + 2 * j] += f.x;
									v[8 * i + 2 * j + 1] += f.y;
								}
							}
						} else {  // a column a thread, handed round
							const float mine = col + lane < p.N ? h2f(b[col + lane], bf) : 0.f;
#pragma unroll
							for (int i = 0; i < 32; ++i) v[i] += __shfl_sync(0xffffffffu, mine, i);
						}
					}
					if (e.preact) {
#pragma unroll
						for (int i = 0; i < 16; ++i) other[i] = pack2(v[2 * i], v[2 * i + 1], bf);
						chunk_store(other, e.preact, e.preact_ld, row0, p.M, col, p.N, slope, e.vec, lane);
					}
					if (inputs) {
						asm volatile("cp.async.wait_all;" ::: "memory");
						__syncwarp();
					}
					if (e.slope_z) {
						chunk_row(other, slope, lane);
						if (e.act == NEUS2B_ACT_RELU) apply_slope<NEUS2B_ACT_RELU>(v, other, bf);
						else if (e.act == NEUS2B_ACT_GELU) apply_slope<NEUS2B_ACT_GELU>(v, other, bf);
						else apply_slope<NEUS2B_ACT_SILU>(v, other, bf);
					} else if (e.act == NEUS2B_ACT_RELU) {
						apply_act<NEUS2B_ACT_RELU>(v);
					} else if (e.act == NEUS2B_ACT_GELU) {
						apply_act<NEUS2B_ACT_GELU>(v);
					} else if (e.act == NEUS2B_ACT_SILU) {
						apply_act<NEUS2B_ACT_SILU>(v);
					}
					if (e.add) {
						chunk_row(other, addend, lane);
#pragma unroll
						for (int i = 0; i < 16; ++i) {
							const float2 f = unpack2(other[i], bf);
							v[2 * i] += f.x;
							v[2 * i + 1] += f.y;
						}
					}
#pragma unroll
					for (int i = 0; i < 16; ++i) other[i] = pack2(v[2 * i], v[2 * i + 1], bf);
					chunk_store(other, e.out, e.out_ld, row0, p.M, col, p.N, result, e.vec, lane);
					if (inputs && c + 32 < kCols) {
						__syncwarp();
						fetch(col + 32);
					}
				}
				if (inputs) __syncwarp();  // before the next tile's inputs come in
				next_buf();
			}
		}
	}
	if (!ok) atomicOr(&g_error, 1u);
	if (single) {
		// every CTA adds up its share of the tile over the cluster's sums, in rank order, and finishes it: two entries at a time, whose
		// inputs are on their way together
		__syncwarp();
		if (p.cluster > 1) cluster_sync();
		else __syncthreads();
		uint32_t mt, nt, split, kb0, kb1;
		locate(first, mt, nt, split, kb0, kb1);
		if (WGRAD && p.want_sums && nt == 0 && rank == 0 && tid < kBM && mt * kBM + tid < p.M) {
			float v = 0.f;
			for (uint32_t s = 0; s < p.cluster; ++s) v += load_peer(sptr(smem) + (kBM * (BN + 1) + tid) * 4, s);
			float* const o = p.column_sums + mt * kBM + tid;
			*o = p.e.accumulate ? *o + v : v;
		}
		const uint32_t joined = sptr(smem), rows = min((uint32_t)kBM, p.M - mt * kBM), cols = min((uint32_t)BN, p.N - nt * BN);
		const uint32_t count = rows * cols, stride = p.cluster * S::kThreads;
		const Epilogue& e = p.e;
		for (uint32_t base = rank * S::kThreads + tid; base < count; base += 2 * stride) {
			float v[2];
			uint32_t at[2], feature[2];
			uint64_t sample[2];
			bool in[2];
			uint16_t z[2], add[2], bias[2];
#pragma unroll
			for (int k = 0; k < 2; ++k) {
				const uint32_t idx = base + k * stride, slow = idx / (SWAP ? rows : cols), fast = idx - slow * (SWAP ? rows : cols);
				const uint32_t m = SWAP ? fast : slow, n = SWAP ? slow : fast;
				in[k] = idx < count;
				at[k] = in[k] ? joined + joined_at<BN, SWAP>(m, n) * 4 : joined;
				feature[k] = SWAP ? mt * kBM + m : nt * BN + n;
				sample[k] = SWAP ? nt * BN + n : mt * kBM + m;
				v[k] = 0.f;
				z[k] = add[k] = bias[k] = 0;
				if (in[k] && e.bias) bias[k] = ((const uint16_t*)e.bias)[feature[k]];
				if (in[k] && e.slope_z) z[k] = ((const uint16_t*)e.slope_z)[sample[k] * e.slope_ld + feature[k]];
				if (in[k] && e.add) add[k] = ((const uint16_t*)e.add)[sample[k] * e.add_ld + feature[k]];
			}
			if (p.cluster > 1) {
				for (uint32_t s = 0; s < p.cluster; ++s)
#pragma unroll
					for (int k = 0; k < 2; ++k) v[k] += load_peer(at[k], s);
			} else {
#pragma unroll
				for (int k = 0; k < 2; ++k) v[k] = load_peer(at[k], 0);
			}
#pragma unroll
			for (int k = 0; k < 2; ++k) {
				if (!in[k]) continue;
				if (WGRAD) {
					float* const o = (float*)e.out + sample[k] * e.out_ld + feature[k];
					*o = e.accumulate ? *o + v[k] : v[k];
					continue;
				}
				float y = v[k] + (e.bias ? h2f(bias[k], bf) : 0.f);
				if (e.preact) ((uint16_t*)e.preact)[sample[k] * e.preact_ld + feature[k]] = f2h(y, bf);
				y = e.slope_z ? y * act_slope(e.act, h2f(z[k], bf)) : act_value(e.act, y);
				if (e.add) y += h2f(add[k], bf);
				((uint16_t*)e.out)[sample[k] * e.out_ld + feature[k]] = f2h(y, bf);
			}
		}
		__syncwarp();
		if (p.cluster > 1) cluster_sync();
	}
	tc::fence_before_sync();
	__syncwarp();
	if (PAIR) cluster_sync();  // the other CTA's MMAs and arrivals reach into this one
	else __syncthreads();
	tc::fence_after_sync();
	if (warp == 0) tmem_dealloc<PAIR>(tmem, S::kTmem);
}

// Sums of the splits' parts.  A thread takes VEC neighbouring entries; the rows of a block's threads share the splits and are joined in
// order.
template <int VEC>
__global__ void __launch_bounds__(1024) join_kernel(const float* __restrict__ partial, uint32_t splits, uint32_t M, uint32_t N, float* __restrict__ out,
                                                    float* __restrict__ sums, int accumulate) {
	extern __shared__ float s[];  // [blockDim.y][VEC][blockDim.x]
	let_next_start();
	wait_for_previous();
	const uint64_t n = (uint64_t)M * N, groups = n / VEC, total = groups + (sums ? M : 0);
	for (uint64_t base = (uint64_t)blockIdx.x * blockDim.x; base < total; base += (uint64_t)gridDim.x * blockDim.x) {
		const uint64_t i = base + threadIdx.x;
		const bool is_sum = i >= groups;
		float v[VEC] = {};
		if (i < total) {
			if (is_sum) {
				const float* q = partial + splits * n + (i - groups);
#pragma unroll 4
				for (uint32_t k = threadIdx.y; k < splits; k += blockDim.y) v[0] += q[(uint64_t)k * M];
			} else if (VEC == 4) {
				const float4* q = reinterpret_cast<const float4*>(partial) + i;
#pragma unroll 4
				for (uint32_t k = threadIdx.y; k < splits; k += blockDim.y) {
					const float4 a = q[k * groups];
					v[0] += a.x, v[1 % VEC] += a.y, v[2 % VEC] += a.z, v[3 % VEC] += a.w;
				}
			} else {
#pragma unroll 4
				for (uint32_t k = threadIdx.y; k < splits; k += blockDim.y) v[0] += partial[k * n + i];
			}
		}
		if (blockDim.y > 1) {
#pragma unroll
			for (int e = 0; e < VEC; ++e) s[(threadIdx.y * VEC + e) * blockDim.x + threadIdx.x] = v[e];
			__syncthreads();
			if (threadIdx.y == 0)
				for (uint32_t k = 1; k < blockDim.y; ++k)
#pragma unroll
					for (int e = 0; e < VEC; ++e) v[e] += s[(k * VEC + e) * blockDim.x + threadIdx.x];
			__syncthreads();
		}
		if (threadIdx.y == 0 && i < total) {
			if (VEC == 4 && !is_sum) {
				float4* o = reinterpret_cast<float4*>(out) + i;
				const float4 a = accumulate ? *o : make_float4(0.f, 0.f, 0.f, 0.f);
				*o = make_float4(a.x + v[0], a.y + v[1 % VEC], a.z + v[2 % VEC], a.w + v[3 % VEC]);
			} else {
				float* o = is_sum ? sums + (i - groups) : out + i;
				*o = accumulate ? *o + v[0] : v[0];
			}
		}
	}
}

template <int BN, bool AMN, bool BMN, bool SWAP, bool WGRAD, bool PAIR>
static int launch(Args& a, uint32_t ctas, cudaStream_t stream) {
	using S = Shape<BN, AMN, BMN, SWAP, WGRAD, PAIR>;
	auto kernel = product_kernel<BN, AMN, BMN, SWAP, WGRAD, PAIR>;
	if (int rc = AMN ? make_map(&a.ta, a.a, a.a_ld, a.K, a.M, 64, a.bf16) : make_map(&a.ta, a.a, a.a_ld, a.M, a.K, kBM, a.bf16)) return rc;
	if (int rc = BMN ? make_map(&a.tb, a.b, a.b_ld, a.K, a.N, 64, a.bf16) : make_map(&a.tb, a.b, a.b_ld, a.N, a.K, S::kBRows, a.bf16)) return rc;
	// one chunk for every epilogue input, and one for z where it does not go the same way as the result
	a.chunks = (a.e.slope_z && a.e.add) || (a.e.preact && a.e.add) ? 2 : 1;
	a.stages = S::stages((int)a.chunks);
	const int smem = (int)a.stages * S::kStage + S::fixed((int)a.chunks);
	N2B_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost));  // (the same from every thread)
	cudaLaunchConfig_t cfg{};
	cfg.gridDim = dim3(ctas);
	cfg.blockDim = dim3(S::kThreads);
	cfg.dynamicSmemBytes = smem;
	cfg.stream = stream;
	cudaLaunchAttribute attr[2];
	attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
	attr[0].val.programmaticStreamSerializationAllowed = 1;
	attr[1].id = cudaLaunchAttributeClusterDimension;
	attr[1].val.clusterDim.x = PAIR ? 2 : a.cluster;
	attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
	cfg.attrs = attr;
	cfg.numAttrs = PAIR || a.cluster > 1 ? 2 : 1;
	const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, (const Args)a);
	if (e != cudaSuccess) return (int)e;
	N2B_CHECK_LAUNCH();
	return NEUS2B_OK;
}

// Over how many CTAs of a cluster a tile's sum is split: as many as run at one time.  A cluster lies within a GPC, so that fewer SMs can
// be used the larger it is (cudaOccupancyMaxActiveClusters with one and two CTAs on an SM); one cluster too many takes the time of a
// second round.  Splitting pays from so many steps of 64 on: with few samples from two for each CTA; with 128 samples a tile the join
// takes 3 us where two CTAs share it and 1.5 where eight do (100 samples, 512 -> 512: 7.4 us over clusters, 8.0 without; 1000 samples: 9.7
// over clusters of two, 8.6 without).
constexpr uint32_t kClusterFit[2][3] = {{148, 132, 120}, {296, 284, 264}};  // CTAs in clusters of 2, 4, 8
static uint32_t cluster_for(uint64_t tiles, uint32_t kblocks, bool swap) {
	constexpr uint32_t kSteps[2][3] = {{16, 8, 16}, {4, 8, 16}};
	for (int c = 2; c >= 0; --c)
		if ((tiles << (c + 1)) <= kClusterFit[swap][c] && kblocks >= kSteps[swap][c]) return 2u << c;
	return 1;
}

template <bool BMN>
static int product_of(const Product& p, cudaStream_t stream) {
	Args a{};
	a.bf16 = p.bf16;
	a.K = p.K;
	a.e = p.e;
	a.splits = a.cluster = 1;
	const uint32_t kblocks = tiles_of(p.K, kBK);
	// grid of one-CTA tiles
	auto grid = [&](uint32_t bn, bool swap) -> uint32_t {
		a.tiles_m = tiles_of(a.M, kBM);
		a.tiles_n = tiles_of(a.N, bn);
		const uint64_t tiles = (uint64_t)a.tiles_m * a.tiles_n;
		if (tiles >= (1ull << 31)) return 0;
		a.cluster = a.splits = bn <= 128 ? cluster_for(tiles, kblocks, swap) : 1u;
		return (uint32_t)(swap || tiles < kSMs ? tiles * a.cluster : kSMs);
	};
#define N2B_GO(BN, AMN, BMN_, SWAP)                                         \
	do {                                                                    \
		const uint32_t ctas = grid(BN, SWAP);                               \
		if (!ctas) return NEUS2B_E_TOO_LARGE;                               \
		return launch<BN, AMN, BMN_, SWAP, false, false>(a, ctas, stream);  \
	} while (0)
	if (p.M <= 64) {
		// few samples: the weights are the 128-row operand, the samples its columns
		a.a = (const uint16_t*)p.b, a.a_ld = p.b_ld, a.M = p.N;
		a.b = (const uint16_t*)p.a, a.b_ld = p.a_ld, a.N = p.M;
		if (p.M <= 32) N2B_GO(32, BMN, false, true);
		N2B_GO(64, BMN, false, true);
	}
	a.a = (const uint16_t*)p.a, a.a_ld = p.a_ld, a.M = p.M;
	a.b = (const uint16_t*)p.b, a.b_ld = p.b_ld, a.N = p.N;
	// The tile with the least time, counted as rounds over the SMs times what a tile costs: its columns, and 64 more for its rows and its
	// epilogue.  A pair's 256 x 256 tile reads each operand half as often as two CTAs' tiles: it counts 0.85 of two.
	const uint64_t rows = tiles_of(p.M, kBM);
	auto cost = [&](uint32_t bn) { return (rows * tiles_of(p.N, bn) + kSMs - 1) / kSMs * (bn + 64) * 20; };
	const uint64_t pairs = (uint64_t)tiles_of(p.M, 2 * kBM) * tiles_of(p.N, 256), pair_cost = (pairs + kSMs / 2 - 1) / (kSMs / 2) * (256 + 64) * 17;
	const uint64_t c64 = cost(64), c128 = cost(128), c256 = cost(256);
	if (pair_cost < c64 && pair_cost < c128 && pair_cost < c256) {
		a.tiles_m = tiles_of(a.M, 2 * kBM);
		a.tiles_n = tiles_of(a.N, 256);
		if (pairs >= (1ull << 31)) return NEUS2B_E_TOO_LARGE;
		return launch<256, false, BMN, false, false, true>(a, 2 * (uint32_t)(pairs < kSMs / 2 ? pairs : kSMs / 2), stream);
	}
	if (c256 < c128 && c256 < c64) N2B_GO(256, false, BMN, false);
	if (c128 < c64) N2B_GO(128, false, BMN, false);
	N2B_GO(64, false, BMN, false);
#undef N2B_GO
}

// Weight gradient: tiles of out_width x in_width, k the samples.  Few tiles share the samples out over the SMs and are joined afterwards.
// One CTA's 128 x 128 tile takes about 430 cycles for 64 samples (its operands' way through shared memory), a pair's 256 x 256 tile 512
// (its MMAs) and, where the column sums are wanted, the pass over dz that takes them: 4 us and 4 TB/s.  The plan with the
// fewest cycles is taken.  Parts are joined by a pass of their own (6000 cycles with its launch), or, where a cluster's CTAs are enough parts,
// through its shared memory (3000): 1328 samples, 160 -> 192: 14.1 us for the whole backward pass, 16.9 with a pass of its own.
struct WgradPlan {
	bool pair;
	uint32_t tiles_m, tiles_n, splits, cluster;
};
static WgradPlan wgrad_plan(uint32_t M, uint32_t N, uint32_t K, bool sums) {
	const uint32_t kblocks = tiles_of(K, kBK);
	uint64_t best = 0;
	WgradPlan plan{};
	for (int pair = 0; pair < 2; ++pair) {
		const uint32_t size = pair ? 256 : 128, slots = pair ? kSMs / 2 : kSMs;
		const uint64_t tiles = (uint64_t)tiles_of(M, size) * tiles_of(N, size), fill = slots / tiles, most = kblocks / kChunk;
		const uint64_t splits = fill < most ? (fill ? fill : 1) : (most ? most : 1);
		const uint64_t cycles = (tiles * splits + slots - 1) / slots * ((kblocks + splits - 1) / splits) * (pair ? 512 : 430) +
		                        (splits > 1 ? 6000 : 0) + (pair && sums ? 8000 + (uint64_t)K * M / 1000 : 0);
		if (!pair || cycles < best) {
			best = cycles;
			plan = WgradPlan{pair != 0, tiles_of(M, size), tiles_of(N, size), (uint32_t)splits, 1};
		}
		for (int c = 0; !pair && c < 3; ++c) {
			const uint64_t together = ((uint64_t)kblocks + (2u << c) - 1) / (2u << c) * 430 + 3000;
			if ((tiles << (c + 1)) > kClusterFit[0][c] || together >= best) continue;
			best = together;
			plan = WgradPlan{false, tiles_of(M, size), tiles_of(N, size), 2u << c, 2u << c};
		}
	}
	return plan;
}
static uint64_t plan_bytes(const WgradPlan& w, uint32_t M, uint32_t N) {
	return w.splits > 1 && w.cluster == 1 ? (uint64_t)w.splits * ((uint64_t)M * N + M) * 4 : 0;
}

// Column sums of a [rows][cols] matrix with rows on 16-byte boundaries.  A cluster of 8 blocks takes COLS columns, its blocks every 8th group of
// rows, a thread 8 columns; rows of a warp are joined by shuffles, warps and blocks in order through shared memory.  Bound by the read: 8192
// x 1024 bf16 6 us (two launches with partial sums between them 7.6).
template <int COLS>
__global__ void __launch_bounds__(512) column_sums_kernel(const uint16_t* __restrict__ a, uint64_t ld, uint32_t rows, uint32_t cols, uint32_t bf16,
                                                          float* __restrict__ out, int accumulate) {
	constexpr int kAcross = COLS / 8, kDown = 512 / kAcross;  // threads of a row, rows of a block
	__shared__ float s[16][COLS], block[COLS];
	wait_for_previous();
	let_next_start();
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
	const uint32_t first = blockIdx.x / 8 * COLS, c = first + threadIdx.x % kAcross * 8, rank = cluster_rank();
	const bool bf = bf16 != 0;
	float v[8] = {};
	if (c + 8 <= cols) {
		for (uint32_t r = rank * kDown + threadIdx.x / kAcross; r < rows; r += 8 * kDown * 8) {
			uint4 q[8];  // on their way together
#pragma unroll
			for (uint32_t k = 0; k < 8; ++k) {
				const uint32_t at = r + k * 8 * kDown;
				q[k] = at < rows ? __ldg(reinterpret_cast<const uint4*>(a + (uint64_t)at * ld + c)) : make_uint4(0, 0, 0, 0);
			}
#pragma unroll
			for (uint32_t k = 0; k < 8; ++k) {
				const uint32_t w[4] = {q[k].x, q[k].y, q[k].z, q[k].w};
#pragma unroll
				for (int i = 0; i < 4; ++i) {
					const float2 f = unpack2(w[i], bf);
					v[2 * i] += f.x, v[2 * i + 1] += f.y;
				}
			}
		}
	} else if (c < cols) {
		for (uint32_t r = rank * kDown + threadIdx.x / kAcross; r < rows; r += 8 * kDown)
#pragma unroll
			for (uint32_t i = 0; i < 8; ++i)
				if (c + i < cols) v[i] += h2f(a[(uint64_t)r * ld + c + i], bf);
	}
	__syncwarp();
#pragma unroll
	for (int i = 0; i < 8; ++i) {
#pragma unroll
		for (int o = kAcross; o < 32; o *= 2) v[i] += __shfl_xor_sync(~0u, v[i], o);
		if (lane < kAcross) s[warp][lane * 8 + i] = v[i];
	}
	__syncthreads();
	if (threadIdx.x < COLS) {
		float t = 0.f;
#pragma unroll
		for (int k = 0; k < 16; ++k) t += s[k][threadIdx.x];
		block[threadIdx.x] = t;
	}
	__syncthreads();
	cluster_sync();
	if (rank == 0 && threadIdx.x < COLS && first + threadIdx.x < cols) {
		float part[8], t = 0.f;
#pragma unroll
		for (int k = 0; k < 8; ++k) part[k] = load_peer(sptr(block + threadIdx.x), k);
#pragma unroll
		for (int k = 0; k < 8; ++k) t += part[k];
		float* const o = out + first + threadIdx.x;
		*o = accumulate ? *o + t : t;
	}
	__syncwarp();
	cluster_sync();  // (before the other blocks' memory goes)
}

}  // namespace lin

using namespace lin;

int read_linear_error(uint32_t* flags) {
	uint32_t narrow = 0;
	const cudaError_t e = cudaMemcpyFromSymbol(flags, g_error, sizeof(*flags));
	if (e != cudaSuccess) return (int)e;
	if (int rc = read_narrow_error(&narrow)) return rc;
	*flags |= narrow;
	return NEUS2B_OK;
}
int write_linear_error(uint32_t flags) {
	const cudaError_t e = cudaMemcpyToSymbol(g_error, &flags, sizeof(flags));
	return e == cudaSuccess ? write_narrow_error(flags) : (int)e;
}

bool operand_aligned(const void* p, uint64_t ld) { return tma_ok(p, ld); }
int run_realign(const Operand* ops, int count, cudaStream_t stream) {
	Realign r{};
	uint64_t units[3] = {}, total = 0;
	for (int k = 0; k < count; ++k) total += units[k] = (uint64_t)ops[k].rows * ((ops[k].cols + 7) / 8);
	for (int k = 0; k < 3; ++k) {
		r.blocks[k + 1] = r.blocks[k];
		if (k >= count) continue;
		r.from[k] = (const uint16_t*)ops[k].from, r.from_ld[k] = ops[k].ld, r.to[k] = (uint16_t*)ops[k].to, r.rows[k] = ops[k].rows, r.cols[k] = ops[k].cols;
		// all blocks run at one time and have alike work
		const uint64_t share = (uint64_t)((double)kRealignBlocks * (double)units[k] / (double)total), need = (units[k] + 255) / 256;
		r.blocks[k + 1] += (uint32_t)std::max<uint64_t>(1, std::min(share, need));
	}
	N2B_CHECK_CUDA(cudaFuncSetAttribute(realign_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRealignSmem));
	return launch_behind(realign_kernel, r.blocks[3], 256, kRealignSmem, stream, r);
}

int run_product(const Product& p, cudaStream_t stream) { return p.b_mn ? product_of<true>(p, stream) : product_of<false>(p, stream); }

uint64_t wgrad_workspace(uint32_t out_width, uint32_t in_width, uint32_t n) {
	// whether the bias gradient is wanted is not known here
	return std::max(plan_bytes(wgrad_plan(out_width, in_width, n, false), out_width, in_width), plan_bytes(wgrad_plan(out_width, in_width, n, true), out_width, in_width));
}

int run_column_sums(const void* a, uint64_t ld, uint32_t rows, uint32_t cols, bool bf16, float* out, int accumulate, cudaStream_t stream) {
	// narrow matrices are shared out over as many SMs by fewer columns a cluster
	const uint32_t each = cols >= 1024 ? 64 : cols >= 512 ? 32 : 16;
	auto kernel = each == 64 ? column_sums_kernel<64> : each == 32 ? column_sums_kernel<32> : column_sums_kernel<16>;
	return launch_behind_in_clusters(8, kernel, 8 * tiles_of(cols, each), 512, 0, stream, (const uint16_t*)a, ld, rows, cols, bf16 ? 1u : 0u, out, accumulate);
}

int run_join(const float* partial, uint32_t splits, uint32_t M, uint32_t N, float* out, float* sums, int accumulate, cudaStream_t stream) {
	const uint64_t n = (uint64_t)M * N;
	const bool vec = n % 4 == 0 && (((uintptr_t)partial | (uintptr_t)out) & 15u) == 0;
	const uint64_t threads = (vec ? n / 4 : n) + (sums ? M : 0);
	// threads for every part where the entries alone do not fill the SMs
	const uint32_t rows = threads >= 512ull * kSMs || splits == 1 ? 1 : splits >= 32 && threads < 64ull * kSMs ? 32 : 8;
	const dim3 block(rows == 1 ? 256 : 32, rows);
	const uint64_t blocks = (threads + block.x - 1) / block.x, most = (uint64_t)kSMs * (rows == 32 ? 2 : 8);
	const uint32_t grid = (uint32_t)(blocks < most ? blocks : most);
	if (vec) return launch_behind(join_kernel<4>, grid, block, rows == 1 ? 0 : block.x * rows * 16, stream, partial, splits, M, N, out, sums, accumulate);
	return launch_behind(join_kernel<1>, grid, block, rows == 1 ? 0 : block.x * rows * 4, stream, partial, splits, M, N, out, sums, accumulate);
}

int run_weight_gradient(const Product& p, cudaStream_t stream) {
	const WgradPlan w = wgrad_plan(p.M, p.N, p.K, p.column_sums != nullptr);
	if (p.workspace_bytes < plan_bytes(w, p.M, p.N)) return NEUS2B_E_INVALID;
	Args a{};
	a.bf16 = p.bf16;
	a.M = p.M, a.N = p.N, a.K = p.K;
	a.a = (const uint16_t*)p.a, a.a_ld = p.a_ld, a.b = (const uint16_t*)p.b, a.b_ld = p.b_ld;
	a.e = p.e;
	a.tiles_m = w.tiles_m, a.tiles_n = w.tiles_n, a.splits = w.splits, a.cluster = w.cluster;
	a.partial = (float*)p.workspace;
	const uint64_t units = (uint64_t)a.tiles_m * a.tiles_n * a.splits;
	if (units >= (1ull << 31)) return NEUS2B_E_TOO_LARGE;
	if (w.pair) {
		// a pair's accumulators fill the tensor memory: the column sums are taken by a pass of their own, ahead of the product, which then
		// finds the matrix in the L2
		if (p.column_sums) {
			if (int rc = run_column_sums(p.a, p.a_ld, p.K, p.M, p.bf16, p.column_sums, p.e.accumulate, stream)) return rc;
		}
		const uint32_t pairs = (uint32_t)(units < (uint64_t)(kSMs / 2) ? units : kSMs / 2);
		if (int rc = launch<256, true, true, false, true, true>(a, 2 * pairs, stream)) return rc;
		return w.splits > 1 ? run_join(a.partial, a.splits, p.M, p.N, (float*)p.e.out, nullptr, p.e.accumulate, stream) : NEUS2B_OK;
	}
	a.column_sums = p.column_sums;
	a.want_sums = p.column_sums != nullptr;
	const uint32_t ctas = (uint32_t)(units < (uint64_t)kSMs ? units : kSMs);
	if (int rc = launch<128, true, true, false, true, false>(a, ctas, stream)) return rc;
	return w.splits > 1 && w.cluster == 1 ? run_join(a.partial, a.splits, p.M, p.N, (float*)p.e.out, p.column_sums, p.e.accumulate, stream) : NEUS2B_OK;
}

}  // namespace n2b
