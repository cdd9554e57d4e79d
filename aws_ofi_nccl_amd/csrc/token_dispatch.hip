/*
 * Tokens sorted by expert: the table of a stable counting sort of (token, choice) pairs, and the rows in its order.
 *
 *   row(p) = #{q : e_q < e_p} + #{q < p : e_q = e_p}     over pairs whose expert lies in [0, n_experts)
 *
 * so that the rows of an expert -- and of a rank that holds a run of experts -- are one piece of memory, which one put carries.
 * No order of atomics shows in the result.
 */
#include "common.hpp"
#include "ofi_amd_hotpath.h"
#include "row_types.hpp"

namespace {

using namespace ofi_amd;

constexpr uint32_t kMaxExperts = 1024;
constexpr uint32_t kMaxTopK = 64;
constexpr uint32_t kMaxRowBytes = 1u << 24;
constexpr uint32_t kTokensOfLaunch = 1u << 22;
constexpr int kSortWaves = 4;
constexpr uint32_t kTile = 2048; /* pairs of a workgroup of the sort */
constexpr uint32_t kTileOfWave = kTile / kSortWaves;

__device__ __forceinline__ uint32_t lanes_below(uint64_t mask)
{
	return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

/* The expert of pair p, or n_experts where it has none */
template <typename I> __device__ __forceinline__ uint32_t expert_at(const I *__restrict__ expert, uint32_t p, uint32_t n_experts)
{
	const I e = expert[p];
	return e >= 0 && e < (I)n_experts ? (uint32_t)e : n_experts;
}

/* counts[tile][e] */
template <typename I>
__global__ __launch_bounds__(64 * kSortWaves) void token_count_kernel(const I *__restrict__ expert, uint32_t n_pairs,
								      uint32_t n_experts, uint32_t *__restrict__ counts)
{
	__shared__ uint32_t count[kMaxExperts + 1];
	for (uint32_t e = threadIdx.x; e <= n_experts; e += 64 * kSortWaves) {
		count[e] = 0;
	}
	__syncthreads();
	const uint32_t lo = blockIdx.x * kTile;
	const uint32_t hi = min(n_pairs - lo, kTile);
	for (uint32_t i = threadIdx.x; i < hi; i += 64 * kSortWaves) {
		atomicAdd(&count[expert_at(expert, lo + i, n_experts)], 1u);
	}
	__syncthreads();
	for (uint32_t e = threadIdx.x; e < n_experts; e += 64 * kSortWaves) {
		counts[(uint64_t)blockIdx.x * n_experts + e] = count[e];
	}
}

/* Rows of a tile's pairs.  Every workgroup adds up the tiles' counts by itself. */
template <typename I>
__global__ __launch_bounds__(64 * kSortWaves) void token_place_kernel(const I *__restrict__ expert, uint32_t n_pairs,
								      uint32_t n_experts, uint32_t n_tiles, uint32_t max_rows,
								      const uint32_t *__restrict__ counts, int32_t *__restrict__ offset,
								      int32_t *__restrict__ row_of, int32_t *__restrict__ pair_of,
								      uint32_t *__restrict__ err)
{
	__shared__ uint32_t base[kMaxExperts + 1];              /* first row of the tile's pairs of an expert */
	__shared__ uint32_t next[kSortWaves][kMaxExperts + 1];  /* next row of a wavefront's pairs of an expert */
	__shared__ uint32_t carry[kSortWaves];
	const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, tile = blockIdx.x;
	uint32_t before = 0; /* rows of all experts in front of this round's */
	for (uint32_t e0 = 0; e0 < n_experts; e0 += 64 * kSortWaves) {
		const uint32_t e = e0 + threadIdx.x;
		uint32_t total = 0, mine = 0;
		if (e < n_experts) {
			for (uint32_t t = 0; t < n_tiles; t++) {
				const uint32_t c = counts[(uint64_t)t * n_experts + e];
				mine = t == tile ? total : mine;
				total += c;
			}
		}
		uint32_t scan = total; /* inclusive over the wavefront */
#pragma unroll
		for (uint32_t d = 1; d < 64; d <<= 1) {
			const uint32_t up = __shfl_up(scan, d);
			scan += lane >= d ? up : 0u;
		}
		if (lane == 63) {
			carry[wave] = scan;
		}
		__syncthreads();
		uint32_t front = before;
#pragma unroll
		for (int w = 0; w < kSortWaves; w++) {
			front += (uint32_t)w < wave ? carry[w] : 0u;
			before += carry[w];
		}
		if (e < n_experts) {
			base[e] = front + scan - total + mine;
			if (tile == 0) {
				offset[e] = (int32_t)min(front + scan - total, max_rows);
			}
		}
		__syncthreads();
	}
	if (tile == 0 && threadIdx.x == 0) {
		offset[n_experts] = (int32_t)min(before, max_rows);
		if (before > max_rows) {
			atomicOr(err, ASYNC_ERR_TOKEN_ROWS);
		}
	}
	if (pair_of) { /* rows behind the last pair's */
		for (uint64_t r = before + (uint64_t)tile * 64 * kSortWaves + threadIdx.x; r < max_rows; r += (uint64_t)gridDim.x * 64 * kSortWaves) {
			pair_of[r] = -1;
		}
	}
	/* what the wavefronts in front of this one place */
	for (uint32_t e = threadIdx.x; e <= n_experts; e += 64 * kSortWaves) {
#pragma unroll
		for (int w = 0; w < kSortWaves; w++) {
			next[w][e] = 0;
		}
	}
	__syncthreads();
	const uint32_t lo = tile * kTile + wave * kTileOfWave;
	const uint32_t mine = lo < n_pairs ? min(n_pairs - lo, kTileOfWave) : 0u;
	for (uint32_t i = lane; i < mine; i += 64) {
		atomicAdd(&next[wave][expert_at(expert, lo + i, n_experts)], 1u);
	}
	__syncthreads();
	for (uint32_t e = threadIdx.x; e < n_experts; e += 64 * kSortWaves) {
		uint32_t at = base[e];
#pragma unroll
		for (int w = 0; w < kSortWaves; w++) {
			const uint32_t c = next[w][e];
			next[w][e] = at;
			at += c;
		}
	}
	__syncthreads();
	const uint32_t bits = 32u - (uint32_t)__builtin_clz(n_experts);
	for (uint32_t i0 = 0; i0 < mine; i0 += 64) {
		const uint32_t p = lo + i0 + lane;
		const bool in = i0 + lane < mine;
		const uint32_t e = in ? expert_at(expert, p, n_experts) : n_experts;
		uint64_t same = ~0ull; /* lanes with this lane's expert */
		for (uint32_t b = 0; b < bits; b++) {
			const bool one = (e >> b) & 1u;
			const uint64_t ones = __ballot(one);
			same &= one ? ones : ~ones;
		}
		const uint32_t rank = lanes_below(same), of = (uint32_t)__popcll(same);
		const uint32_t first = next[wave][e];
		__builtin_amdgcn_wave_barrier(); /* every lane has read before the last of an expert's lanes writes */
		if (e < n_experts && rank == of - 1u) {
			next[wave][e] = first + of;
		}
		__builtin_amdgcn_wave_barrier();
		if (in) {
			const uint32_t row = first + rank;
			const bool placed = e < n_experts && row < max_rows;
			row_of[p] = placed ? (int32_t)row : -1;
			if (placed && pair_of) {
				pair_of[row] = (int32_t)p;
			}
		}
	}
}

struct rows_t { /* rows of bytes and where they go */
	const uint8_t *from;
	uint64_t from_pitch;
	uint8_t *to;
	uint64_t to_pitch;
	uint32_t bytes;
};

/* One wavefront per 4 KiB of a token's row: it is read once and written to each of its places */
constexpr uint32_t kSpan = 4096;
__global__ __launch_bounds__(64) void token_rows_kernel(const int32_t *__restrict__ row_of, uint32_t first, uint32_t top_k, uint32_t spans,
						        rows_t a, rows_t b)
{
	const uint32_t lane = threadIdx.x;
	const uint32_t token = first + blockIdx.x;
	const bool second = blockIdx.y >= spans;
	const rows_t r = second ? b : a;
	const uint32_t at = (blockIdx.y - (second ? spans : 0u)) * kSpan;
	const uint32_t n = min(r.bytes - at, kSpan);
	const uint8_t *from = r.from + token * r.from_pitch + at;
	const int32_t *rows = row_of + (uint64_t)token * top_k;
	u32x4_t v[4];
	const uint32_t whole = n >> 4;
#pragma unroll
	for (uint32_t i = 0; i < 4; i++) {
		if (i * 64u + lane < whole) {
			v[i] = reinterpret_cast<const any16_t *>(from + 16u * (i * 64u + lane))->v;
		}
	}
	const uint32_t rest = n & 15u;
	uint8_t tail = 0;
	if (lane < rest) {
		tail = from[16u * whole + lane];
	}
	for (uint32_t k = 0; k < top_k; k++) {
		const int32_t row = rows[k];
		if (row < 0) {
			continue;
		}
		uint8_t *to = r.to + (uint64_t)row * r.to_pitch + at;
#pragma unroll
		for (uint32_t i = 0; i < 4; i++) {
			if (i * 64u + lane < whole) {
				reinterpret_cast<any16_t *>(to + 16u * (i * 64u + lane))->v = v[i];
			}
		}
		if (lane < rest) {
			to[16u * whole + lane] = tail;
		}
	}
}

inline uint32_t tiles_of(uint64_t n_pairs)
{
	return n_pairs == 0 ? 1u : (uint32_t)((n_pairs + kTile - 1) / kTile);
}

} // namespace

extern "C" {

uint64_t ofi_amd_token_dispatch_work_bytes(uint32_t n_tokens, uint32_t top_k, uint32_t n_experts)
{
	return (uint64_t)tiles_of((uint64_t)n_tokens * top_k) * n_experts * sizeof(uint32_t);
}

int ofi_amd_token_dispatch(const void *d_expert, int expert_type, uint32_t n_tokens, uint32_t top_k, uint32_t n_experts,
			   uint32_t max_rows, int32_t *d_offset, int32_t *d_row_of, int32_t *d_pair_of, const void *d_x, uint64_t x_pitch,
			   void *d_rows, uint64_t rows_pitch, uint32_t row_bytes, const void *d_scale, uint64_t scale_pitch,
			   void *d_scale_rows, uint64_t scale_rows_pitch, uint32_t scale_bytes, void *d_work, uint64_t work_bytes,
			   void *stream)
{
	int rc = require_device();
	if (rc != 0) {
		return rc;
	}
	if ((expert_type != OFI_AMD_INT32 && expert_type != OFI_AMD_INT64) || top_k == 0 || n_experts == 0 || !d_offset ||
	    (reinterpret_cast<uintptr_t>(d_offset) & 3u) || (reinterpret_cast<uintptr_t>(d_pair_of) & 3u) || (!d_x != !d_rows) ||
	    (!d_scale != !d_scale_rows) || (d_scale && !d_x)) {
		return -EINVAL;
	}
	const uint64_t n_pairs = (uint64_t)n_tokens * top_k;
	if (n_experts > kMaxExperts || top_k > kMaxTopK || n_pairs > 0x7fffffffull || max_rows > 0x7fffffffu ||
	    (d_x && row_bytes > kMaxRowBytes) || (d_scale && scale_bytes > kMaxRowBytes)) {
		return -E2BIG;
	}
	const uintptr_t index = expert_type == OFI_AMD_INT64 ? 7u : 3u;
	if (n_pairs != 0 && (!d_expert || (reinterpret_cast<uintptr_t>(d_expert) & index) || !d_row_of ||
			     (reinterpret_cast<uintptr_t>(d_row_of) & 3u))) {
		return -EINVAL;
	}
	if ((d_x && (row_bytes == 0 || !rows_ok(d_x, x_pitch, n_tokens, row_bytes, 1) || !rows_ok(d_rows, rows_pitch, max_rows, row_bytes, 1))) ||
	    (d_scale && (scale_bytes == 0 || !rows_ok(d_scale, scale_pitch, n_tokens, scale_bytes, 1) ||
			 !rows_ok(d_scale_rows, scale_rows_pitch, max_rows, scale_bytes, 1)))) {
		return -EINVAL;
	}
	const uint64_t need = ofi_amd_token_dispatch_work_bytes(n_tokens, top_k, n_experts);
	if (need && (!d_work || (reinterpret_cast<uintptr_t>(d_work) & 3u) || work_bytes < need)) {
		return -EINVAL;
	}
	uint32_t *err = async_error_word();
	if (!err) {
		return -ENOMEM;
	}
	const uint32_t tiles = tiles_of(n_pairs);
	auto sort = [&](const auto *expert) {
		using I = typename std::remove_cv<typename std::remove_pointer<decltype(expert)>::type>::type;
		launch_kernel(token_count_kernel<I>, dim3(tiles), dim3(64 * kSortWaves), 0, as_stream(stream), expert, (uint32_t)n_pairs,
			      n_experts, static_cast<uint32_t *>(d_work));
		launch_kernel(token_place_kernel<I>, dim3(tiles), dim3(64 * kSortWaves), 0, as_stream(stream), expert, (uint32_t)n_pairs,
			      n_experts, tiles, max_rows, static_cast<const uint32_t *>(d_work), d_offset, d_row_of, d_pair_of, err);
	};
	if (expert_type == OFI_AMD_INT64) {
		sort(static_cast<const int64_t *>(d_expert));
	} else {
		sort(static_cast<const int32_t *>(d_expert));
	}
	if (d_x && n_tokens != 0) {
		const rows_t a = { static_cast<const uint8_t *>(d_x), x_pitch, static_cast<uint8_t *>(d_rows), rows_pitch, row_bytes };
		const rows_t b = { static_cast<const uint8_t *>(d_scale), scale_pitch, static_cast<uint8_t *>(d_scale_rows), scale_rows_pitch,
				   scale_bytes };
		const uint32_t spans = (row_bytes + kSpan - 1) / kSpan, more = d_scale ? (scale_bytes + kSpan - 1) / kSpan : 0;
		for (uint32_t first = 0; first < n_tokens; first += kTokensOfLaunch) {
			launch_kernel(token_rows_kernel, dim3(n_tokens - first < kTokensOfLaunch ? n_tokens - first : kTokensOfLaunch, spans + more),
				      dim3(64), 0, as_stream(stream), d_row_of, first, top_k, spans, a, b);
		}
	}
	OFI_AMD_HIP_TRY(hipGetLastError());
	return 0;
}

} /* extern "C" */
