/*
 * Tokens sorted by expert: the table of a stable counting sort of (token, choice) pairs, and the rows in its order.
 *
 *   row(p) = #{q : e_q < e_p} + #{q < p : e_q = e_p}     over pairs whose expert lies in [0, n_experts)
 *
 * so that the rows of an expert -- and of a rank that holds a run of experts -- are one piece of memory, which one put carries.
 * No order of atomics shows in the result: they only count.
 *
 * Up to 2048 pairs are one launch, up to 8192 two (table, rows), more three (counts of the tiles first), beyond 1,048,576 four (sums of
 * the counts).  32,768 tokens of 8 KiB to 8 of 128 experts: counts 4.9 us, table 8.8, rows 476 for 2.42 GB read and written (5.1 TB/s; the
 * same kernel with the rows written one after the other 441, which is what reading once and writing eight times comes to on this part).
 */
#include "common.hpp"
#include "ofi_amd_hotpath.h"
#include "row_types.hpp"

namespace {

using namespace ofi_amd;

constexpr uint32_t kMaxExperts = 1024;
constexpr uint32_t kMaxTopK = 64;
constexpr uint32_t kMaxRowBytes = 1u << 24;
constexpr uint32_t kTokensOfLaunch = 1u << 21;
constexpr int kSortWaves = 16;
constexpr uint32_t kMostRounds = 8; /* pairs of a lane of the sort */
constexpr uint32_t kManyTiles = 64;
constexpr uint32_t kTilesAtOnce = 32;

/* Beyond so many tiles their counts are summed up first, by one more launch: every tile of the table adding up all of them would be a
 * time by the square of the pairs.  The table alone, us with everybody's own sums and with one: 1,048,576 pairs (128 tiles) of 64 / 256 /
 * 1024 experts 17.9 19.5, 20.7 22.0, 28.6 24.7; twice as many 24.9 23.2, 28.1 26.0, 47.0 35.5; 8,388,608 161 66, 175 78, 355 105;
 * 67,108,864 of 256 and 1024 7,200 568, 17,150 742. */
constexpr uint32_t kTilesSummed = 128;

/* A workgroup of the sort has 1024 pairs a round.  Everybody adds up the counts of all (up to kTilesSummed) tiles, 32 at a time, and
 * each unit's scattered stores of pair_of take their turns: 262,144 pairs as 32 tiles of 8 rounds 11.6 us, 64 of 4 8.8, 128 of 2 9.2, 256 of one 11.9. */
inline uint32_t rounds_of(uint64_t n_pairs)
{
	const uint64_t one = 64 * kSortWaves;
	if (n_pairs <= one * kMostRounds) { /* a single tile */
		return n_pairs <= one ? 1 : n_pairs <= 2 * one ? 2 : n_pairs <= 4 * one ? 4 : 8;
	}
	return n_pairs <= one * kManyTiles ? 1 : n_pairs <= 2 * one * kManyTiles ? 2 : n_pairs <= 4 * one * kManyTiles ? 4 : 8;
}

__device__ __forceinline__ uint32_t lanes_below(uint64_t mask)
{
	return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

/* The expert of pair p, or n_experts where it has none */
template <typename I> __device__ __forceinline__ uint32_t known_expert(I e, uint32_t n_experts)
{
	return e >= 0 && e < (I)n_experts ? (uint32_t)e : n_experts;
}

/* Each count becomes the sum of those of its expert up to its own tile: a workgroup has kSumExperts experts, and shares the tiles of
 * each among kSumParts lanes */
constexpr uint32_t kSumExperts = 16, kSumParts = 64 * kSortWaves / kSumExperts, kSumAtOnce = 16;
static_assert(kMaxExperts <= kSumExperts * kTilesSummed, "as many workgroups as tiles are enough");
__device__ __forceinline__ void sum_counts(uint32_t n_experts, uint32_t n_tiles, uint32_t *counts, uint32_t *s)
{
	const uint32_t x = threadIdx.x % kSumExperts, part = threadIdx.x / kSumExperts, e = blockIdx.x * kSumExperts + x;
	const uint32_t each = (n_tiles + kSumParts - 1) / kSumParts, lo = min(part * each, n_tiles), hi = min(lo + each, n_tiles);
	auto over = [&](auto f) { /* f(tile, its count) */
		for (uint32_t t0 = lo; t0 < hi && e < n_experts; t0 += kSumAtOnce) {
			uint32_t c[kSumAtOnce];
#pragma unroll
			for (uint32_t t = 0; t < kSumAtOnce; t++) {
				c[t] = counts[(uint64_t)min(t0 + t, hi - 1) * n_experts + e];
			}
#pragma unroll
			for (uint32_t t = 0; t < kSumAtOnce; t++) {
				if (t0 + t < hi) {
					f(t0 + t, c[t]);
				}
			}
		}
	};
	uint32_t sum = 0;
	over([&](uint32_t, uint32_t c) { sum += c; });
	s[threadIdx.x] = sum;
	__syncthreads();
	sum = 0;
	for (uint32_t p = 0; p < part; p++) {
		sum += s[p * kSumExperts + x];
	}
	over([&](uint32_t t, uint32_t c) {
		sum += c;
		counts[(uint64_t)t * n_experts + e] = sum;
	});
}

/* counts[tile][e]; a second launch, with n_tiles, has as many workgroups, of which the first sum them up */
template <typename I, uint32_t ROUNDS>
__global__ __launch_bounds__(64 * kSortWaves) void token_count_kernel(const I *__restrict__ expert, uint32_t n_pairs,
								      uint32_t n_experts, uint32_t *__restrict__ counts, uint32_t n_tiles)
{
	__shared__ uint32_t count[kMaxExperts + 1];
	if (n_tiles) {
		if (blockIdx.x * kSumExperts < n_experts) {
			sum_counts(n_experts, n_tiles, counts, count);
		}
		return;
	}
	const uint64_t lo = (uint64_t)blockIdx.x * (64 * kSortWaves * ROUNDS);
	I ids[ROUNDS];
#pragma unroll
	for (uint32_t i = 0; i < ROUNDS; i++) {
		const uint64_t p = lo + i * 64 * kSortWaves + threadIdx.x;
		ids[i] = p < n_pairs ? expert[p] : (I)-1;
	}
	for (uint32_t e = threadIdx.x; e <= n_experts; e += 64 * kSortWaves) {
		count[e] = 0;
	}
	__syncthreads();
#pragma unroll
	for (uint32_t i = 0; i < ROUNDS; i++) {
		const uint32_t e = known_expert(ids[i], n_experts);
		if (e < n_experts) {
			atomicAdd(&count[e], 1u);
		}
	}
	__syncthreads();
	for (uint32_t e = threadIdx.x; e < n_experts; e += 64 * kSortWaves) {
		counts[(uint64_t)blockIdx.x * n_experts + e] = count[e];
	}
}

/*
 * Rows that no pair can have, from n_pairs to max_rows, which a caller's buffers may have many more of than a call has pairs: their -1 in
 * pair_of come from workgroups of their own behind the others, kFillsOfLane of them a lane (beyond kMostFills workgroups more).  8 pairs
 * into 1,048,576 rows 5.4 us a call, 415 with one workgroup for all of them.
 */
constexpr uint32_t kFillsOfLane = 16, kMostFills = 2048;
inline uint32_t fill_blocks(const int32_t *pair_of, uint64_t n_pairs, uint32_t max_rows, uint32_t lanes)
{
	if (!pair_of || max_rows <= n_pairs) {
		return 0;
	}
	const uint64_t blocks = (max_rows - n_pairs + lanes * kFillsOfLane - 1) / (lanes * kFillsOfLane);
	return blocks < kMostFills ? (uint32_t)blocks : kMostFills;
}
__device__ __forceinline__ void fill_rows(int32_t *__restrict__ pair_of, uint32_t n_pairs, uint32_t max_rows, uint32_t block, uint32_t blocks)
{
	for (uint64_t r = (uint64_t)n_pairs + block * blockDim.x + threadIdx.x; r < max_rows; r += (uint64_t)blocks * blockDim.x) {
		pair_of[r] = -1;
	}
}

/*
 * Rows of a tile's pairs: each wavefront ranks its own -- lanes with the same expert find each other by a ballot for each bit of its
 * number, the rounds beside each other --, the counts of the wavefronts and of the other tiles say where they begin.  A tile that is
 * alone needs no counts, one of more than kTilesSummed finds their sums.  LDS: kSortWaves counters an expert, and for the pairs without one.
 */
template <typename I, uint32_t ROUNDS>
__global__ __launch_bounds__(64 * kSortWaves) void token_place_kernel(const I *__restrict__ expert, uint32_t n_pairs,
								      uint32_t n_experts, uint32_t n_tiles, uint32_t max_rows,
								      const uint32_t *__restrict__ counts, int32_t *__restrict__ offset,
								      int32_t *__restrict__ row_of, int32_t *__restrict__ pair_of,
								      uint32_t *__restrict__ err)
{
	extern __shared__ uint32_t next[]; /* [wavefront][expert]: first its pairs so far, then its first row */
	__shared__ uint32_t carry[kSortWaves];
	const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, tile = blockIdx.x, stride = n_experts + 1;
	if (tile >= n_tiles) {
		fill_rows(pair_of, n_pairs, max_rows, tile - n_tiles, gridDim.x - n_tiles);
		return;
	}
	const uint64_t lo = ((uint64_t)tile * kSortWaves + wave) * (64 * ROUNDS); /* its pairs in order: lanes first, then rounds */
	I ids[ROUNDS];
#pragma unroll
	for (uint32_t i = 0; i < ROUNDS; i++) {
		const uint64_t p = lo + i * 64 + lane;
		ids[i] = p < n_pairs ? expert[p] : (I)-1;
	}
	/* one expert a lane: there are at most as many as lanes */
	static_assert(kMaxExperts <= 64 * kSortWaves, "one expert a lane");
	uint32_t total = 0, mine = 0;
	if (n_tiles > kTilesSummed && threadIdx.x < n_experts) {
		mine = tile ? counts[(uint64_t)(tile - 1) * n_experts + threadIdx.x] : 0u;
		total = counts[(uint64_t)(n_tiles - 1) * n_experts + threadIdx.x];
	} else if (n_tiles > 1 && threadIdx.x < n_experts) {
		for (uint32_t t0 = 0; t0 < n_tiles; t0 += kTilesAtOnce) {
			uint32_t c[kTilesAtOnce];
#pragma unroll
			for (uint32_t t = 0; t < kTilesAtOnce; t++) {
				c[t] = counts[(uint64_t)min(t0 + t, n_tiles - 1) * n_experts + threadIdx.x];
			}
#pragma unroll
			for (uint32_t t = 0; t < kTilesAtOnce; t++) {
				mine += t0 + t < tile ? c[t] : 0u;
				total += t0 + t < n_tiles ? c[t] : 0u;
			}
		}
	}
	for (uint32_t i = threadIdx.x; i < kSortWaves * stride; i += 64 * kSortWaves) {
		next[i] = 0;
	}
	__syncthreads();
	const uint32_t bits = 32u - (uint32_t)__builtin_clz(n_experts);
	uint32_t *own = next + wave * stride;
	uint64_t same[ROUNDS]; /* lanes with this lane's expert; the rounds beside each other, as each bit waits for its ballot */
#pragma unroll
	for (uint32_t i = 0; i < ROUNDS; i++) {
		same[i] = ~0ull;
	}
	for (uint32_t b = 0; b < bits; b++) {
#pragma unroll
		for (uint32_t i = 0; i < ROUNDS; i++) {
			const uint32_t one = 0u - ((known_expert(ids[i], n_experts) >> b) & 1u);
			const uint64_t ones = __ballot(one);
			same[i] &= ~(ones ^ ((uint64_t)one << 32 | one));
		}
	}
	uint32_t rank[ROUNDS];
#pragma unroll
	for (uint32_t i = 0; i < ROUNDS; i++) {
		const uint32_t e = known_expert(ids[i], n_experts), before = own[e];
		const uint32_t below = lanes_below(same[i]), of = (uint32_t)__popcll(same[i]);
		rank[i] = before + below;
		__builtin_amdgcn_wave_barrier(); /* every lane has read before the last of an expert's lanes writes */
		if (below == of - 1u) {
			own[e] = before + of;
		}
		__builtin_amdgcn_wave_barrier();
	}
	__syncthreads();
	/* the expert's rows in front of each wavefront's; total: of all tiles */
	uint32_t here = 0;
	if (threadIdx.x < n_experts) {
#pragma unroll
		for (int w = 0; w < kSortWaves; w++) {
			here += next[w * stride + threadIdx.x];
		}
		total = n_tiles > 1 ? total : here;
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
	uint32_t front = 0, all = 0;
#pragma unroll
	for (int w = 0; w < kSortWaves; w++) {
		front += (uint32_t)w < wave ? carry[w] : 0u;
		all += carry[w];
	}
	front += scan - total;
	if (threadIdx.x < n_experts) {
		uint32_t at = front + mine;
#pragma unroll
		for (int w = 0; w < kSortWaves; w++) {
			const uint32_t c = next[w * stride + threadIdx.x];
			next[w * stride + threadIdx.x] = at;
			at += c;
		}
		if (tile == 0) {
			offset[threadIdx.x] = (int32_t)min(front, max_rows);
		}
	}
	if (tile == 0 && threadIdx.x == 0) {
		offset[n_experts] = (int32_t)min(all, max_rows);
		if (all > max_rows) {
			atomicOr(err, ASYNC_ERR_TOKEN_ROWS);
		}
	}
	__syncthreads();
#pragma unroll
	for (uint32_t i = 0; i < ROUNDS; i++) {
		const uint64_t p = lo + i * 64 + lane;
		if (p < n_pairs) {
			const uint32_t e = known_expert(ids[i], n_experts);
			const uint32_t row = e < n_experts ? own[e] + rank[i] : ~0u;
			const bool placed = row < max_rows;
			row_of[p] = placed ? (int32_t)row : -1;
			if (placed && pair_of) {
				pair_of[row] = (int32_t)p;
			}
		}
	}
	if (pair_of) { /* rows behind the last pair's, as far as there are pairs */
		const uint32_t end = min(n_pairs, max_rows);
		for (uint64_t r = all + (uint64_t)tile * 64 * kSortWaves + threadIdx.x; r < end; r += (uint64_t)n_tiles * 64 * kSortWaves) {
			pair_of[r] = -1;
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

constexpr uint32_t kRows = 2; /* of 1 KiB */
constexpr uint32_t kSpan = 1024 * kRows;
constexpr uint32_t kMostWaves = 8;
constexpr uint32_t kAtOnce = 8;

/*
 * A token's rows: 2 KiB are read at a time by a wavefront and written to each of the places (a row number each, max_rows or more:
 * none).  The first row_waves wavefronts have row a, the one behind them row b.  Reading a row once and writing it everywhere beats
 * reading it for each place (560 us and more for 455); ordinary stores beat streaming ones here (455 and 464), as do 2 KiB a wavefront
 * 4 and 8 (466, 475) -- times of this copy alone, 32,768 rows of 8 KiB to 8 places each.
 */
template <typename P>
__device__ __forceinline__ void copy_rows(uint32_t token, uint32_t wave, uint32_t row_waves, const rows_t &a, const rows_t &b,
					  uint32_t top_k, uint32_t max_rows, P place)
{
	const uint32_t lane = threadIdx.x & 63u;
	const bool second = wave >= row_waves;
	const rows_t r = second ? b : a;
	const uint32_t stride = second ? kSpan : row_waves * kSpan;
	for (uint32_t k0 = 0; k0 < top_k; k0 += kAtOnce) {
		uint32_t row[kAtOnce], least = ~0u;
#pragma unroll
		for (uint32_t k = 0; k < kAtOnce; k++) {
			row[k] = k0 + k < top_k ? place(k0 + k) : ~0u;
			least = min(least, row[k]);
		}
		if (least >= max_rows) {
			continue; /* nobody asks for this token */
		}
		for (uint32_t at = second ? 0u : wave * kSpan; at < r.bytes; at += stride) {
			const uint8_t *from = r.from + token * r.from_pitch + at;
			u32x4_t v[kRows];
			if (r.bytes - at >= kSpan) {
#pragma unroll
				for (uint32_t i = 0; i < kRows; i++) {
					v[i] = *reinterpret_cast<const any16_t *>(from + 16u * (i * 64u + lane));
				}
#pragma unroll
				for (uint32_t k = 0; k < kAtOnce; k++) {
					if (row[k] < max_rows) {
						uint8_t *to = r.to + row[k] * r.to_pitch + at;
#pragma unroll
						for (uint32_t i = 0; i < kRows; i++) {
							*reinterpret_cast<any16_t *>(to + 16u * (i * 64u + lane)) = v[i];
						}
					}
				}
				continue;
			}
			const uint32_t n = r.bytes - at, whole = n >> 4, rest = n & 15u;
#pragma unroll
			for (uint32_t i = 0; i < kRows; i++) {
				if (i * 64u + lane < whole) {
					v[i] = *reinterpret_cast<const any16_t *>(from + 16u * (i * 64u + lane));
				}
			}
			uint8_t tail = 0;
			if (lane < rest) {
				tail = from[16u * whole + lane];
			}
#pragma unroll
			for (uint32_t k = 0; k < kAtOnce; k++) {
				if (row[k] < max_rows) {
					uint8_t *to = r.to + row[k] * r.to_pitch + at;
#pragma unroll
					for (uint32_t i = 0; i < kRows; i++) {
						if (i * 64u + lane < whole) {
							*reinterpret_cast<any16_t *>(to + 16u * (i * 64u + lane)) = v[i];
						}
					}
					if (lane < rest) {
						to[16u * whole + lane] = tail;
					}
				}
			}
		}
	}
}

/*
 * Short rows (scales) by their place: a wavefront has rows in order, so that their lines are written whole by one die, where every
 * token's own copy would leave pieces of lines to eight.  The rows read for them lie in the caches.  A row has a power of two of
 * lanes, a wavefront two rounds of kShortAtOnce rows for each of them.  us a call with the tokens' own copies and so: 16,384 x 8 rows of
 * 7168 bytes and 224 247 and 229, of 5120 and 160 (4096 tokens) 48.9 and 46.7, 32,768 x 8 of 256 and 8 42 and 31, 16,384 x 8 of 8192
 * and 256, whose lines are whole anyway, 256 and 260.
 */
constexpr uint32_t kShortBytes = 255, kShortAtOnce = 8;
__host__ __device__ inline uint32_t lanes_of_short(uint32_t bytes)
{
	uint32_t lanes = 1;
	while (lanes * 4 < bytes) {
		lanes *= 2;
	}
	return lanes;
}
__device__ __forceinline__ void gather_rows(uint64_t wave, const int32_t *__restrict__ pair_of, uint32_t top_k, uint32_t max_rows, const rows_t &b)
{
	const uint32_t lane = threadIdx.x & 63u, words = b.bytes >> 2, lanes = lanes_of_short(b.bytes);
	const uint32_t rows = 64u / lanes, word = lane & (lanes - 1u), mine = lane / lanes;
	for (uint32_t round = 0; round < 2; round++) {
		const uint64_t r0 = (wave * 2 + round) * kShortAtOnce * rows + mine;
		uint32_t v[kShortAtOnce];
		int32_t pair[kShortAtOnce];
#pragma unroll
		for (uint32_t i = 0; i < kShortAtOnce; i++) {
			pair[i] = r0 + i * rows < max_rows && word < words ? pair_of[r0 + i * rows] : -1;
		}
#pragma unroll
		for (uint32_t i = 0; i < kShortAtOnce; i++) {
			if (pair[i] >= 0) {
				v[i] = reinterpret_cast<const uint32_t *>(b.from + (uint32_t)pair[i] / top_k * b.from_pitch)[word];
			}
		}
#pragma unroll
		for (uint32_t i = 0; i < kShortAtOnce; i++) {
			if (pair[i] >= 0) {
				reinterpret_cast<uint32_t *>(b.to + (r0 + i * rows) * b.to_pitch)[word] = v[i];
			}
		}
	}
}

/* The first workgroups have the short rows, those behind them blockDim.y tokens each */
__global__ __launch_bounds__(64 * kMostWaves) void token_rows_kernel(const int32_t *__restrict__ row_of,
								     const int32_t *__restrict__ pair_of, uint32_t first, uint32_t n_tokens,
								     uint32_t top_k, uint32_t row_waves, uint32_t max_rows,
								     uint32_t short_blocks, uint32_t short_first, rows_t a, rows_t b)
{
	if (blockIdx.x < short_blocks) {
		const uint32_t waves = (blockDim.x >> 6) * blockDim.y, wave = threadIdx.y * (blockDim.x >> 6) + (threadIdx.x >> 6);
		gather_rows((uint64_t)(short_first + blockIdx.x) * waves + wave, pair_of, top_k, max_rows, b);
		return;
	}
	const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
	const uint32_t token = first + (blockIdx.x - short_blocks) * blockDim.y + (uint32_t)__builtin_amdgcn_readfirstlane((int)threadIdx.y);
	if (token >= n_tokens) {
		return;
	}
	const int32_t *rows = row_of + (uint64_t)token * top_k;
	copy_rows(token, wave, row_waves, a, b, top_k, max_rows, [&](uint32_t k) { return (uint32_t)rows[k]; });
}

/*
 * Few pairs: table and rows in one launch.  The workgroup of a token counts the pairs in front of each of its own -- of a smaller
 * expert, or of the same and a smaller number, which is one comparison of expert * kFew + pair -- and copies its rows there; the
 * workgroup behind them makes the offsets.  8 pairs 4.0 us on the GPU (table and rows apart: 7.2 and 2.2).  Every workgroup looks at all pairs:
 * 2048 of 256 tokens 10.9 us a call, 2056 in two launches 13.4; 2000 of as many tokens 14.0 in one and 13.3 in two, 4096 of 512 15.8
 * and 14.7.
 */
constexpr uint32_t kFew = 2048, kFewTokens = 1024;
constexpr uint32_t kFewWaves = 4; /* at least, to count more than 512, however short the rows are: 4096 by one wavefront 21.8 us for 15.8,
				   * 8 by four 4.4 for 4.0 */
static_assert((uint64_t)kMaxExperts * kFew < 0x7fffffffull, "keys within 32 bits");
template <typename I>
__global__ __launch_bounds__(64 * kMostWaves) void token_few_kernel(const I *__restrict__ expert, uint32_t n_tokens, uint32_t top_k,
								    uint32_t n_experts, uint32_t row_waves, uint32_t max_rows, rows_t a,
								    rows_t b, int32_t *__restrict__ offset, int32_t *__restrict__ row_of,
								    int32_t *__restrict__ pair_of, uint32_t *__restrict__ err)
{
	__shared__ uint32_t counts[kMaxExperts > kMostWaves * kMaxTopK ? kMaxExperts : kMostWaves * kMaxTopK];
	__shared__ uint32_t carry[kMostWaves];
	const uint32_t lane = threadIdx.x & 63u, waves = blockDim.x >> 6, token = blockIdx.x, n_pairs = n_tokens * top_k;
	const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
	if (token > n_tokens) {
		fill_rows(pair_of, n_pairs, max_rows, token - n_tokens - 1, gridDim.x - n_tokens - 1);
		return;
	}
	if (token == n_tokens) { /* behind those of the tokens */
		const uint32_t per = (n_experts + blockDim.x - 1) / blockDim.x, lo = threadIdx.x * per; /* experts of a lane */
		for (uint32_t e = threadIdx.x; e < n_experts; e += blockDim.x) {
			counts[e] = 0;
		}
		__syncthreads();
		for (uint32_t p = threadIdx.x; p < n_pairs; p += blockDim.x) {
			const uint32_t e = known_expert(expert[p], n_experts);
			if (e < n_experts) {
				atomicAdd(&counts[e], 1u);
			}
		}
		__syncthreads();
		uint32_t own = 0;
		for (uint32_t e = lo; e < min(lo + per, n_experts); e++) {
			own += counts[e];
		}
		uint32_t scan = own;
#pragma unroll
		for (uint32_t d = 1; d < 64; d <<= 1) {
			const uint32_t up = __shfl_up(scan, d);
			scan += lane >= d ? up : 0u;
		}
		if (lane == 63) {
			carry[wave] = scan;
		}
		__syncthreads();
		uint32_t at = scan - own, all = 0;
		for (uint32_t w = 0; w < waves; w++) {
			at += w < wave ? carry[w] : 0u;
			all += carry[w];
		}
		for (uint32_t e = lo; e < min(lo + per, n_experts); e++) {
			offset[e] = (int32_t)min(at, max_rows);
			at += counts[e];
		}
		if (threadIdx.x == 0) {
			offset[n_experts] = (int32_t)min(all, max_rows);
			if (all > max_rows) {
				atomicOr(err, ASYNC_ERR_TOKEN_ROWS);
			}
		}
		if (pair_of) {
			for (uint32_t r = all + threadIdx.x; r < min(n_pairs, max_rows); r += blockDim.x) {
				pair_of[r] = -1;
			}
		}
		return;
	}
	const uint32_t p0 = token * top_k;
	for (uint32_t k0 = 0; k0 < top_k; k0 += kAtOnce) {
		uint32_t key[kAtOnce], before[kAtOnce];
#pragma unroll
		for (uint32_t k = 0; k < kAtOnce; k++) {
			const uint32_t p = p0 + min(k0 + k, top_k - 1u);
			key[k] = known_expert(expert[p], n_experts) * kFew + p;
			before[k] = 0;
		}
		for (uint32_t q = threadIdx.x; q - lane < n_pairs; q += blockDim.x) {
			const uint32_t of = q < n_pairs ? known_expert(expert[q], n_experts) * kFew + q : ~0u;
#pragma unroll
			for (uint32_t k = 0; k < kAtOnce; k++) {
				before[k] += (uint32_t)__popcll(__ballot(of < key[k]));
			}
		}
		if (lane == 0) {
#pragma unroll
			for (uint32_t k = 0; k < kAtOnce; k++) {
				if (k0 + k < top_k) {
					counts[wave * top_k + k0 + k] = before[k];
				}
			}
		}
	}
	__syncthreads();
	for (uint32_t k = threadIdx.x; k < top_k; k += blockDim.x) {
		uint32_t row = 0;
		for (uint32_t w = 0; w < waves; w++) {
			row += counts[w * top_k + k];
		}
		const bool placed = row < max_rows && known_expert(expert[p0 + k], n_experts) < n_experts;
		row_of[p0 + k] = placed ? (int32_t)row : -1;
		if (placed && pair_of) {
			pair_of[row] = (int32_t)(p0 + k);
		}
		counts[k] = placed ? row : ~0u; /* the first wavefront's, which this lane has read */
	}
	__syncthreads();
	if (wave < row_waves + (b.to ? 1u : 0u)) {
		copy_rows(token, wave, row_waves, a, b, top_k, max_rows,
			  [&](uint32_t k) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)counts[k]); });
	}
}

inline uint32_t tiles_of(uint64_t n_pairs)
{
	const uint64_t tile = 64ull * kSortWaves * rounds_of(n_pairs);
	return n_pairs == 0 ? 1u : (uint32_t)((n_pairs + tile - 1) / tile);
}

template <typename F> void with_rounds(uint32_t rounds, F f)
{
	if (rounds == 1) {
		f(std::integral_constant<uint32_t, 1>{});
	} else if (rounds == 2) {
		f(std::integral_constant<uint32_t, 2>{});
	} else if (rounds == 4) {
		f(std::integral_constant<uint32_t, 4>{});
	} else {
		f(std::integral_constant<uint32_t, kMostRounds>{});
	}
}

} // namespace

extern "C" {

uint64_t ofi_amd_token_dispatch_work_bytes(uint32_t n_tokens, uint32_t top_k, uint32_t n_experts)
{
	const uint64_t tiles = tiles_of((uint64_t)n_tokens * top_k);
	return tiles == 1 ? 0 : tiles * n_experts * sizeof(uint32_t);
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
	if (n_tokens == 0 || max_rows == 0) { /* nothing to copy, and empty buffers may be NULL */
		d_x = d_scale = nullptr;
		d_rows = d_scale_rows = nullptr;
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
	const rows_t a = { static_cast<const uint8_t *>(d_x), x_pitch, static_cast<uint8_t *>(d_rows), rows_pitch, row_bytes };
	const rows_t b = { static_cast<const uint8_t *>(d_scale), scale_pitch, static_cast<uint8_t *>(d_scale_rows), scale_rows_pitch,
			   scale_bytes };
	const uint32_t spans = d_x ? (row_bytes + kSpan - 1) / kSpan : 0, more = d_scale ? 1 : 0;
	const uint32_t row_waves = d_x ? even_waves(64 * spans, kMostWaves - more) : 0;
	auto run = [&](const auto *expert) {
		using I = typename std::remove_cv<typename std::remove_pointer<decltype(expert)>::type>::type;
		if (d_x && n_pairs <= kFew && n_tokens <= kFewTokens) {
			const uint32_t least = n_pairs > 512 ? kFewWaves : 1, waves = row_waves + more < least ? least : row_waves + more;
			const uint32_t fills = fill_blocks(d_pair_of, n_pairs, max_rows, 64 * waves);
			launch_kernel(token_few_kernel<I>, dim3(n_tokens + 1 + fills), dim3(64 * waves), 0, as_stream(stream), expert, n_tokens, top_k,
				      n_experts, row_waves, max_rows, a, b, d_offset, d_row_of, d_pair_of, err);
			return;
		}
		const uint32_t tiles = tiles_of(n_pairs), fills = fill_blocks(d_pair_of, n_pairs, max_rows, 64 * kSortWaves);
		with_rounds(rounds_of(n_pairs), [&](auto rounds) {
			constexpr uint32_t R = decltype(rounds)::value;
			if (tiles > 1) {
				launch_kernel(token_count_kernel<I, R>, dim3(tiles), dim3(64 * kSortWaves), 0, as_stream(stream), expert,
					      (uint32_t)n_pairs, n_experts, static_cast<uint32_t *>(d_work), 0u);
			}
			if (tiles > kTilesSummed) {
				launch_kernel(token_count_kernel<I, R>, dim3(tiles), dim3(64 * kSortWaves), 0, as_stream(stream), expert,
					      (uint32_t)n_pairs, n_experts, static_cast<uint32_t *>(d_work), tiles);
			}
			launch_kernel(token_place_kernel<I, R>, dim3(tiles + fills), dim3(64 * kSortWaves),
				      kSortWaves * (n_experts + 1) * sizeof(uint32_t), as_stream(stream), expert, (uint32_t)n_pairs, n_experts, tiles,
				      max_rows, static_cast<const uint32_t *>(d_work), d_offset, d_row_of, d_pair_of, err);
		});
		if (!d_x) {
			return; /* the table alone */
		}
		/* the scales by their place where the table says which pair is there */
		const bool apart = more && d_pair_of && scale_bytes <= kShortBytes &&
				   ((reinterpret_cast<uintptr_t>(d_scale) | reinterpret_cast<uintptr_t>(d_scale_rows) | scale_pitch | scale_rows_pitch |
				     scale_bytes) & 3u) == 0;
		const uint32_t waves = row_waves + (apart ? 0 : more), tokens = waves <= 2 ? 4 / waves : 1;
		/* workgroups of the short rows, as many with each launch as it has of the tokens */
		const uint32_t each = waves * tokens * 2 * kShortAtOnce * (apart ? 64 / lanes_of_short(scale_bytes) : 1);
		const uint32_t most = n_pairs < max_rows ? (uint32_t)n_pairs : max_rows, all_short = apart ? (most + each - 1) / each : 0;
		const uint32_t launches = (n_tokens + kTokensOfLaunch - 1) / kTokensOfLaunch;
		uint32_t short_first = 0;
		for (uint32_t first = 0; first < n_tokens; first += kTokensOfLaunch) {
			const uint32_t n = n_tokens - first < kTokensOfLaunch ? n_tokens - first : kTokensOfLaunch;
			const uint32_t part = (all_short + launches - 1) / launches, left = all_short - short_first;
			const uint32_t short_blocks = left < part ? left : part;
			launch_kernel(token_rows_kernel, dim3(short_blocks + (n + tokens - 1) / tokens), dim3(64 * waves, tokens), 0, as_stream(stream),
				      d_row_of, d_pair_of, first, first + n, top_k, row_waves, max_rows, short_blocks, short_first, a, b);
			short_first += short_blocks;
		}
	};
	if (expert_type == OFI_AMD_INT64) {
		run(static_cast<const int64_t *>(d_expert));
	} else {
		run(static_cast<const int32_t *>(d_expert));
	}
	OFI_AMD_HIP_TRY(hipGetLastError());
	return 0;
}

} /* extern "C" */
