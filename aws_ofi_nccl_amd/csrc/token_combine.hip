/*
 * Tokens back from their experts: the weighted sum of a token's rows, and its gradient.
 *
 *   out_t = add_t + sum_k w_tk y[row_tk]        dy[row_tk] = w_tk dout_t        dw_tk = <dout_t, y[row_tk]>
 *
 * A pair without a row (an index outside the rows) is passed over, whatever its weight is.
 *
 * Memory bounds both: 16,384 tokens of 8 rows of 8 KiB, sums and an addend 1.34 GB in 235 us = 5.7 TB/s, gradients 2.28 GB in 439 us =
 * 5.2 TB/s (nine streams read and eight written; the same reads and writes without the arithmetic 445).  Counters: every byte once.
 */
#include "common.hpp"
#include "ofi_amd_hotpath.h"
#include "row_types.hpp"

namespace {

using namespace ofi_amd;

constexpr uint32_t kMaxTopK = 64;
constexpr uint32_t kMaxWidth = 1u << 20;
constexpr uint32_t kMostWaves = 8; /* a workgroup has all of a row of up to 8 KiB in flight at once */
constexpr int kAtOnce = 8; /* rows of a token that are read together */

/* A workgroup of threadIdx.x lanes along a row and threadIdx.y tokens.  A lane asks for ROWS rows' chunks before it uses the first, of
 * one chunk of the output at a time, or of four where a token has at most two rows, so that enough is in flight there too.
 * Eight wavefronts a row are faster than four with two chunks a lane or one with all of them for eight rows (237, 239, 245 us of reads
 * and writes alone), a token's rows are not brought closer by giving each die a run of tokens (246).  Four chunks against one, 10,636
 * tokens of 4,224 floats on no more than 4 bytes: one row 61 for 93 us, two rows 91 for 104; of 4,096 bf16 and an addend, 16,384
 * tokens: 66 for 69 and 88 for 89, but 3,000 tokens of two rows 18.9 for 18.4. */
template <typename T, uint32_t V, int ROWS, flow_t FLOW>
__global__ __launch_bounds__(64 * kMostWaves) void token_combine_kernel(const int32_t *__restrict__ row_of,
									const float *__restrict__ weight, const T *__restrict__ rows,
									const T *add, T *out, uint64_t rows_pitch, uint64_t add_pitch,
									uint64_t out_pitch, uint32_t n_tokens, uint32_t max_rows,
									uint32_t top_k, uint32_t width)
{
	constexpr int U = ROWS <= 2 ? 4 : 1; /* chunks of a lane */
	const uint32_t token = blockIdx.x * blockDim.y + (uint32_t)__builtin_amdgcn_readfirstlane((int)threadIdx.y);
	if (token >= n_tokens) {
		return;
	}
	row_of += (uint64_t)token * top_k;
	weight += weight ? (uint64_t)token * top_k : 0;
	const uint32_t step = blockDim.x * V;
	for (uint32_t at = threadIdx.x * V; at < width; at += U * step) {
		place_t here[U];
		raw_t<T, V> first[U];
#pragma unroll
		for (int u = 0; u < U; u++) {
			here[u] = place_of<V>(at + u * step, width);
			if (add) {
				first[u] = load_raw<FLOW != STREAM_NONE, T, V>(row_at(add, add_pitch, token) + here[u].from);
			}
		}
		float sum[U][V];
		for (uint32_t k0 = 0; k0 < top_k; k0 += ROWS) {
			raw_t<T, V> c[ROWS][U];
			uint32_t row[ROWS];
			float w[ROWS];
#pragma unroll
			for (uint32_t k = 0; k < ROWS; k++) {
				const uint32_t at_k = min(k0 + k, top_k - 1u);
				row[k] = k0 + k < top_k ? (uint32_t)row_of[at_k] : ~0u;
				w[k] = weight ? weight[at_k] : 1.0f;
			}
#pragma unroll
			for (uint32_t k = 0; k < ROWS; k++) {
				if (row[k] < max_rows) {
#pragma unroll
					for (int u = 0; u < U; u++) {
						c[k][u] = load_raw<FLOW != STREAM_NONE, T, V>(row_at(rows, rows_pitch, row[k]) + here[u].from);
					}
				}
			}
			if (k0 == 0) {
#pragma unroll
				for (int u = 0; u < U; u++) {
#pragma unroll
					for (uint32_t i = 0; i < V; i++) {
						sum[u][i] = add ? (float)first[u][i] : 0.0f;
					}
				}
			}
#pragma unroll
			for (uint32_t k = 0; k < ROWS; k++) {
				if (row[k] < max_rows) {
#pragma unroll
					for (int u = 0; u < U; u++) {
#pragma unroll
						for (uint32_t i = 0; i < V; i++) {
							sum[u][i] = __builtin_fmaf(w[k], (float)c[k][u][i], sum[u][i]);
						}
					}
				}
			}
		}
#pragma unroll
		for (int u = 0; u < U; u++) {
			if (at + u * step < width) {
				store_piece<FLOW == STREAM_BOTH, T, V>(row_at(out, out_pitch, token) + here[u].from, here[u].skip, sum[u]);
			}
		}
	}
}

/* One workgroup of `waves` wavefronts per token.  All rows that are read together are asked for before the first is written, so
 * that drows may be rows.  Registers for six wavefronts a SIMD: left to itself the compiler takes 98 for floats, which leaves room for
 * two workgroups of six wavefronts where four fit (8,000 x 8 rows of 4,224 floats 587 us, with six 462; of 8,107 492 and 479; rows of
 * 2,048, eight wavefronts once, 445 and 450).  Tokens of one row have a kernel for one row: 16,384 of 4,096 bf16 72 us for 85, 10,636
 * of 4,224 floats 100 for 108; two and four rows at once gain nothing (126 for 123, 232 for 232). */
template <typename T, uint32_t V, int ROWS, flow_t FLOW>
__global__ __launch_bounds__(64 * kMostWaves, 6) void token_combine_grad_kernel(const int32_t *__restrict__ row_of,
									     const float *__restrict__ weight,
									     const T *__restrict__ dout, const T *rows, T *drows,
									     float *__restrict__ dweight, uint64_t dout_pitch,
									     uint64_t rows_pitch, uint64_t drows_pitch, uint32_t max_rows,
									     uint32_t top_k, uint32_t width)
{
	__shared__ float part[kMostWaves][kAtOnce];
	const uint64_t token = blockIdx.x;
	const uint32_t waves = blockDim.x >> 6;
	const T *dr = row_at(dout, dout_pitch, token);
	row_of += token * top_k;
	weight += weight ? token * top_k : 0;
	for (uint32_t k0 = 0; k0 < top_k; k0 += ROWS) {
		float dot[kAtOnce] = {}, w[ROWS];
		uint32_t row[ROWS];
#pragma unroll
		for (uint32_t k = 0; k < ROWS; k++) {
			const uint32_t at_k = min(k0 + k, top_k - 1u);
			row[k] = k0 + k < top_k ? (uint32_t)row_of[at_k] : ~0u;
			w[k] = weight ? weight[at_k] : 1.0f;
		}
		for (uint32_t at = threadIdx.x * V; at < width; at += blockDim.x * V) {
			const place_t here = place_of<V>(at, width);
			const raw_t<T, V> dc = load_raw<FLOW != STREAM_NONE, T, V>(dr + here.from);
			raw_t<T, V> c[ROWS];
			if (dweight) {
#pragma unroll
				for (uint32_t k = 0; k < ROWS; k++) {
					if (row[k] < max_rows) {
						c[k] = load_raw<FLOW != STREAM_NONE, T, V>(row_at(rows, rows_pitch, row[k]) + here.from);
					}
				}
			}
			float d[V];
			to_floats<T, V>(dc, 0, d);
			if (drows) {
#pragma unroll
				for (uint32_t k = 0; k < ROWS; k++) {
					if (row[k] < max_rows) {
						float f[V];
#pragma unroll
						for (uint32_t i = 0; i < V; i++) {
							f[i] = w[k] * d[i];
						}
						store_piece<FLOW == STREAM_BOTH, T, V>(row_at(drows, drows_pitch, row[k]) + here.from, here.skip, f);
					}
				}
			}
			if (dweight) {
				if (here.skip) {
#pragma unroll
					for (uint32_t i = 0; i < V; i++) {
						d[i] = i < here.skip ? 0.0f : d[i];
					}
				}
#pragma unroll
				for (uint32_t k = 0; k < ROWS; k++) {
					if (row[k] < max_rows) {
						float f[V];
						to_floats<T, V>(c[k], here.skip, f);
#pragma unroll
						for (uint32_t i = 0; i < V; i++) {
							dot[k] = __builtin_fmaf(d[i], f[i], dot[k]);
						}
					}
				}
			}
		}
		if (!dweight) {
			continue;
		}
		const uint32_t lane = threadIdx.x & 63u;
		const float sum = eight_sums(dot, lane);
		if ((lane & 7u) == 0) {
			part[threadIdx.x >> 6][lane >> 3] = sum;
		}
		__syncthreads();
		if (threadIdx.x < ROWS && k0 + threadIdx.x < top_k) {
			float d = part[0][threadIdx.x];
			for (uint32_t v = 1; v < waves; v++) {
				d += part[v][threadIdx.x];
			}
			dweight[token * top_k + k0 + threadIdx.x] = d;
		}
		__syncthreads();
	}
}

constexpr uint32_t kTokensOfLaunch = 1u << 22; /* with 512 lanes each within the 32 bits of a launch's size */

int check_call(uint32_t max_rows, const int32_t *d_row_of, const float *d_weight, uint32_t top_k, uint32_t width, uint32_t size,
	       uint32_t n_tokens)
{
	if (!size || top_k == 0 || width == 0) {
		return -EINVAL;
	}
	if (top_k > kMaxTopK || width > kMaxWidth || max_rows > 0x7fffffffu || (uint64_t)n_tokens * top_k > 0x7fffffffull) {
		return -E2BIG;
	}
	if (n_tokens != 0 && (!d_row_of || (reinterpret_cast<uintptr_t>(d_row_of) & 3u) || (reinterpret_cast<uintptr_t>(d_weight) & 3u))) {
		return -EINVAL;
	}
	return 0;
}

} // namespace

extern "C" {

int ofi_amd_token_combine(const void *d_rows, uint64_t rows_pitch, uint32_t max_rows, const int32_t *d_row_of, const float *d_weight,
			  uint32_t n_tokens, uint32_t top_k, uint32_t width, int type, const void *d_add, uint64_t add_pitch, void *d_out,
			  uint64_t out_pitch, void *stream)
{
	int rc = require_device();
	if (rc != 0) {
		return rc;
	}
	const uint32_t size = row_type_size(type);
	rc = check_call(max_rows, d_row_of, d_weight, top_k, width, size, n_tokens);
	if (rc != 0 || n_tokens == 0) {
		return rc;
	}
	const uint64_t bytes = (uint64_t)width * size;
	if ((max_rows != 0 && !rows_ok(d_rows, rows_pitch, max_rows, bytes, size)) ||
	    (d_add && !rows_ok(d_add, add_pitch, n_tokens, bytes, size)) || !rows_ok(d_out, out_pitch, n_tokens, bytes, size)) {
		return -EINVAL;
	}
	const uint64_t pairs = (uint64_t)n_tokens * top_k, named = pairs < max_rows ? pairs : max_rows;
	const flow_t flow = flow_of((named + n_tokens * (1ull + !!d_add)) * bytes);
	with_row_type(type, width, [&](auto element, auto v) {
		using T = decltype(element);
		constexpr uint32_t V = decltype(v)::value;
		const bool few = V > 1 && top_k <= 2; /* four chunks of a lane, token_combine_kernel */
		const uint32_t chunks = (width + V - 1) / V, waves = even_waves(few ? (chunks + 3) / 4 : chunks, kMostWaves);
		const uint32_t tokens = waves < 4 ? 4 / waves : 1;
		auto kernel = by_flow(flow, token_combine_kernel<T, V, kAtOnce, STREAM_NONE>, token_combine_kernel<T, V, kAtOnce, STREAM_LOADS>,
				      token_combine_kernel<T, V, kAtOnce, STREAM_BOTH>);
		if constexpr (V > 1) {
			if (top_k == 1) {
				kernel = by_flow(flow, token_combine_kernel<T, V, 1, STREAM_NONE>, token_combine_kernel<T, V, 1, STREAM_LOADS>,
						 token_combine_kernel<T, V, 1, STREAM_BOTH>);
			} else if (few) {
				kernel = by_flow(flow, token_combine_kernel<T, V, 2, STREAM_NONE>, token_combine_kernel<T, V, 2, STREAM_LOADS>,
						 token_combine_kernel<T, V, 2, STREAM_BOTH>);
			}
		}
		for (uint32_t at = 0; at < n_tokens; at += kTokensOfLaunch) {
			const uint32_t n = n_tokens - at < kTokensOfLaunch ? n_tokens - at : kTokensOfLaunch;
			launch_kernel(kernel,
				      dim3((n + tokens - 1) / tokens), dim3(64 * waves, tokens), 0, as_stream(stream),
				      d_row_of + (uint64_t)at * top_k, d_weight ? d_weight + (uint64_t)at * top_k : nullptr,
				      static_cast<const T *>(d_rows), d_add ? row_at(static_cast<const T *>(d_add), add_pitch, at) : nullptr,
				      row_at(static_cast<T *>(d_out), out_pitch, at), rows_pitch, add_pitch, out_pitch, n, max_rows, top_k, width);
		}
	});
	OFI_AMD_HIP_TRY(hipGetLastError());
	return 0;
}

int ofi_amd_token_combine_grad(const void *d_dout, uint64_t dout_pitch, const void *d_rows, uint64_t rows_pitch, uint32_t max_rows,
			       const int32_t *d_row_of, const float *d_weight, uint32_t n_tokens, uint32_t top_k, uint32_t width, int type,
			       void *d_drows, uint64_t drows_pitch, float *d_dweight, void *stream)
{
	int rc = require_device();
	if (rc != 0) {
		return rc;
	}
	const uint32_t size = row_type_size(type);
	rc = check_call(max_rows, d_row_of, d_weight, top_k, width, size, n_tokens);
	if (rc != 0 || n_tokens == 0) {
		return rc;
	}
	const uint64_t bytes = (uint64_t)width * size;
	if (!rows_ok(d_dout, dout_pitch, n_tokens, bytes, size) || (max_rows != 0 && !d_drows && !d_dweight) ||
	    (reinterpret_cast<uintptr_t>(d_dweight) & 3u) ||
	    (max_rows != 0 && ((d_dweight && !rows_ok(d_rows, rows_pitch, max_rows, bytes, size)) ||
			       (d_drows && !rows_ok(d_drows, drows_pitch, max_rows, bytes, size))))) {
		return -EINVAL;
	}
	if (!d_drows && !d_dweight) { /* gradients of no rows, whose buffer may be NULL */
		return 0;
	}
	const uint64_t pairs = (uint64_t)n_tokens * top_k, named = pairs < max_rows ? pairs : max_rows;
	/* As many rows are written as read, and their ends share lines with other rows.  Where the rows do not start on 64 bytes and do not
	 * stay in the caches, streaming costs more than it gives: 2280 MB, us with neither, streaming loads, both: rows of 8190 bytes
	 * 485 522 525, of 8176 465 491 484, of 8128 457 472 452 (285 MB of 8190 66.8 67.7 -, 143 MB 36.6 31.5 -) */
	const uint64_t moved = (named * (!!d_dweight + !!d_drows) + n_tokens) * bytes;
	const bool aligned = ((reinterpret_cast<uintptr_t>(d_drows) | drows_pitch) & 63u) == 0;
	const flow_t flow = flow_of(moved) == STREAM_BOTH && !aligned ? STREAM_NONE : flow_of(moved);
	with_row_type(type, width, [&](auto element, auto v) {
		using T = decltype(element);
		constexpr uint32_t V = decltype(v)::value;
		const uint32_t waves = even_waves((width + V - 1) / V, kMostWaves);
		auto kernel = by_flow(flow, token_combine_grad_kernel<T, V, kAtOnce, STREAM_NONE>,
				      token_combine_grad_kernel<T, V, kAtOnce, STREAM_LOADS>,
				      token_combine_grad_kernel<T, V, kAtOnce, STREAM_BOTH>);
		if constexpr (V > 1) {
			if (top_k == 1) {
				kernel = by_flow(flow, token_combine_grad_kernel<T, V, 1, STREAM_NONE>, token_combine_grad_kernel<T, V, 1, STREAM_LOADS>,
						 token_combine_grad_kernel<T, V, 1, STREAM_BOTH>);
			}
		}
		for (uint32_t at = 0; at < n_tokens; at += kTokensOfLaunch) {
			launch_kernel(kernel,
				      dim3(n_tokens - at < kTokensOfLaunch ? n_tokens - at : kTokensOfLaunch), dim3(64 * waves), 0,
				      as_stream(stream), d_row_of + (uint64_t)at * top_k,
				      d_weight ? d_weight + (uint64_t)at * top_k : nullptr,
				      row_at(static_cast<const T *>(d_dout), dout_pitch, at), static_cast<const T *>(d_rows),
				      static_cast<T *>(d_drows), d_dweight ? d_dweight + (uint64_t)at * top_k : nullptr, dout_pitch, rows_pitch,
				      drows_pitch, max_rows, top_k, width);
		}
	});
	OFI_AMD_HIP_TRY(hipGetLastError());
	return 0;
}

} /* extern "C" */
