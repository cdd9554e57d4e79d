/*
 * Tokens back from their experts: the weighted sum of a token's rows, and its gradient.
 *
 *   out_t = add_t + sum_k w_tk y[row_tk]        dy[row_tk] = w_tk dout_t        dw_tk = <dout_t, y[row_tk]>
 *
 * A pair without a row (an index outside the rows) is passed over, whatever its weight is.
 */
#include "common.hpp"
#include "ofi_amd_hotpath.h"
#include "row_types.hpp"

namespace {

using namespace ofi_amd;

constexpr uint32_t kMaxTopK = 64;
constexpr uint32_t kMaxWidth = 1u << 20;
constexpr int kWaves = 4;
constexpr uint32_t kAtOnce = 8; /* rows of a token that are read together */

/* One chunk of the output per lane */
template <typename T>
__global__ __launch_bounds__(64 * kWaves) void token_combine_kernel(const int32_t *__restrict__ row_of, const float *__restrict__ weight,
								    const T *__restrict__ rows, const T *add, T *out, uint64_t rows_pitch,
								    uint64_t add_pitch, uint64_t out_pitch, uint32_t max_rows, uint32_t top_k,
								    uint32_t width)
{
	constexpr uint32_t V = kChunk<T>;
	const uint32_t token = blockIdx.x;
	const uint32_t at = (blockIdx.y * 64u * kWaves + threadIdx.x) * V;
	if (at >= width) {
		return;
	}
	float sum[V];
#pragma unroll
	for (uint32_t i = 0; i < V; i++) {
		sum[i] = 0.0f;
	}
	if (add) {
		load_chunk(row_at(add, add_pitch, token) + at, width - at, sum);
	}
	for (uint32_t k = 0; k < top_k; k++) {
		const uint64_t p = (uint64_t)token * top_k + k;
		const uint32_t row = (uint32_t)row_of[p];
		if (row < max_rows) {
			const float w = weight ? weight[p] : 1.0f;
			float f[V];
			load_chunk(row_at(rows, rows_pitch, row) + at, width - at, f);
#pragma unroll
			for (uint32_t i = 0; i < V; i++) {
				sum[i] = __builtin_fmaf(w, f[i], sum[i]);
			}
		}
	}
	store_chunk(row_at(out, out_pitch, token) + at, width - at, sum);
}

/* One workgroup per token, up to kAtOnce of its rows at a time */
template <typename T>
__global__ __launch_bounds__(64 * kWaves) void token_combine_grad_kernel(const int32_t *__restrict__ row_of,
									 const float *__restrict__ weight, const T *__restrict__ dout,
									 const T *rows, T *drows, float *__restrict__ dweight,
									 uint64_t dout_pitch, uint64_t rows_pitch, uint64_t drows_pitch,
									 uint32_t max_rows, uint32_t top_k, uint32_t width)
{
	constexpr uint32_t V = kChunk<T>;
	__shared__ float part[kWaves][kAtOnce];
	const uint64_t token = blockIdx.x;
	const T *dr = row_at(dout, dout_pitch, token);
	for (uint32_t k0 = 0; k0 < top_k; k0 += kAtOnce) {
		float dot[kAtOnce];
#pragma unroll
		for (uint32_t k = 0; k < kAtOnce; k++) {
			dot[k] = 0.0f;
		}
		for (uint32_t at = threadIdx.x * V; at < width; at += 64u * kWaves * V) {
			float d[V];
			load_chunk(dr + at, width - at, d);
#pragma unroll
			for (uint32_t k = 0; k < kAtOnce; k++) {
				if (k0 + k >= top_k) {
					break;
				}
				const uint64_t p = token * top_k + k0 + k;
				const uint32_t row = (uint32_t)row_of[p];
				if (row >= max_rows) {
					continue;
				}
				if (dweight) {
					float f[V];
					load_chunk(row_at(rows, rows_pitch, row) + at, width - at, f);
#pragma unroll
					for (uint32_t i = 0; i < V; i++) {
						dot[k] = __builtin_fmaf(d[i], f[i], dot[k]);
					}
				}
				if (drows) {
					const float w = weight ? weight[p] : 1.0f;
					float f[V];
#pragma unroll
					for (uint32_t i = 0; i < V; i++) {
						f[i] = w * d[i];
					}
					store_chunk(row_at(drows, drows_pitch, row) + at, width - at, f);
				}
			}
		}
		if (!dweight) {
			continue;
		}
#pragma unroll
		for (uint32_t k = 0; k < kAtOnce; k++) {
			const float d = sum_over<64>(dot[k]);
			if ((threadIdx.x & 63u) == 0) {
				part[threadIdx.x >> 6][k] = d;
			}
		}
		__syncthreads();
		if (threadIdx.x < kAtOnce && k0 + threadIdx.x < top_k) {
			float d = part[0][threadIdx.x];
#pragma unroll
			for (int w = 1; w < kWaves; w++) {
				d += part[w][threadIdx.x];
			}
			dweight[token * top_k + k0 + threadIdx.x] = d;
		}
		__syncthreads();
	}
}

constexpr uint32_t kTokensOfLaunch = 1u << 22; /* with 256 lanes each within the 32 bits of a launch's size */

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
	with_row_type(type, [&](auto element) {
		using T = decltype(element);
		constexpr uint32_t span = 64 * kWaves * kChunk<T>;
		for (uint32_t at = 0; at < n_tokens; at += kTokensOfLaunch) {
			launch_kernel(token_combine_kernel<T>,
				      dim3(n_tokens - at < kTokensOfLaunch ? n_tokens - at : kTokensOfLaunch, (width + span - 1) / span),
				      dim3(64 * kWaves), 0, as_stream(stream), d_row_of + (uint64_t)at * top_k,
				      d_weight ? d_weight + (uint64_t)at * top_k : nullptr, static_cast<const T *>(d_rows),
				      d_add ? row_at(static_cast<const T *>(d_add), add_pitch, at) : nullptr,
				      row_at(static_cast<T *>(d_out), out_pitch, at), rows_pitch, add_pitch, out_pitch, max_rows, top_k, width);
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
	if (!rows_ok(d_dout, dout_pitch, n_tokens, bytes, size) || (!d_drows && !d_dweight) ||
	    (reinterpret_cast<uintptr_t>(d_dweight) & 3u) ||
	    (max_rows != 0 && ((d_dweight && !rows_ok(d_rows, rows_pitch, max_rows, bytes, size)) ||
			       (d_drows && !rows_ok(d_drows, drows_pitch, max_rows, bytes, size))))) {
		return -EINVAL;
	}
	with_row_type(type, [&](auto element) {
		using T = decltype(element);
		for (uint32_t at = 0; at < n_tokens; at += kTokensOfLaunch) {
			launch_kernel(token_combine_grad_kernel<T>, dim3(n_tokens - at < kTokensOfLaunch ? n_tokens - at : kTokensOfLaunch),
				      dim3(64 * kWaves), 0, as_stream(stream), d_row_of + (uint64_t)at * top_k,
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
