/*
 * Root-mean-square norm of rows with the residual's addition and an 8-bit output, and its gradient.
 *
 *   s = x + r,  rstd = 1 / sqrt(mean(s^2) + eps),  n = s rstd g,  q = e4m3(n / scale),  scale = max(amax|n| / 448, 2^-126)
 *
 * per group of columns or per row.  One workgroup holds a row in registers, so that x and r are read once.
 */
#include <type_traits>

#include "common.hpp"
#include "ofi_amd_hotpath.h"
#include "row_types.hpp"

namespace {

using namespace ofi_amd;

constexpr uint32_t kMaxWidth = 32768;
constexpr uint32_t kRowsOfLaunch = 1u << 21; /* with 1024 lanes each within the 32 bits of a launch's size */

struct norm_out_t {
	void *sum;
	uint64_t sum_pitch;
	void *out;
	uint64_t out_pitch;
	uint8_t *q;
	uint64_t q_pitch;
	float *scale;
	uint64_t scale_pitch;
	float *rstd;
};

/* f * inverse as e4m3 */
template <uint32_t V>
__device__ __forceinline__ void store_q(uint8_t *__restrict__ p, uint32_t left, const float (&f)[V], float inverse)
{
	uint32_t w[V / 4];
#pragma unroll
	for (uint32_t i = 0; i < V / 4; i++) {
		w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i] * inverse, f[4 * i + 1] * inverse, 0, false);
		w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2] * inverse, f[4 * i + 3] * inverse, (int)w[i], true);
	}
	if (left >= V) {
		struct __attribute__((packed, aligned(1))) words_t {
			uint32_t w[V / 4];
		} all;
#pragma unroll
		for (uint32_t i = 0; i < V / 4; i++) {
			all.w[i] = w[i];
		}
		*reinterpret_cast<words_t *>(p) = all;
	} else {
#pragma unroll
		for (uint32_t i = 0; i < V; i++) {
			if (i < left) {
				p[i] = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
			}
		}
	}
}

/* The largest of each group of `lanes` neighbours (4 to 64), in all of them */
__device__ __forceinline__ uint32_t max_bits_of_group(uint32_t m, uint32_t lanes)
{
	m = max_bits_over<4>(m);
	if (lanes >= 8) {
		m = max(m, dpp<0x141>(m));
	}
	if (lanes >= 16) {
		m = max(m, dpp<0x140>(m));
	}
	if (lanes >= 32) {
		m = max(m, (uint32_t)__shfl_xor((int)m, 16));
	}
	if (lanes >= 64) {
		m = max(m, (uint32_t)__shfl_xor((int)m, 32));
	}
	return m;
}

template <typename T>
__device__ __forceinline__ void load_gain(const void *__restrict__ gain, bool gain_f32, uint32_t at, uint32_t left, float (&g)[kChunk<T>])
{
	if (!gain_f32) {
		load_chunk(static_cast<const T *>(gain) + at, left, g);
		return;
	}
#pragma unroll
	for (uint32_t i = 0; i < kChunk<T>; i++) {
		g[i] = i < left ? static_cast<const float *>(gain)[at + i] : 0.0f;
	}
}

__device__ __forceinline__ float scale_of(uint32_t amax_bits)
{
	/* __builtin_fmaxf would drop a NaN, which every value of its group is then to show */
	const float s = __uint_as_float(amax_bits) / 448.0f;
	return s < 0x1p-126f ? 0x1p-126f : s;
}

/* sum may be x or residual: a lane reads what it writes, and first.  group_lanes: lanes that share a scale, 0: the whole row does */
template <typename T, int WAVES, int R>
__global__ __launch_bounds__(64 * WAVES) void rms_norm_kernel(const T *x, const T *residual, const void *__restrict__ gain,
							      uint64_t x_pitch, uint64_t residual_pitch, uint32_t first, uint32_t width,
							      float eps, uint32_t group_lanes, bool gain_f32, norm_out_t o)
{
	constexpr uint32_t V = kChunk<T>, B = 64 * WAVES;
	__shared__ float part[2 * WAVES];
	const uint64_t row = first + blockIdx.x;
	const T *xr = row_at(x, x_pitch, row);
	const T *rr = residual ? row_at(residual, residual_pitch, row) : nullptr;
	float v[R][V];
	float squares = 0.0f;
#pragma unroll
	for (int k = 0; k < R; k++) {
		const uint32_t at = (k * B + threadIdx.x) * V;
#pragma unroll
		for (uint32_t i = 0; i < V; i++) {
			v[k][i] = 0.0f;
		}
		if (at < width) {
			load_chunk(xr + at, width - at, v[k]);
			if (rr) {
				float f[V];
				load_chunk(rr + at, width - at, f);
#pragma unroll
				for (uint32_t i = 0; i < V; i++) {
					v[k][i] += f[i];
				}
			}
		}
#pragma unroll
		for (uint32_t i = 0; i < V; i++) {
			squares = __builtin_fmaf(v[k][i], v[k][i], squares);
		}
	}
	const float rstd = 1.0f / __builtin_sqrtf(block_sum<WAVES>(squares, part) / (float)width + eps);
	if (o.rstd && threadIdx.x == 0) {
		o.rstd[row] = rstd;
	}
	uint32_t most = 0;
#pragma unroll
	for (int k = 0; k < R; k++) {
		const uint32_t at = (k * B + threadIdx.x) * V;
		uint32_t m = 0;
		if (at < width) {
			if (o.sum) {
				store_chunk(row_at(static_cast<T *>(o.sum), o.sum_pitch, row) + at, width - at, v[k]);
			}
			float g[V];
			load_gain<T>(gain, gain_f32, at, width - at, g);
#pragma unroll
			for (uint32_t i = 0; i < V; i++) {
				v[k][i] = v[k][i] * rstd * g[i];
				m = max(m, i < width - at ? abs_bits(v[k][i]) : 0u); /* beyond: 0 rstd, a NaN where the row has none left */
			}
			if (o.out) {
				store_chunk(row_at(static_cast<T *>(o.out), o.out_pitch, row) + at, width - at, v[k]);
			}
		}
		if (!o.q) {
			continue;
		}
		if (group_lanes == 0) {
			most = max(most, m);
			continue;
		}
		const float scale = scale_of(max_bits_of_group(m, group_lanes));
		if (at < width) {
			const uint32_t chunk = k * B + threadIdx.x;
			store_q(o.q + row * o.q_pitch + at, width - at, v[k], 1.0f / scale);
			if ((chunk & (group_lanes - 1u)) == 0) {
				row_at(o.scale, o.scale_pitch, row)[chunk / group_lanes] = scale;
			}
		}
	}
	if (o.q && group_lanes == 0) {
		const float scale = scale_of(block_max_bits<WAVES>(most, reinterpret_cast<uint32_t *>(part) + WAVES));
#pragma unroll
		for (int k = 0; k < R; k++) {
			const uint32_t at = (k * B + threadIdx.x) * V;
			if (at < width) {
				store_q(o.q + row * o.q_pitch + at, width - at, v[k], 1.0f / scale);
			}
		}
		if (threadIdx.x == 0) {
			row_at(o.scale, o.scale_pitch, row)[0] = scale;
		}
	}
}

/* dx = ds + rstd (g dn - h mean(g dn h)), h = s rstd; dg = sum over rows of dn h: each workgroup sums its own rows and the
 * partial sums are added up in the order of the workgroups, so that the result is the same every time */
template <typename T, int WAVES, int R>
__global__ __launch_bounds__(64 * WAVES) void rms_norm_grad_kernel(const T *dout, const T *__restrict__ s,
								   const float *__restrict__ rstds, const void *__restrict__ gain,
								   const T *dsum, uint64_t dout_pitch, uint64_t s_pitch,
								   uint64_t dsum_pitch, uint32_t n_rows, uint32_t width, bool gain_f32,
								   T *dx, uint64_t dx_pitch, float *__restrict__ partial)
{
	constexpr uint32_t V = kChunk<T>, B = 64 * WAVES;
	__shared__ float part[2][WAVES];
	float g[R][V], dg[R][V];
#pragma unroll
	for (int k = 0; k < R; k++) {
		const uint32_t at = (k * B + threadIdx.x) * V;
#pragma unroll
		for (uint32_t i = 0; i < V; i++) {
			dg[k][i] = g[k][i] = 0.0f;
		}
		if (at < width) {
			load_gain<T>(gain, gain_f32, at, width - at, g[k]);
		}
	}
	uint32_t turn = 0;
	for (uint64_t row = blockIdx.x; row < n_rows; row += gridDim.x, turn ^= 1u) {
		const T *dr = row_at(dout, dout_pitch, row), *sr = row_at(s, s_pitch, row);
		const float rstd = rstds[row];
		float d[R][V], h[R][V], along = 0.0f;
#pragma unroll
		for (int k = 0; k < R; k++) {
			const uint32_t at = (k * B + threadIdx.x) * V;
#pragma unroll
			for (uint32_t i = 0; i < V; i++) {
				d[k][i] = h[k][i] = 0.0f;
			}
			if (at < width) {
				load_chunk(dr + at, width - at, d[k]);
				load_chunk(sr + at, width - at, h[k]);
			}
#pragma unroll
			for (uint32_t i = 0; i < V; i++) {
				h[k][i] *= rstd;
				dg[k][i] = __builtin_fmaf(d[k][i], h[k][i], dg[k][i]);
				d[k][i] *= g[k][i];
				along = __builtin_fmaf(d[k][i], h[k][i], along);
			}
		}
		const float mean = block_sum<WAVES>(along, part[turn]) / (float)width;
#pragma unroll
		for (int k = 0; k < R; k++) {
			const uint32_t at = (k * B + threadIdx.x) * V;
			if (at < width) {
				float r[V];
#pragma unroll
				for (uint32_t i = 0; i < V; i++) {
					r[i] = 0.0f;
				}
				if (dsum) {
					load_chunk(row_at(dsum, dsum_pitch, row) + at, width - at, r);
				}
#pragma unroll
				for (uint32_t i = 0; i < V; i++) {
					r[i] = __builtin_fmaf(rstd, __builtin_fmaf(-h[k][i], mean, d[k][i]), r[i]);
				}
				store_chunk(row_at(dx, dx_pitch, row) + at, width - at, r);
			}
		}
	}
	if (!partial) {
		return;
	}
#pragma unroll
	for (int k = 0; k < R; k++) {
		const uint32_t at = (k * B + threadIdx.x) * V;
		if (at < width) {
			store_chunk(partial + (uint64_t)blockIdx.x * width + at, width - at >= 4 ? 4 : width - at,
				    reinterpret_cast<float(&)[4]>(dg[k][0]));
			if (V == 8 && at + 4 < width) {
				store_chunk(partial + (uint64_t)blockIdx.x * width + at + 4, width - at - 4,
					    reinterpret_cast<float(&)[4]>(dg[k][V - 4]));
			}
		}
	}
}

/* 64 columns of a workgroup, its wavefronts at the parts by turns */
constexpr int kGainWaves = 16;
__global__ __launch_bounds__(64 * kGainWaves) void rms_norm_gain_kernel(const float *__restrict__ partial, float *__restrict__ dgain,
									uint32_t parts, uint32_t width)
{
	__shared__ float sums[kGainWaves][64];
	const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, column = blockIdx.x * 64u + lane;
	float total = 0.0f;
	if (column < width) {
		for (uint32_t p = wave; p < parts; p += kGainWaves) {
			total += partial[(uint64_t)p * width + column];
		}
	}
	sums[wave][lane] = total;
	__syncthreads();
	if (wave == 0 && column < width) {
#pragma unroll
		for (int w = 1; w < kGainWaves; w++) {
			total += sums[w][lane];
		}
		dgain[column] = total;
	}
}

/* Workgroups of the gradient: each reads and writes a row at a time */
inline uint32_t grad_blocks(uint32_t n_rows)
{
	return n_rows < 1024u ? n_rows : 1024u;
}

/* Calls f with the wavefronts of a workgroup and the chunks of a lane that hold a row of `chunks` */
template <typename T, typename F> void with_row_shape(uint32_t chunks, F f)
{
	if (chunks <= 64) {
		f(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
	} else if (chunks <= 256) {
		f(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{});
	} else if (chunks <= 512) {
		f(std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{});
	} else if (chunks <= 1024) {
		f(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
	} else if (chunks <= 2048) {
		f(std::integral_constant<int, 16>{}, std::integral_constant<int, 2>{});
	} else if (kChunk<T> == 8 || chunks <= 4096) {
		f(std::integral_constant<int, 16>{}, std::integral_constant<int, 4>{});
	} else {
		f(std::integral_constant<int, 16>{}, std::integral_constant<int, 32 / (int)kChunk<T>>{});
	}
}

} // namespace

extern "C" {

int ofi_amd_rms_norm(const void *d_x, uint64_t x_pitch, const void *d_residual, uint64_t residual_pitch, const void *d_gain,
		     int gain_type, uint32_t n_rows, uint32_t width, int type, float eps, void *d_sum, uint64_t sum_pitch, void *d_out,
		     uint64_t out_pitch, void *d_q, uint64_t q_pitch, float *d_scale, uint64_t scale_pitch, uint32_t group, float *d_rstd,
		     void *stream)
{
	int rc = require_device();
	if (rc != 0) {
		return rc;
	}
	const uint32_t size = row_type_size(type);
	if (!size || (gain_type != type && gain_type != OFI_AMD_FLOAT32) || width == 0 || !(eps >= 0.0f)) {
		return -EINVAL;
	}
	if (width > kMaxWidth || n_rows > 0x7fffffffu) {
		return -E2BIG;
	}
	if (d_q && group != 0 && group != 32 && group != 64 && group != 128 && group != 256) {
		return -EINVAL;
	}
	if (n_rows == 0) {
		return 0;
	}
	const uint64_t bytes = (uint64_t)width * size;
	const uint32_t groups = group == 0 ? 1 : (width + group - 1) / group;
	if (!rows_ok(d_x, x_pitch, n_rows, bytes, size) || (d_residual && !rows_ok(d_residual, residual_pitch, n_rows, bytes, size)) ||
	    !rows_ok(d_gain, 0, 1, 0, gain_type == OFI_AMD_FLOAT32 ? 4 : size) || (d_sum && !rows_ok(d_sum, sum_pitch, n_rows, bytes, size)) ||
	    (d_out && !rows_ok(d_out, out_pitch, n_rows, bytes, size)) || (!d_q != !d_scale) ||
	    (d_q && (!rows_ok(d_q, q_pitch, n_rows, width, 1) || !rows_ok(d_scale, scale_pitch, n_rows, 4ull * groups, 4))) ||
	    (d_rstd && (reinterpret_cast<uintptr_t>(d_rstd) & 3u)) || (!d_sum && !d_out && !d_q && !d_rstd)) {
		return -EINVAL;
	}
	const norm_out_t o = { d_sum, sum_pitch, d_out, out_pitch, static_cast<uint8_t *>(d_q), q_pitch, d_scale, scale_pitch, d_rstd };
	with_row_type(type, [&](auto element) {
		using T = decltype(element);
		with_row_shape<T>((width + kChunk<T> - 1) / kChunk<T>, [&](auto waves, auto r) {
			for (uint32_t first = 0; first < n_rows; first += kRowsOfLaunch) {
				launch_kernel(rms_norm_kernel<T, decltype(waves)::value, decltype(r)::value>,
					      dim3(n_rows - first < kRowsOfLaunch ? n_rows - first : kRowsOfLaunch), dim3(64 * waves), 0,
					      as_stream(stream), static_cast<const T *>(d_x), static_cast<const T *>(d_residual), d_gain, x_pitch,
					      residual_pitch, first, width, eps, group / kChunk<T>, gain_type == OFI_AMD_FLOAT32, o);
			}
		});
	});
	OFI_AMD_HIP_TRY(hipGetLastError());
	return 0;
}

uint64_t ofi_amd_rms_norm_grad_work_bytes(uint32_t n_rows, uint32_t width)
{
	return (uint64_t)grad_blocks(n_rows) * width * sizeof(float);
}

int ofi_amd_rms_norm_grad(const void *d_dout, uint64_t dout_pitch, const void *d_s, uint64_t s_pitch, const float *d_rstd,
			  const void *d_gain, int gain_type, uint32_t n_rows, uint32_t width, int type, const void *d_dsum,
			  uint64_t dsum_pitch, void *d_dx, uint64_t dx_pitch, float *d_dgain, void *d_work, uint64_t work_bytes, void *stream)
{
	int rc = require_device();
	if (rc != 0) {
		return rc;
	}
	const uint32_t size = row_type_size(type);
	if (!size || (gain_type != type && gain_type != OFI_AMD_FLOAT32) || width == 0) {
		return -EINVAL;
	}
	if (width > kMaxWidth || n_rows > 0x7fffffffu) {
		return -E2BIG;
	}
	if (d_dgain && ((reinterpret_cast<uintptr_t>(d_dgain) & 3u) || (n_rows != 0 &&
	    (!d_work || (reinterpret_cast<uintptr_t>(d_work) & 3u) || work_bytes < ofi_amd_rms_norm_grad_work_bytes(n_rows, width))))) {
		return -EINVAL;
	}
	const uint64_t bytes = (uint64_t)width * size;
	if (n_rows != 0 && (!rows_ok(d_dout, dout_pitch, n_rows, bytes, size) || !rows_ok(d_s, s_pitch, n_rows, bytes, size) ||
			    !rows_ok(d_rstd, 0, 1, 0, 4) || !rows_ok(d_gain, 0, 1, 0, gain_type == OFI_AMD_FLOAT32 ? 4 : size) ||
			    (d_dsum && !rows_ok(d_dsum, dsum_pitch, n_rows, bytes, size)) || !rows_ok(d_dx, dx_pitch, n_rows, bytes, size))) {
		return -EINVAL;
	}
	const uint32_t blocks = grad_blocks(n_rows);
	float *partial = d_dgain ? static_cast<float *>(d_work) : nullptr;
	if (n_rows != 0) {
		with_row_type(type, [&](auto element) {
			using T = decltype(element);
			with_row_shape<T>((width + kChunk<T> - 1) / kChunk<T>, [&](auto waves, auto r) {
				launch_kernel(rms_norm_grad_kernel<T, decltype(waves)::value, decltype(r)::value>, dim3(blocks),
					      dim3(64 * waves), 0, as_stream(stream), static_cast<const T *>(d_dout),
					      static_cast<const T *>(d_s), d_rstd, d_gain, static_cast<const T *>(d_dsum), dout_pitch, s_pitch,
					      dsum_pitch, n_rows, width, gain_type == OFI_AMD_FLOAT32, static_cast<T *>(d_dx), dx_pitch, partial);
			});
		});
	}
	if (d_dgain) { /* of no rows: zeros */
		launch_kernel(rms_norm_gain_kernel, dim3((width + 63u) / 64u), dim3(64 * kGainWaves), 0, as_stream(stream), partial, d_dgain,
			      blocks, width);
	}
	OFI_AMD_HIP_TRY(hipGetLastError());
	return 0;
}

} /* extern "C" */
