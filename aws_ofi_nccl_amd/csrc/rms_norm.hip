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

/* A chunk's own elements times `inverse` as e4m3 */
template <uint32_t V> __device__ __forceinline__ void store_q(uint8_t *p, uint32_t skip, const float (&f)[V], float inverse)
{
	if constexpr (V == 1) {
		if (skip == 0) {
			p[0] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[0] * inverse, 0.0f, 0, false);
		}
	} else {
		typedef uint32_t words_t __attribute__((ext_vector_type(V / 4), aligned(1)));
		words_t w;
#pragma unroll
		for (uint32_t i = 0; i < V / 4; i++) {
			const int low = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i] * inverse, f[4 * i + 1] * inverse, 0, false);
			w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2] * inverse, f[4 * i + 3] * inverse, low, true);
		}
		if (skip == 0) {
			*reinterpret_cast<words_t *>(p) = w;
		} else {
#pragma unroll
			for (uint32_t i = 0; i < V; i++) {
				if (i >= skip) {
					p[i] = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
				}
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

template <typename T, uint32_t V>
__device__ __forceinline__ void load_gain(const void *__restrict__ gain, bool gain_f32, uint32_t from, float (&g)[V])
{
	if (!gain_f32) {
		to_floats<T, V>(load_raw<false, T, V>(static_cast<const T *>(gain) + from), 0, g);
		return;
	}
#pragma unroll
	for (uint32_t i = 0; i < V; i++) {
		g[i] = static_cast<const float *>(gain)[from + i];
	}
}

/* A chunk's own elements of a row of floats */
template <uint32_t V> __device__ __forceinline__ void store_floats(float *p, uint32_t skip, const float (&f)[V])
{
	if constexpr (V == 8) {
		if (skip == 0) {
			store_piece<false, float, 4>(p, 0, reinterpret_cast<const float(&)[4]>(f[0]));
			store_piece<false, float, 4>(p + 4, 0, reinterpret_cast<const float(&)[4]>(f[4]));
		} else {
#pragma unroll
			for (uint32_t i = 0; i < V; i++) {
				if (i >= skip) {
					p[i] = f[i];
				}
			}
		}
	} else {
		store_piece<false, float, V>(p, skip, f);
	}
}

__device__ __forceinline__ float scale_of(uint32_t amax_bits)
{
	/* __builtin_fmaxf would drop a NaN, which every value of its group is then to show */
	const float s = __uint_as_float(amax_bits) / 448.0f;
	return s < 0x1p-126f ? 0x1p-126f : s;
}

/* sum may be x or residual: a lane has read what it writes before any lane of its row writes.  group_lanes: lanes that share a
 * scale, 0: the whole row does */
template <typename T, uint32_t V, int WAVES, int R, bool STREAM>
__global__ __launch_bounds__(64 * WAVES) void rms_norm_kernel(const T *x, const T *residual, const void *__restrict__ gain,
							      uint64_t x_pitch, uint64_t residual_pitch, uint32_t first, uint32_t width,
							      float eps, uint32_t group_lanes, bool gain_f32, norm_out_t o)
{
	constexpr uint32_t B = 64 * WAVES;
	__shared__ float part[2 * WAVES];
	const uint64_t row = first + blockIdx.x;
	raw_t<T, V> c[R], d[R];
#pragma unroll
	for (int k = 0; k < R; k++) {
		c[k] = load_raw<STREAM, T, V>(row_at(x, x_pitch, row) + place_of<V>((k * B + threadIdx.x) * V, width).from);
	}
	if (residual) {
#pragma unroll
		for (int k = 0; k < R; k++) {
			d[k] = load_raw<STREAM, T, V>(row_at(residual, residual_pitch, row) +
						      place_of<V>((k * B + threadIdx.x) * V, width).from);
		}
	}
	float v[R][V];
	float squares = 0.0f;
#pragma unroll
	for (int k = 0; k < R; k++) {
		const uint32_t skip = place_of<V>((k * B + threadIdx.x) * V, width).skip;
		to_floats<T, V>(c[k], skip, v[k]);
		if (residual) {
			float f[V];
			to_floats<T, V>(d[k], skip, f);
#pragma unroll
			for (uint32_t i = 0; i < V; i++) {
				v[k][i] += f[i];
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
		const place_t here = place_of<V>(at, width);
		if (o.sum && at < width) {
			store_piece<false, T, V>(row_at(static_cast<T *>(o.sum), o.sum_pitch, row) + here.from, here.skip, v[k]);
		}
		float g[V];
		load_gain<T, V>(gain, gain_f32, here.from, g);
#pragma unroll
		for (uint32_t i = 0; i < V; i++) {
			v[k][i] = v[k][i] * rstd * g[i];
		}
		if (o.out && at < width) {
			store_piece<false, T, V>(row_at(static_cast<T *>(o.out), o.out_pitch, row) + here.from, here.skip, v[k]);
		}
		if (!o.q) {
			continue;
		}
		uint32_t m = 0;
#pragma unroll
		for (uint32_t i = 0; i < V; i++) {
			m = max(m, i < here.skip ? 0u : abs_bits(v[k][i])); /* a skipped 0 times a rstd or a gain that is no number is none */
		}
		if (group_lanes == 0) {
			most = max(most, m);
			continue;
		}
		const float scale = scale_of(max_bits_of_group(m, group_lanes));
		if (at < width) {
			store_q<V>(o.q + row * o.q_pitch + here.from, here.skip, v[k], 1.0f / scale);
			const uint32_t chunk = k * B + threadIdx.x;
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
			const place_t here = place_of<V>(at, width);
			if (at < width) {
				store_q<V>(o.q + row * o.q_pitch + here.from, here.skip, v[k], 1.0f / scale);
			}
		}
		if (threadIdx.x == 0) {
			row_at(o.scale, o.scale_pitch, row)[0] = scale;
		}
	}
}

/* dx = ds + rstd (g dn - h mean(g dn h)), h = s rstd; dg = sum over rows of dn h: each workgroup sums its own rows and the
 * partial sums are added up in the order of the workgroups, so that the result is the same every time.  dx may be dout or dsum:
 * a lane has read what it writes. */
template <typename T, uint32_t V, int WAVES, int R, bool STREAM>
__global__ __launch_bounds__(64 * WAVES) void rms_norm_grad_kernel(const T *dout, const T *__restrict__ s,
								   const float *__restrict__ rstds, const void *__restrict__ gain,
								   const T *dsum, uint64_t dout_pitch, uint64_t s_pitch, uint64_t dsum_pitch,
								   uint32_t n_rows, uint32_t width, bool gain_f32, T *dx, uint64_t dx_pitch,
								   float *__restrict__ partial)
{
	constexpr uint32_t B = 64 * WAVES;
	__shared__ float part[2][WAVES];
	float g[R][V], dg[R][V];
#pragma unroll
	for (int k = 0; k < R; k++) {
		load_gain<T, V>(gain, gain_f32, place_of<V>((k * B + threadIdx.x) * V, width).from, g[k]);
#pragma unroll
		for (uint32_t i = 0; i < V; i++) {
			dg[k][i] = 0.0f;
		}
	}
	uint32_t turn = 0;
	for (uint64_t row = blockIdx.x; row < n_rows; row += gridDim.x, turn ^= 1u) {
		raw_t<T, V> dc[R], sc[R], pc[R];
#pragma unroll
		for (int k = 0; k < R; k++) {
			const uint32_t from = place_of<V>((k * B + threadIdx.x) * V, width).from;
			dc[k] = load_raw<STREAM, T, V>(row_at(dout, dout_pitch, row) + from);
			sc[k] = load_raw<STREAM, T, V>(row_at(s, s_pitch, row) + from);
		}
		if (dsum) {
#pragma unroll
			for (int k = 0; k < R; k++) {
				pc[k] = load_raw<STREAM, T, V>(row_at(dsum, dsum_pitch, row) +
							       place_of<V>((k * B + threadIdx.x) * V, width).from);
			}
		}
		const float rstd = rstds[row];
		float d[R][V], h[R][V], along = 0.0f;
#pragma unroll
		for (int k = 0; k < R; k++) {
			const uint32_t skip = place_of<V>((k * B + threadIdx.x) * V, width).skip;
			to_floats<T, V>(dc[k], skip, d[k]);
			to_floats<T, V>(sc[k], skip, h[k]);
#pragma unroll
			for (uint32_t i = 0; i < V; i++) {
				h[k][i] *= rstd;
				dg[k][i] = __builtin_fmaf(d[k][i], h[k][i], dg[k][i]);
				d[k][i] *= g[k][i];
				along = i < skip ? along : __builtin_fmaf(d[k][i], h[k][i], along);
			}
		}
		const float mean = block_sum<WAVES>(along, part[turn]) / (float)width;
#pragma unroll
		for (int k = 0; k < R; k++) {
			const uint32_t at = (k * B + threadIdx.x) * V;
			const place_t here = place_of<V>(at, width);
			if (at < width) {
				float r[V];
#pragma unroll
				for (uint32_t i = 0; i < V; i++) {
					r[i] = 0.0f;
				}
				if (dsum) {
					to_floats<T, V>(pc[k], 0, r);
				}
#pragma unroll
				for (uint32_t i = 0; i < V; i++) {
					r[i] = __builtin_fmaf(rstd, __builtin_fmaf(-h[k][i], mean, d[k][i]), r[i]);
				}
				store_piece<false, T, V>(row_at(dx, dx_pitch, row) + here.from, here.skip, r);
			}
		}
	}
	if (!partial) {
		return;
	}
#pragma unroll
	for (int k = 0; k < R; k++) {
		const uint32_t at = (k * B + threadIdx.x) * V;
		const place_t here = place_of<V>(at, width);
		if (at < width) {
			store_floats<V>(partial + (uint64_t)blockIdx.x * width + here.from, here.skip, dg[k]);
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
#pragma unroll 8
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

constexpr uint32_t kGradBlocks = 512;
/* Workgroups of the gradient: each reads and writes a row at a time */
inline uint32_t grad_blocks(uint32_t n_rows)
{
	return n_rows < kGradBlocks ? n_rows : kGradBlocks;
}

/* Calls f with the wavefronts of a workgroup and the chunks of a lane that hold a row of `chunks` */
template <uint32_t V, typename F> void with_row_shape(uint32_t chunks, F f)
{
	auto with = [&](auto waves, auto r) { f(waves, r); };
	if constexpr (V == 1) { /* narrower than a chunk */
		with(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
	} else {
		if (chunks <= 64) {
			with(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
		} else if (chunks <= 128) {
			with(std::integral_constant<int, 2>{}, std::integral_constant<int, 1>{});
		} else if (chunks <= 256) {
			with(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{});
		} else if (chunks <= 512) {
			with(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
		} else if (chunks <= 1024) {
			with(std::integral_constant<int, 8>{}, std::integral_constant<int, 2>{});
		} else if (chunks <= 2048) {
			with(std::integral_constant<int, 16>{}, std::integral_constant<int, 2>{});
		} else if (V == 8 || chunks <= 4096) {
			with(std::integral_constant<int, 16>{}, std::integral_constant<int, 4>{});
		} else {
			with(std::integral_constant<int, 16>{}, std::integral_constant<int, V == 4 ? 8 : 4>{});
		}
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
	const bool stream_rows = on_chunks(d_x, x_pitch) && on_chunks(d_residual, residual_pitch);
	with_row_type(type, width, [&](auto element, auto v) {
		using T = decltype(element);
		constexpr uint32_t V = decltype(v)::value;
		const uint32_t group_lanes = V == 1 ? 0 : group / V; /* narrower rows are one group, however long it is */
		with_row_shape<V>((width + V - 1) / V, [&](auto waves, auto r) {
			constexpr int W = decltype(waves)::value, R = decltype(r)::value;
			for (uint32_t first = 0; first < n_rows; first += kRowsOfLaunch) {
				launch_kernel(stream_rows ? rms_norm_kernel<T, V, W, R, true> : rms_norm_kernel<T, V, W, R, false>,
					      dim3(n_rows - first < kRowsOfLaunch ? n_rows - first : kRowsOfLaunch), dim3(64 * W), 0,
					      as_stream(stream), static_cast<const T *>(d_x), static_cast<const T *>(d_residual), d_gain, x_pitch,
					      residual_pitch, first, width, eps, group_lanes, gain_type == OFI_AMD_FLOAT32, o);
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
		const bool stream_rows = on_chunks(d_dout, dout_pitch) && on_chunks(d_s, s_pitch) && on_chunks(d_dsum, dsum_pitch);
		with_row_type(type, width, [&](auto element, auto v) {
			using T = decltype(element);
			constexpr uint32_t V = decltype(v)::value;
			with_row_shape<V>((width + V - 1) / V, [&](auto waves, auto r) {
				constexpr int W = decltype(waves)::value, R = decltype(r)::value;
				launch_kernel(stream_rows ? rms_norm_grad_kernel<T, V, W, R, true> : rms_norm_grad_kernel<T, V, W, R, false>,
					      dim3(blocks), dim3(64 * W), 0, as_stream(stream), static_cast<const T *>(d_dout),
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
