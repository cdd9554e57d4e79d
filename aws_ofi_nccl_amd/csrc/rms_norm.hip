/*
 * Root-mean-square norm of rows with the residual's addition and an 8-bit output, and its gradient.
 *
 *   s = x + r,  rstd = 1 / sqrt(mean(s^2) + eps),  n = s rstd g,  q = e4m3(n / scale),  scale = max(amax|n| / 448, 2^-126)
 *
 * per group of columns or per row.  A row is held in registers from its reading to its writing, so that every byte crosses the memory
 * interface once, and memory is what bounds it: 16,384 rows of 8192 bfloat16 with residual to e4m3, 944 MB, 155.5 us = 6.1 TB/s
 * (counters: 537 MB read, 406 MB written, which is every input and output once).
 */
#include <type_traits>

#include "common.hpp"
#include "ofi_amd_hotpath.h"
#include "row_types.hpp"

namespace {

using namespace ofi_amd;

constexpr uint32_t kMaxWidth = 32768;
constexpr int kMostWaves = 16;
constexpr int kGradWaves = 8;
constexpr uint32_t kGradBlocks = 512;
constexpr uint32_t kFewRows = 256, kFewWaves = 16;
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

/*
 * Quotients by a scale, rounded as a division rounds them: the product with its inverse, and what that product leaves over times the
 * inverse once more, three operations where a division takes ten (16,384 rows of 8192 bfloat16 155.6 us, with the product alone 155.3;
 * thirty in a row on the same tensors, which the clocks give way to, 164 and 161).
 * An infinite scale leaves nothing over: the finite values beside it are 0.
 */
struct divisor_t {
	float inverse, finite;
};
__device__ __forceinline__ divisor_t divisor_of(float scale)
{
	return { 1.0f / scale, scale < __builtin_inff() ? scale : 0.0f };
}
__device__ __forceinline__ float quotient(float f, divisor_t by)
{
	const float q = f * by.inverse;
	return __builtin_fmaf(-__builtin_fmaf(q, by.finite, -f), by.inverse, q); /* so that -0 stays -0 */
}

/* A chunk's own elements, divided, as e4m3 */
template <bool STREAM, uint32_t V> __device__ __forceinline__ void store_q(uint8_t *p, uint32_t skip, const float (&f)[V], divisor_t by)
{
	if constexpr (V == 1) {
		if (skip == 0) {
			p[0] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(quotient(f[0], by), 0.0f, 0, false);
		}
	} else {
		typedef uint32_t words_t __attribute__((ext_vector_type(V / 4), aligned(1)));
		words_t w;
#pragma unroll
		for (uint32_t i = 0; i < V / 4; i++) {
			const int low = __builtin_amdgcn_cvt_pk_fp8_f32(quotient(f[4 * i], by), quotient(f[4 * i + 1], by), 0, false);
			w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(quotient(f[4 * i + 2], by), quotient(f[4 * i + 3], by), low, true);
		}
		if (skip == 0 && STREAM) {
			__builtin_nontemporal_store(w, reinterpret_cast<words_t *>(p));
		} else if (skip == 0) {
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
		uint32_t o = m;
		swap_rows16(m, o);
		m = max(m, o);
	}
	if (lanes >= 64) {
		uint32_t o = m;
		swap_halves(m, o);
		m = max(m, o);
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

/*
 * A row is held by the LANES lanes of a part of a wavefront, or (LANES 64) by the wavefronts along x, R chunks a lane.  sum may be x or
 * residual: a lane has read what it writes before any lane of its row writes.  group_lanes: lanes that share a scale, 0: the
 * whole row does.
 */
template <typename T, uint32_t V, int R, int LANES, flow_t FLOW>
__global__ __launch_bounds__(64 * kMostWaves) void rms_norm_kernel(const T *x, const T *residual, const void *__restrict__ gain,
								   uint64_t x_pitch, uint64_t residual_pitch, uint32_t first,
								   uint32_t n_rows, uint32_t width, float eps, uint32_t group_lanes,
								   bool gain_f32, norm_out_t o)
{
	const uint32_t B = LANES < 64 ? LANES : blockDim.x, waves = LANES < 64 ? 1 : blockDim.x >> 6;
	const uint32_t lane = LANES < 64 ? threadIdx.x & (LANES - 1) : threadIdx.x;
	__shared__ uint32_t part[2][LANES < 64 ? 1 : kMostWaves];
	const uint32_t wanted = LANES < 64 ? first + (blockIdx.x * blockDim.x + threadIdx.x) / LANES : first + blockIdx.x;
	const bool in = LANES == 64 || wanted < n_rows;
	const uint64_t row = in ? wanted : n_rows - 1;
	const T *xr = row_at(x, x_pitch, row), *rr = residual ? row_at(residual, residual_pitch, row) : nullptr;
	const uint32_t x_lag = lag_of<V>(xr), r_lag = lag_of<V>(rr);
	raw_t<T, V> c[R], d[R];
	uint32_t c_rest[R], d_rest[R];
#pragma unroll
	for (int k = 0; k < R; k++) {
		c[k] = load_raw<FLOW != STREAM_NONE, T, V>(xr + place_of<V>((k * B + lane) * V, width).from - x_lag);
	}
	if (rr) {
#pragma unroll
		for (int k = 0; k < R; k++) {
			d[k] = load_raw<FLOW != STREAM_NONE, T, V>(rr + place_of<V>((k * B + lane) * V, width).from - r_lag);
		}
	}
	if (x_lag) {
#pragma unroll
		for (int k = 0; k < R; k++) {
			c_rest[k] = load_rest<T, V, LANES>(xr + place_of<V>((k * B + lane) * V, width).from, x_lag, (k * B + lane) * V, width);
		}
	}
	if (r_lag) {
#pragma unroll
		for (int k = 0; k < R; k++) {
			d_rest[k] = load_rest<T, V, LANES>(rr + place_of<V>((k * B + lane) * V, width).from, r_lag, (k * B + lane) * V, width);
		}
	}
	float v[R][V];
	float squares = 0.0f;
#pragma unroll
	for (int k = 0; k < R; k++) {
		const uint32_t skip = place_of<V>((k * B + lane) * V, width).skip;
		catch_up<T, V, LANES>(c[k], c_rest[k], x_lag, (k * B + lane) * V, width);
		to_floats<T, V>(c[k], skip, v[k]);
		if (rr) {
			float f[V];
			catch_up<T, V, LANES>(d[k], d_rest[k], r_lag, (k * B + lane) * V, width);
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
	squares = LANES < 64 ? sum_over<LANES>(squares) : block_sum(squares, part[0], waves);
	const float rstd = 1.0f / __builtin_sqrtf(squares / (float)width + eps);
	if (o.rstd && in && lane == 0) {
		o.rstd[row] = rstd;
	}
	uint32_t most = 0;
#pragma unroll
	for (int k = 0; k < R; k++) {
		const uint32_t at = (k * B + lane) * V;
		const place_t here = place_of<V>(at, width);
		const bool mine = in && at < width;
		if (o.sum && mine) {
			store_piece<FLOW == STREAM_BOTH, T, V>(row_at(static_cast<T *>(o.sum), o.sum_pitch, row) + here.from, here.skip, v[k]);
		}
		float g[V];
		load_gain<T, V>(gain, gain_f32, here.from, g);
#pragma unroll
		for (uint32_t i = 0; i < V; i++) {
			v[k][i] = v[k][i] * rstd * g[i];
		}
		if (o.out && mine) {
			store_piece<FLOW == STREAM_BOTH, T, V>(row_at(static_cast<T *>(o.out), o.out_pitch, row) + here.from, here.skip, v[k]);
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
		if (mine) {
			store_q<FLOW == STREAM_BOTH, V>(o.q + row * o.q_pitch + here.from, here.skip, v[k], divisor_of(scale));
			const uint32_t chunk = k * B + lane;
			if ((chunk & (group_lanes - 1u)) == 0) {
				row_at(o.scale, o.scale_pitch, row)[chunk / group_lanes] = scale;
			}
		}
	}
	if (o.q && group_lanes == 0) {
		const float scale = scale_of(LANES < 64 ? max_bits_over<LANES>(most) : block_max_bits(most, part[1], waves));
		const divisor_t by = divisor_of(scale);
#pragma unroll
		for (int k = 0; k < R; k++) {
			const uint32_t at = (k * B + lane) * V;
			const place_t here = place_of<V>(at, width);
			if (in && at < width) {
				store_q<FLOW == STREAM_BOTH, V>(o.q + row * o.q_pitch + here.from, here.skip, v[k], by);
			}
		}
		if (in && lane == 0) {
			row_at(o.scale, o.scale_pitch, row)[0] = scale;
		}
	}
}

/*
 * dx = ds + rstd (g dn - h mean(g dn h)), h = s rstd; dg = sum over rows of dn h: each workgroup sums its own rows and the
 * partial sums are added up in the order of the workgroups, so that the result is the same every time.
 *
 * The wavefronts along x hold a row, a chunk a lane; a workgroup has blockDim.y rows at once and asks for the next
 * ones before it waits for the sum of these.  dx may be dout or dsum: a lane has read what it writes.
 *
 * Memory bounds it: 16,384 rows of 4096 bfloat16 with dsum, 537 MB, 88 us and 5 for the parts = 5.8 TB/s.  512 workgroups: with 384,
 * 768, 1024 of them 105, 105, 109 us in all for 97.  Two rows ahead were no faster (103), nor rows next to each other in a workgroup
 * (110).
 */
template <typename T, uint32_t V, int MOST, flow_t FLOW>
__global__ __launch_bounds__(64 * MOST)
void rms_norm_grad_kernel(const T *dout, const T *__restrict__ s, const float *__restrict__ rstds, const void *__restrict__ gain,
			  const T *dsum, uint64_t dout_pitch, uint64_t s_pitch, uint64_t dsum_pitch, uint32_t n_rows, uint32_t width,
			  bool gain_f32, T *dx, uint64_t dx_pitch, float *__restrict__ partial)
{
	__shared__ uint32_t part[2][kGradWaves][kMostWaves];
	__shared__ float others[MOST == kGradWaves ? (MOST - 1) * 64 * V : 1]; /* [row but the first][element][lane] */
	const uint32_t waves = blockDim.x >> 6, y = (uint32_t)__builtin_amdgcn_readfirstlane((int)threadIdx.y);
	const place_t here = place_of<V>(threadIdx.x * V, width);
	float g[V], dg[V];
	load_gain<T, V>(gain, gain_f32, here.from, g);
#pragma unroll
	for (uint32_t i = 0; i < V; i++) {
		dg[i] = 0.0f;
	}
	const uint32_t at = threadIdx.x * V;
	struct asked_t { /* a chunk on its way */
		raw_t<T, V> c;
		uint32_t rest, lag;
	} dc, sc, pc;
	float rstd = 0.0f;
	auto ask_one = [&](asked_t &a, const T *r) {
		a.lag = lag_of<V>(r);
		a.c = load_raw<FLOW != STREAM_NONE, T, V>(r + here.from - a.lag);
	};
	auto ask_rest = [&](asked_t &a, const T *r) { a.rest = load_rest<T, V, 64>(r + here.from, a.lag, at, width); };
	auto ask = [&](uint64_t row) {
		const T *dr = row_at(dout, dout_pitch, row), *sr = row_at(s, s_pitch, row);
		const T *pr = dsum ? row_at(dsum, dsum_pitch, row) : nullptr;
		ask_one(dc, dr);
		ask_one(sc, sr);
		if (pr) {
			ask_one(pc, pr);
		} else {
			pc.lag = 0;
		}
		if (dc.lag | sc.lag | pc.lag) {
			ask_rest(dc, dr);
			ask_rest(sc, sr);
			ask_rest(pc, pr);
		}
		rstd = rstds[row];
	};
	const uint64_t stride = (uint64_t)gridDim.x * blockDim.y;
	uint64_t row = (uint64_t)blockIdx.x * blockDim.y + y;
	if (row < n_rows) {
		ask(row);
	}
	uint32_t turn = 0;
	for (uint64_t first = (uint64_t)blockIdx.x * blockDim.y; first < n_rows; first += stride, row += stride, turn ^= 1u) {
		const bool in = row < n_rows;
		raw_t<T, V> p0 = pc.c;
		const float r0 = rstd;
		float d[V], h[V], along = 0.0f;
		if (in) {
			catch_up<T, V, 64>(dc.c, dc.rest, dc.lag, at, width);
			catch_up<T, V, 64>(sc.c, sc.rest, sc.lag, at, width);
			catch_up<T, V, 64>(p0, pc.rest, pc.lag, at, width);
			to_floats<T, V>(dc.c, here.skip, d);
			to_floats<T, V>(sc.c, here.skip, h);
#pragma unroll
			for (uint32_t i = 0; i < V; i++) {
				h[i] *= r0;
				dg[i] = __builtin_fmaf(d[i], h[i], dg[i]);
				d[i] *= g[i];
				along = i < here.skip ? along : __builtin_fmaf(d[i], h[i], along);
			}
			if (row + stride < n_rows) {
				ask(row + stride);
			}
		}
		const float mean = block_sum(along, part[turn][y], waves) / (float)width;
		if (in && threadIdx.x * V < width) {
			float r[V];
#pragma unroll
			for (uint32_t i = 0; i < V; i++) {
				r[i] = 0.0f;
			}
			if (dsum) {
				to_floats<T, V>(p0, 0, r);
			}
#pragma unroll
			for (uint32_t i = 0; i < V; i++) {
				r[i] = __builtin_fmaf(r0, __builtin_fmaf(-h[i], mean, d[i]), r[i]);
			}
			store_piece<FLOW == STREAM_BOTH, T, V>(row_at(dx, dx_pitch, row) + here.from, here.skip, r);
		}
	}
	if (!partial) {
		return;
	}
	if (MOST == kGradWaves && blockDim.y > 1) {
		float *o = others + threadIdx.x;
		if (y > 0) {
#pragma unroll
			for (uint32_t i = 0; i < V; i++) {
				o[((y - 1) * V + i) * blockDim.x] = dg[i];
			}
		}
		__syncthreads();
		if (y > 0) {
			return;
		}
		for (uint32_t k = 0; k + 1 < blockDim.y; k++) {
#pragma unroll
			for (uint32_t i = 0; i < V; i++) {
				dg[i] += o[(k * V + i) * blockDim.x];
			}
		}
	}
	if (threadIdx.x * V < width) {
		store_floats<V>(partial + (uint64_t)blockIdx.x * width + here.from, here.skip, dg);
	}
}

/*
 * The same for rows of more than 1024 chunks, R a lane, without the next row's beside them: 8192 rows of 16,384 bfloat16 217 us (5.0 TB/s).
 * KEPT: a row is held over its sum as it lies in memory (as floats it would not fit).  The longest rows, 32 values a lane, do not fit
 * beside their sums either way -- 2000 rows of 32,768 bfloat16 took 284 us so, and 639 with floats -- and are read again, out of
 * the caches: 159, and 4000 of 20,000, whose workgroups fit a CU twice if no lane holds gains, 170 for 216 (3000 of 24,000 floats
 * 292 for 287).
 */
template <int R, uint32_t V> constexpr bool kKept = R * V <= 16;
template <typename T, uint32_t V, int R, flow_t FLOW>
__global__ __launch_bounds__(64 * kMostWaves) void rms_norm_grad_wide_kernel(const T *dout, const T *s, const float *__restrict__ rstds,
								  const void *__restrict__ gain, const T *dsum, uint64_t dout_pitch,
								  uint64_t s_pitch, uint64_t dsum_pitch, uint32_t n_rows, uint32_t width,
								  bool gain_f32, T *dx, uint64_t dx_pitch, float *__restrict__ partial)
{
	__shared__ uint32_t part[2][kMostWaves];
	float dg[R][V];
#pragma unroll
	for (int k = 0; k < R; k++) {
#pragma unroll
		for (uint32_t i = 0; i < V; i++) {
			dg[k][i] = 0.0f;
		}
	}
	uint32_t turn = 0;
	for (uint64_t row = blockIdx.x; row < n_rows; row += gridDim.x, turn ^= 1u) {
		constexpr int H = kKept<R, V> ? R : 1; /* chunks held */
		raw_t<T, V> dc[H], sc[H];
		auto ask = [&](int k, int slot) {
			const uint32_t from = place_of<V>((k * blockDim.x + threadIdx.x) * V, width).from;
			dc[slot] = load_raw<FLOW != STREAM_NONE, T, V>(row_at(dout, dout_pitch, row) + from);
			sc[slot] = load_raw<FLOW != STREAM_NONE, T, V>(row_at(s, s_pitch, row) + from);
		};
		const float rstd = rstds[row];
		const void *gains = gain;
		if constexpr (!kKept<R, V>) {
			asm volatile("" : "+s"(gains)); /* read with every row: held over them they cost the second workgroup of a CU */
		}
		float along = 0.0f;
		auto sum = [&](int k, int slot) {
			const place_t here = place_of<V>((k * blockDim.x + threadIdx.x) * V, width);
			float g[V], d[V], h[V];
			to_floats<T, V>(dc[slot], here.skip, d);
			to_floats<T, V>(sc[slot], here.skip, h);
			load_gain<T, V>(gains, gain_f32, here.from, g);
#pragma unroll
			for (uint32_t i = 0; i < V; i++) {
				along = i < here.skip ? along : __builtin_fmaf(d[i] * g[i], h[i] * rstd, along);
			}
		};
		if constexpr (kKept<R, V>) {
#pragma unroll
			for (int k = 0; k < R; k++) {
				ask(k, k);
			}
#pragma unroll
			for (int k = 0; k < R; k++) {
				sum(k, k);
				asm volatile("" : "+v"(dc[k]), "+v"(sc[k])); /* nothing made of them is kept */
			}
		} else {
#pragma unroll 1
			for (int k = 0; k < R; k++) {
				ask(k, 0);
				sum(k, 0);
			}
		}
		const float mean = block_sum(along, part[turn], blockDim.x >> 6) / (float)width;
#pragma unroll
		for (int k = 0; k < R; k++) {
			const uint32_t at = (k * blockDim.x + threadIdx.x) * V;
			if (at < width) {
				const place_t here = place_of<V>(at, width);
				float g[V], d[V], h[V], r[V];
				const int slot = kKept<R, V> ? k : 0;
				if (!kKept<R, V>) {
					ask(k, slot);
				}
				to_floats<T, V>(dc[slot], here.skip, d);
				to_floats<T, V>(sc[slot], here.skip, h);
				load_gain<T, V>(gains, gain_f32, here.from, g);
#pragma unroll
				for (uint32_t i = 0; i < V; i++) {
					r[i] = 0.0f;
				}
				if (dsum) {
					to_floats<T, V>(load_raw<FLOW != STREAM_NONE, T, V>(row_at(dsum, dsum_pitch, row) + here.from), 0, r);
				}
#pragma unroll
				for (uint32_t i = 0; i < V; i++) {
					h[i] *= rstd;
					dg[k][i] = __builtin_fmaf(d[i], h[i], dg[k][i]);
					r[i] = __builtin_fmaf(rstd, __builtin_fmaf(-h[i], mean, d[i] * g[i]), r[i]);
				}
				store_piece<FLOW == STREAM_BOTH, T, V>(row_at(dx, dx_pitch, row) + here.from, here.skip, r);
			}
		}
	}
#pragma unroll
	for (int k = 0; k < R; k++) {
		const uint32_t at = (k * blockDim.x + threadIdx.x) * V;
		if (partial && at < width) {
			const place_t here = place_of<V>(at, width);
			store_floats<V>(partial + (uint64_t)blockIdx.x * width + here.from, here.skip, dg[k]);
		}
	}
}

/*
 * Few rows, in one launch: rstd is an input, so that dg needs nothing of dx.  The first n_rows workgroups make a row of dx each, those
 * behind them 64 columns of dg, their wavefronts at the rows by turns.  They read dout too, so that dx may not be dout.  Rows of 4096
 * bfloat16, us a call in one launch and in two: 1 to 128 rows 10.0 and 13.9, 256 10.4 and 13.8, 384 12.0 and 13.8, 512 17 and 13.7.
 */
template <typename T, uint32_t V>
__global__ __launch_bounds__(64 * kMostWaves) void rms_norm_grad_few_kernel(const T *__restrict__ dout, const T *__restrict__ s,
									    const float *__restrict__ rstds, const void *__restrict__ gain,
									    const T *dsum, uint64_t dout_pitch, uint64_t s_pitch,
									    uint64_t dsum_pitch, uint32_t n_rows, uint32_t width,
									    bool gain_f32, T *dx, uint64_t dx_pitch,
									    float *__restrict__ dgain)
{
	__shared__ float sums[kMostWaves][64];
	__shared__ uint32_t part[kMostWaves];
	const uint32_t waves = blockDim.x >> 6;
	if (blockIdx.x < n_rows) {
		const uint64_t row = blockIdx.x;
		const uint32_t at = threadIdx.x * V;
		const place_t here = place_of<V>(at, width);
		const raw_t<T, V> dc = load_raw<false, T, V>(row_at(dout, dout_pitch, row) + here.from);
		const raw_t<T, V> sc = load_raw<false, T, V>(row_at(s, s_pitch, row) + here.from);
		raw_t<T, V> pc = dc;
		if (dsum) {
			pc = load_raw<false, T, V>(row_at(dsum, dsum_pitch, row) + here.from);
		}
		const float rstd = rstds[row];
		float g[V], d[V], h[V], along = 0.0f;
		load_gain<T, V>(gain, gain_f32, here.from, g);
		to_floats<T, V>(dc, here.skip, d);
		to_floats<T, V>(sc, here.skip, h);
#pragma unroll
		for (uint32_t i = 0; i < V; i++) {
			h[i] *= rstd;
			d[i] *= g[i];
			along = i < here.skip ? along : __builtin_fmaf(d[i], h[i], along);
		}
		const float mean = block_sum(along, part, waves) / (float)width;
		if (at < width) {
			float r[V];
			to_floats<T, V>(pc, 0, r);
#pragma unroll
			for (uint32_t i = 0; i < V; i++) {
				r[i] = __builtin_fmaf(rstd, __builtin_fmaf(-h[i], mean, d[i]), dsum ? r[i] : 0.0f);
			}
			store_piece<false, T, V>(row_at(dx, dx_pitch, row) + here.from, here.skip, r);
		}
		return;
	}
	const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, column = (blockIdx.x - n_rows) * 64u + lane;
	float total = 0.0f;
	if (column < width) {
#pragma unroll 8
		for (uint32_t row = wave; row < n_rows; row += waves) {
			total = __builtin_fmaf((float)row_at(dout, dout_pitch, row)[column], (float)row_at(s, s_pitch, row)[column] * rstds[row], total);
		}
	}
	sums[wave][lane] = total;
	__syncthreads();
	if (wave == 0 && column < width) {
		for (uint32_t w = 1; w < waves; w++) {
			total += sums[w][lane];
		}
		dgain[column] = total;
	}
}

/* kGainColumns columns of a workgroup, its lanes at the parts by turns, with all of their loads on the way at once: 5 us for 512 parts of
 * 4096 (64 columns 5.5), most of it the way of fresh lines from the other dies */
constexpr uint32_t kGainColumns = 32, kGainTurns = 1024 / kGainColumns, kPartsOfLane = kGradBlocks / kGainTurns;
static_assert(kGradBlocks % kGainTurns == 0, "all parts are added");
__global__ __launch_bounds__(1024) void rms_norm_gain_kernel(const float *__restrict__ partial, float *__restrict__ dgain, uint32_t parts,
							     uint32_t width)
{
	__shared__ float sums[kGainTurns][kGainColumns];
	const uint32_t x = threadIdx.x % kGainColumns, turn = threadIdx.x / kGainColumns, column = blockIdx.x * kGainColumns + x;
	float total = 0.0f;
	if (column < width && turn < parts) {
		float f[kPartsOfLane];
#pragma unroll
		for (uint32_t p = 0; p < kPartsOfLane; p++) {
			f[p] = partial[(uint64_t)min(turn + p * kGainTurns, parts - 1) * width + column];
		}
#pragma unroll
		for (uint32_t p = 0; p < kPartsOfLane; p++) {
			total += turn + p * kGainTurns < parts ? f[p] : 0.0f;
		}
	}
	sums[turn][x] = total;
	__syncthreads();
	if (turn == 0 && column < width) {
#pragma unroll
		for (uint32_t t = 1; t < kGainTurns; t++) {
			total += sums[t][x];
		}
		dgain[column] = total;
	}
}

/* Workgroups of the gradient */
inline uint32_t grad_blocks(uint32_t n_rows)
{
	return n_rows < kGradBlocks ? n_rows : kGradBlocks;
}

/* Calls f with the chunks of a lane, at least `least`, for which a row of `chunks` has a lane of a workgroup of the most wavefronts */
template <uint32_t V, typename F> void with_chunks_of_lane(uint32_t chunks, uint32_t least, F f)
{
	constexpr uint32_t lanes = 64 * kMostWaves;
	if constexpr (V == 1) {
		f(std::integral_constant<int, 1>{});
	} else if (chunks <= lanes && least <= 1) {
		f(std::integral_constant<int, 1>{});
	} else if (chunks <= 2 * lanes) {
		f(std::integral_constant<int, 2>{});
	} else if (V == 8 || chunks <= 4 * lanes) {
		f(std::integral_constant<int, 4>{});
	} else {
		f(std::integral_constant<int, V == 8 ? 4 : 8>{});
	}
}

/*
 * Chunks of a lane of the norm.  One where the rows have no more chunks than the chip has lanes (256 units of 2048): the most
 * wavefronts, the shortest wait.  Beyond, two: half the wavefronts for each sum.  Rows of 4096 and 8192 bfloat16 to e4m3 by us with
 * one / two: 1 row 2.6 / 3.6 and 3.1 / 3.8; 256 rows 4.1 / 5.0 and 5.4 / 6.0; 1024 rows 8.6 / 9.3 and 14.0 / 13.5; 8192 rows
 * 44.7 / 44.0 and 91.3 / 80.6; 16,384 rows 82.3 / 79.1 and 176 / 158 (three to four: 82.8 and 162).
 */
inline uint32_t least_chunks(uint32_t n_rows, uint32_t chunks)
{
	return chunks > 64 && (uint64_t)n_rows * chunks > (1u << 19) ? 2 : 1;
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
	const flow_t flow = flow_of(n_rows * (bytes * (1u + !!d_residual + !!d_sum + !!d_out) + (d_q ? width : 0)));
	with_row_type(type, width, [&](auto element, auto v) {
		using T = decltype(element);
		constexpr uint32_t V = decltype(v)::value;
		const uint32_t chunks = (width + V - 1) / V;
		const uint32_t group_lanes = group >= width ? 0 : group / V; /* a row within one group is one */
		auto launch = [&](auto kernel, uint32_t rows, uint32_t lanes) { /* workgroups of so many rows and lanes */
			for (uint32_t first = 0; first < n_rows; first += kRowsOfLaunch) {
				const uint32_t n = n_rows - first < kRowsOfLaunch ? n_rows - first : kRowsOfLaunch;
				launch_kernel(kernel, dim3((n + rows - 1) / rows), dim3(lanes), 0, as_stream(stream), static_cast<const T *>(d_x),
					      static_cast<const T *>(d_residual), d_gain, x_pitch, residual_pitch, first, n_rows, width, eps,
					      group_lanes, gain_type == OFI_AMD_FLOAT32, o);
			}
		};
		/* narrow rows share a wavefront: 30,000 rows of 256 bfloat16 to e4m3 15.9 us with one to each, 12.8 with two */
		if (chunks <= 16) {
			launch(by_flow(flow, rms_norm_kernel<T, V, 1, 16, STREAM_NONE>, rms_norm_kernel<T, V, 1, 16, STREAM_LOADS>,
				       rms_norm_kernel<T, V, 1, 16, STREAM_BOTH>), 16, 256);
		} else if (chunks <= 32) {
			launch(by_flow(flow, rms_norm_kernel<T, V, 1, 32, STREAM_NONE>, rms_norm_kernel<T, V, 1, 32, STREAM_LOADS>,
				       rms_norm_kernel<T, V, 1, 32, STREAM_BOTH>), 8, 256);
		} else {
			with_chunks_of_lane<V>(chunks, least_chunks(n_rows, chunks), [&](auto r) {
				constexpr int R = decltype(r)::value;
				launch(by_flow(flow, rms_norm_kernel<T, V, R, 64, STREAM_NONE>, rms_norm_kernel<T, V, R, 64, STREAM_LOADS>,
					       rms_norm_kernel<T, V, R, 64, STREAM_BOTH>), 1, (chunks + 64 * R - 1) / (64 * R) * 64);
			});
		}
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
	const uint32_t size_chunk = width >= 16 / size ? 16 / size : 1, all_chunks = (width + size_chunk - 1) / size_chunk;
	if (d_dgain && n_rows != 0 && n_rows <= kFewRows && all_chunks <= 64 * kMostWaves && d_dx != d_dout) {
		with_row_type(type, width, [&](auto element, auto v) {
			using T = decltype(element);
			const uint32_t waves = (all_chunks + 63) / 64;
			launch_kernel(rms_norm_grad_few_kernel<T, decltype(v)::value>, dim3(n_rows + (width + 63) / 64),
				      dim3(64 * (waves < kFewWaves ? kFewWaves : waves)), 0, as_stream(stream), static_cast<const T *>(d_dout),
				      static_cast<const T *>(d_s), d_rstd, d_gain, static_cast<const T *>(d_dsum), dout_pitch, s_pitch, dsum_pitch,
				      n_rows, width, gain_type == OFI_AMD_FLOAT32, static_cast<T *>(d_dx), dx_pitch, d_dgain);
		});
		OFI_AMD_HIP_TRY(hipGetLastError());
		return 0;
	}
	const uint32_t blocks = grad_blocks(n_rows);
	float *partial = d_dgain ? static_cast<float *>(d_work) : nullptr;
	if (n_rows != 0) {
		const flow_t flow = flow_of(n_rows * bytes * (3u + !!d_dsum));
		with_row_type(type, width, [&](auto element, auto v) {
			using T = decltype(element);
			constexpr uint32_t V = decltype(v)::value;
			auto launch = [&](auto kernel, dim3 block) {
				launch_kernel(kernel, dim3(blocks), block, 0, as_stream(stream), static_cast<const T *>(d_dout),
					      static_cast<const T *>(d_s), d_rstd, d_gain, static_cast<const T *>(d_dsum), dout_pitch, s_pitch,
					      dsum_pitch, n_rows, width, gain_type == OFI_AMD_FLOAT32, static_cast<T *>(d_dx), dx_pitch, partial);
			};
			const uint32_t chunks = (width + V - 1) / V, waves = (chunks + 63) / 64;
			with_chunks_of_lane<V>(chunks, 1, [&](auto r) {
				constexpr int R = decltype(r)::value;
				if constexpr (R > 1) {
					const dim3 lanes(64 * ((waves + R - 1) / R));
					if constexpr (kKept<R, V>) {
						launch(by_flow(flow, rms_norm_grad_wide_kernel<T, V, R, STREAM_NONE>,
							       rms_norm_grad_wide_kernel<T, V, R, STREAM_LOADS>,
							       rms_norm_grad_wide_kernel<T, V, R, STREAM_BOTH>),
						       lanes);
					} else {
						launch(rms_norm_grad_wide_kernel<T, V, R, STREAM_NONE>, lanes);
					}
				} else if (waves > (uint32_t)kGradWaves) {
					launch(by_flow(flow, rms_norm_grad_kernel<T, V, kMostWaves, STREAM_NONE>,
						       rms_norm_grad_kernel<T, V, kMostWaves, STREAM_LOADS>,
						       rms_norm_grad_kernel<T, V, kMostWaves, STREAM_BOTH>),
					       dim3(64 * waves));
				} else {
					/* rows of a workgroup at once, so that it has eight wavefronts (30,000 rows of 1024 bfloat16 60.2 us with
					 * one row, 43.8 with four), but fewer where that would leave workgroups without any */
					const uint32_t most = kGradWaves / waves, each = (n_rows + kGradBlocks - 1) / kGradBlocks;
					launch(by_flow(flow, rms_norm_grad_kernel<T, V, kGradWaves, STREAM_NONE>,
						       rms_norm_grad_kernel<T, V, kGradWaves, STREAM_LOADS>,
						       rms_norm_grad_kernel<T, V, kGradWaves, STREAM_BOTH>),
					       dim3(64 * waves, each < most ? each : most));
				}
			});
		});
	}
	if (d_dgain) { /* of no rows: zeros */
		launch_kernel(rms_norm_gain_kernel, dim3((width + kGainColumns - 1) / kGainColumns), dim3(1024), 0, as_stream(stream), partial,
			      d_dgain, blocks, width);
	}
	OFI_AMD_HIP_TRY(hipGetLastError());
	return 0;
}

} /* extern "C" */
