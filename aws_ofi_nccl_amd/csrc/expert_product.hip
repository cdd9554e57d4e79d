/*
 * Products of rows sorted by expert with their expert's weights:
 *   gated      h = act(x G^T) (x U^T), both projections in one kernel, and what the activation was taken of kept for the way back
 *   product    y = act(x W^T + b) + r
 * x and the weights run along the summed axis.  Rows of e4m3 and their weights have a scale for every 128 of it, which are what one
 * step sums: a step's sums are multiplied by both scales in 32 bits and added.  Their products run as float16, which holds every e4m3 value: both 8-bit
 * matrix instructions, of 32 and of 128 summed values, keep sums of about 16 bits (normal values: 1.5e-5 off, as float16 1e-8 to 8e-8).
 * Bound by the matrix cores: 32,768 rows of 32 experts, bfloat16, gated 4096 to 2048 with a checkpoint of 8 bits 1080 us (1,018 TFLOP/s), product 2048 to
 * 4096 575 us (956); one expert, 8192 rows, 4096 to 4096 with bias, gelu and residual 267 us (1,030); 16,384 rows in 8 bits, gated 4096 to 2048
 * into 8 bits 612 us (898).  A step of a tile of 256 x 256 is 1.6 us, 1,340 TFLOP/s; besides, a tile costs 11.5 us and an
 * expert's last one may be part of one.
 */
#include "expert_forward.hpp"

namespace ofi_amd {
namespace {

struct forward_args_t {
	rows_t of;
	const uint8_t *x, *w;
	uint64_t x_pitch, w_pitch, expert_pitch;
	uint32_t width, n, first_tile;
	forward_t o;
};

template <typename T, uint32_t BM, uint32_t THREADS> struct forward_operands_t {
	along_t<T, BM, THREADS> rows;
	along_t<T, kBlock, THREADS> part0, part1;
	const uint8_t *scale; /* of the first row, for 8-bit ones: one word of each row in a step */
	uint32_t scale_pitch;
	forward_tile_t place;
	static constexpr bool kScaled = sizeof(T) == 1;
	static constexpr uint32_t kRowsBytes = decltype(rows)::kBytes, kPartBytes = decltype(part0)::kBytes, kScalesAt = kRowsBytes + 2 * kPartBytes;
	static constexpr uint32_t kBytes = kScalesAt + (kScaled ? BM * 4 : 0);
	static constexpr uint32_t kFills = decltype(rows)::kChunks + 2 * decltype(part0)::kChunks + (kScaled ? 1 : 0);

	/* direct: a part without columns is not read; else the first column stands for them */
	__device__ __forceinline__ void set(const forward_args_t *a, const tile_t &tile, bool direct)
	{
		const bool gated = a->o.gated;
		const uint32_t n = a->n, c0 = tile.nt * (gated ? kBlock : 2 * kBlock), c1 = gated ? c0 : c0 + kBlock;
		const uint32_t there0 = n - c0 < kBlock ? n - c0 : kBlock, there1 = c1 >= n ? 0 : n - c1 < kBlock ? n - c1 : kBlock;
		const uint8_t *const weights = a->w + tile.expert * a->expert_pitch;
		const int64_t bytes = (int64_t)a->width * sizeof(T);
		place = { tile.from, tile.rows, c0, c1, there0, there1, n, tile.expert };
		rows.set(a->x + tile.from * a->x_pitch, a->x_pitch, tile.rows, bytes);
		part0.set(weights + c0 * a->w_pitch, a->w_pitch, there0, bytes);
		if (kScaled) {
			scale = reinterpret_cast<const uint8_t *>(row_at(a->o.scale, a->o.scale_pitch, tile.from));
			scale_pitch = (uint32_t)a->o.scale_pitch;
		}
		part1.set(weights + (there1 ? (gated ? (uint64_t)n : 0) + c1 : 0) * a->w_pitch, a->w_pitch, there1 || direct ? there1 : 1, bytes);
	}
	__device__ __forceinline__ void load(uint32_t step)
	{
		rows.load(step);
		part0.load(step);
		part1.load(step);
	}
	__device__ __forceinline__ void store(uint32_t step, uint8_t *to) const
	{
		rows.store(step, to);
		part0.store(step, to + kRowsBytes);
		part1.store(step, to + kRowsBytes + kPartBytes);
	}
	__device__ __forceinline__ void fill(uint32_t step, uint8_t *to) const
	{
		rows.fill(step, to);
		part0.fill(step, to + kRowsBytes);
		part1.fill(step, to + kRowsBytes + kPartBytes);
		if (kScaled) { /* every wavefront has one, so that all count alike: they are as many times BM / 64 */
			const uint32_t some = uniform(threadIdx.x >> 6) % (BM / 64) * 64, r = some + (threadIdx.x & 63u);
			const int bytes = (int)((place.rows - 1) * scale_pitch) + 4;
			words_to_lds(scale + step * 4, step * kStepBytes < (uint32_t)rows.bytes ? bytes : 0, r * scale_pitch, to + kScalesAt + some * 4);
		}
	}
};

/* sums += all steps of 8-bit rows, each with its scales: sum_steps without fragments on their way, for want of registers.  The rows' scales come
 * with the tile, so that no load of a lane's own is waited for, which would wait for the tiles on their way. */
template <uint32_t WM, uint32_t WN, uint32_t MF, bool DIRECT, uint32_t STAGES, typename Operands>
__device__ __forceinline__ void sum_scaled_steps(f32x4_t (&sums)[MF][2][8 / WN], uint32_t steps, uint8_t *lds, Operands &of)
{
	constexpr uint32_t G = 8 / WN;
	const uint32_t lane = threadIdx.x & 63u, wave = uniform(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
	const along_frag_t row_frag(wm * 16 * MF, lane), column_frag(wn * 16 * G, lane);
	const forward_args_t *const a = argument<forward_args_t>();
	const forward_tile_t &place = of.place;
	const float *row_scale[MF], *weight_scale[2];
	const uint32_t k_blocks = blocks_of(a->width), n_blocks = blocks_of(place.n);
	const float *const of_expert = a->o.weight_scale + (uint64_t)place.expert * (a->o.gated ? 2 : 1) * n_blocks * k_blocks;
	weight_scale[0] = of_expert + (uint64_t)(place.c0 / kBlock) * k_blocks;
	weight_scale[1] = place.there1 ? of_expert + (uint64_t)((a->o.gated ? n_blocks : 0) + place.c1 / kBlock) * k_blocks : weight_scale[0];
	float row_next[MF], weight_next[2];
	auto scales_of = [&](uint32_t step) __attribute__((always_inline)) {
		if (!DIRECT) {
#pragma unroll
			for (int m = 0; m < (int)MF; m++) {
				row_next[m] = row_scale[m][step];
			}
		}
		weight_next[0] = weight_scale[0][step];
		weight_next[1] = weight_scale[1][step];
	};
	if (DIRECT) {
#pragma unroll
		for (uint32_t s = 0; s + 1 < STAGES; s++) {
			of.fill(s, lds + s * Operands::kBytes);
		}
	} else {
#pragma unroll
		for (int m = 0; m < (int)MF; m++) {
			const uint32_t r = (wm * MF + m) * 16 + (lane & 15u);
			row_scale[m] = row_at(a->o.scale, a->o.scale_pitch, place.from + (r < place.rows ? r : place.rows - 1));
		}
		of.load(0);
	}
	scales_of(0);
	uint32_t at = 0;
	for (uint32_t step = 0; step < steps; step++) {
		uint8_t *const now = lds + at, *const last = lds + (at ? at - Operands::kBytes : (STAGES - 1) * Operands::kBytes);
		at = at + Operands::kBytes < STAGES * Operands::kBytes ? at + Operands::kBytes : 0;
		if (DIRECT) {
			landed<(STAGES - 2) * Operands::kFills>();
		} else {
			of.store(step, now);
		}
		workgroup_meets<DIRECT>(); /* this tile is there, and the last one's readers are past it */
		float by[MF][2];
#pragma unroll
		for (int m = 0; m < (int)MF; m++) {
			const float s = DIRECT ? reinterpret_cast<const float *>(now + Operands::kScalesAt)[(wm * MF + m) * 16 + (lane & 15u)] : row_next[m];
			by[m][0] = s * weight_next[0];
			by[m][1] = s * weight_next[1];
		}
		if (step + 1 < steps) {
			scales_of(step + 1);
			if (!DIRECT) {
				of.load(step + 1);
			}
		}
		if (DIRECT) {
			of.fill(step + STAGES - 1, last);
		}
		u32x4_t r[MF][4];
#pragma unroll
		for (int m = 0; m < (int)MF; m++) {
#pragma unroll
			for (uint32_t half = 0; half < 2; half++) {
				const u32x4_t q = row_frag.get(now, m * 16, half);
				r[m][2 * half] = widened(q.x, q.y);
				r[m][2 * half + 1] = widened(q.z, q.w);
			}
		}
#pragma unroll
		for (int j = 0; j < (int)(2 * G); j++) {
			const uint8_t *const columns = now + Operands::kRowsBytes;
			const u32x4_t q0 = column_frag.get(columns, j / G * kBlock + j % G * 16, 0);
			const u32x4_t q1 = column_frag.get(columns, j / G * kBlock + j % G * 16, 1);
			const u32x4_t c[4] = { widened(q0.x, q0.y), widened(q0.z, q0.w), widened(q1.x, q1.y), widened(q1.z, q1.w) };
			f32x4_t part[MF] = {};
#pragma unroll
			for (int k = 0; k < 4; k++) {
#pragma unroll
				for (int m = 0; m < (int)MF; m++) {
					part[m] = multiply<f16_t>(c[k], r[m][k], part[m]);
				}
			}
#pragma unroll
			for (int m = 0; m < (int)MF; m++) {
				f32x4_t &to = sums[m][j / G][j % G];
#pragma unroll
				for (int i = 0; i < 4; i++) {
					to[i] = __builtin_fmaf(part[m][i], by[m][j / G], to[i]);
				}
			}
		}
	}
	if (DIRECT) {
		landed<0>(); /* what follows writes there */
	}
}

template <typename T, uint32_t WM, uint32_t WN, uint32_t MF, bool DIRECT>
__global__ __launch_bounds__(64 * WM * WN) void expert_forward_kernel(forward_args_t)
{
	constexpr uint32_t BM = 16 * MF * WM, THREADS = 64 * WM * WN, G = 8 / WN;
	constexpr bool SCALED = sizeof(T) == 1;
	using operands_t = forward_operands_t<T, BM, THREADS>;
	constexpr uint32_t kStages = DIRECT && WM < 4 ? 3 : 2;
	__shared__ __attribute__((aligned(1024))) uint8_t lds[kStages * operands_t::kBytes];

	operands_t of;
	uint32_t steps;
	{
		const forward_args_t *const a = argument<forward_args_t>();
		steps = (a->width + kStepOf<T> - 1) / kStepOf<T>;
		const tile_t tile = find_tile<BM>(a->of, a->first_tile + blockIdx.x);
		if (!tile.any) {
			return;
		}
		of.set(a, tile, DIRECT);
	}
	const uint32_t lane = threadIdx.x & 63u, wave = uniform(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
	f32x4_t sums[MF][2][G] = {};
	if constexpr (SCALED) {
		sum_scaled_steps<WM, WN, MF, DIRECT, kStages>(sums, steps, lds, of);
	} else {
		sum_steps<T, DIRECT, kStages, operands_t::kFills>(
			sums, wm * 16 * MF < of.place.rows, steps, lds, operands_t::kBytes, operands_t::kRowsBytes, along_frag_t(wm * 16 * MF, lane),
			along_frag_t(wn * 16 * G, lane), [&](uint32_t step, uint8_t *to) __attribute__((always_inline)) { of.fill(step, to); },
			[&](uint32_t step) __attribute__((always_inline)) { of.load(step); },
			[&](uint32_t step, uint8_t *to) __attribute__((always_inline)) { of.store(step, to); }, [](const u32x4_t(&)[MF]) {});
	}
	const forward_tile_t place = of.place;
	for_rows<WM, WN, MF, false>(
		sums, lds, place.rows == BM && place.there0 == kBlock && place.there1 == kBlock,
		[&](auto all, uint32_t r, uint32_t part_lane) __attribute__((always_inline)) {
			return forward_load<decltype(all)::value>(argument<forward_args_t>()->o, place, r, part_lane * 8);
		},
		[&](auto all, uint32_t r, uint32_t part_lane, f32x8_t p0, f32x8_t p1, const forward_in_t &in) __attribute__((always_inline)) {
			forward_finish<decltype(all)::value>(argument<forward_args_t>()->o, place, r, part_lane * 8, p0, p1, in);
		});
}

int forward(const void *d_rows, uint64_t rows_pitch, int type, const int32_t *d_offset, uint32_t n_experts, uint32_t max_rows,
	    const void *d_weight, uint64_t weight_pitch, uint64_t expert_pitch, uint32_t width, uint32_t n, const forward_t &o, void *stream)
{
	const uint64_t bytes = (uint64_t)width * product_type_size(type);
	const bool direct = in_chunks(d_rows, rows_pitch, bytes) && in_chunks(d_weight, weight_pitch, bytes) && expert_pitch % 16 == 0 &&
			    (type != OFI_AMD_E4M3 || o.scale_pitch <= kMostPitch);
	const uint32_t n_tiles = (n + (o.gated ? kBlock : 2 * kBlock) - 1) / (o.gated ? kBlock : 2 * kBlock);
	const uint32_t bm = row_tile_for(max_rows, n_experts, n_tiles, direct);
	if (forward_is_few(max_rows, n_experts, n_tiles)) {
		return forward_few(d_rows, rows_pitch, type, d_offset, n_experts, max_rows, d_weight, weight_pitch, expert_pitch, width, n, o, stream);
	}
	const uint64_t tiles = most_row_tiles(max_rows, n_experts, bm) * n_tiles;
	if (tiles > 0x7fffffffull) {
		return -E2BIG;
	}
	forward_args_t args = { { d_offset, n_experts, max_rows, n_tiles }, static_cast<const uint8_t *>(d_rows), static_cast<const uint8_t *>(d_weight),
				rows_pitch, weight_pitch, expert_pitch, width, n, 0, o };
	auto with = [&](auto element) {
		using T = decltype(element);
		auto kernel = direct ? (bm == 256 ? expert_forward_kernel<T, 4, 2, 4, true>
						: bm == 128 ? expert_forward_kernel<T, 2, 4, 4, true> : expert_forward_kernel<T, 1, 8, 4, true>)
				     : bm == 128 ? expert_forward_kernel<T, 2, 4, 4, false> : expert_forward_kernel<T, 1, 8, 4, false>;
		launch_tiles(tiles, 512, [&](uint32_t first, uint32_t count) {
			args.first_tile = first;
			return launch_kernel(kernel, dim3(count), dim3(512), 0, as_stream(stream), args);
		});
	};
	if (type == OFI_AMD_BFLOAT16) {
		with(bf16_t{});
	} else if (type == OFI_AMD_FLOAT16) {
		with(f16_t{});
	} else {
		with(e4m3_t{});
	}
	OFI_AMD_HIP_TRY(hipGetLastError());
	return 0;
}

/* Rows that are written: `columns` values in parts of n */
bool output_ok(const matrix_t &m, uint64_t rows, uint32_t n, uint32_t parts)
{
	const uint32_t size = product_type_size(m.type);
	return size && rows_ok(m.p, m.pitch, rows, (uint64_t)parts * n * size, size) &&
	       (m.type != OFI_AMD_E4M3 || scales_ok(m.scale, m.scale_pitch, rows, parts * blocks_of(n)));
}

matrix_t matrix(void *p, uint64_t pitch, int type, float *scale, uint64_t scale_pitch)
{
	return { static_cast<uint8_t *>(p), pitch, type, scale, scale_pitch };
}

/* 16-bit rows have 16-bit outputs of their own type or 8-bit ones; 8-bit rows have any */
bool types_fit(int type, int other) { return product_type_size(other) && (type == OFI_AMD_E4M3 || other == OFI_AMD_E4M3 || other == type); }

} // namespace
} // namespace ofi_amd

using namespace ofi_amd;

extern "C" {

int ofi_amd_expert_gated(const void *d_rows, uint64_t rows_pitch, const float *d_scale, uint64_t scale_pitch, int type, const int32_t *d_offset,
			 uint32_t n_experts, uint32_t max_rows, const void *d_weight, uint64_t weight_pitch, uint64_t expert_pitch,
			 const float *d_weight_scale, uint32_t width, uint32_t inner, int activation, void *d_out, uint64_t out_pitch,
			 int out_type, float *d_out_scale, uint64_t out_scale_pitch, void *d_saved, uint64_t saved_pitch, int saved_type,
			 float *d_saved_scale, uint64_t saved_scale_pitch, void *stream)
{
	int rc = require_device();
	if (rc != 0) {
		return rc;
	}
	const uint32_t size = product_type_size(type);
	if (!size || !activation_ok(activation) || !types_fit(type, out_type) || (d_saved && !types_fit(type, saved_type))) {
		return -EINVAL;
	}
	rc = check_experts(d_offset, n_experts, max_rows, width, inner);
	if (rc != 0 || max_rows == 0) {
		return rc;
	}
	forward_t o = {};
	o.scale = d_scale;
	o.scale_pitch = scale_pitch;
	o.weight_scale = d_weight_scale;
	o.activation = activation;
	o.gated = true;
	o.out = matrix(d_out, out_pitch, out_type, d_out_scale, out_scale_pitch);
	o.saved = matrix(d_saved, saved_pitch, saved_type, d_saved_scale, saved_scale_pitch);
	if (!rows_ok(d_rows, rows_pitch, max_rows, (uint64_t)width * size, size) ||
	    !stack_ok(d_weight, weight_pitch, expert_pitch, n_experts, 2ull * inner, (uint64_t)width * size, size) ||
	    !output_ok(o.out, max_rows, inner, 1) || (d_saved && !output_ok(o.saved, max_rows, inner, 2)) ||
	    (type == OFI_AMD_E4M3 && (!scales_ok(d_scale, scale_pitch, max_rows, blocks_of(width)) || !scales_ok(d_weight_scale, 4, 1, 1)))) {
		return -EINVAL;
	}
	return forward(d_rows, rows_pitch, type, d_offset, n_experts, max_rows, d_weight, weight_pitch, expert_pitch, width, inner, o, stream);
}

int ofi_amd_expert_product(const void *d_rows, uint64_t rows_pitch, const float *d_scale, uint64_t scale_pitch, int type,
			   const int32_t *d_offset, uint32_t n_experts, uint32_t max_rows, const void *d_weight, uint64_t weight_pitch,
			   uint64_t expert_pitch, const float *d_weight_scale, uint32_t width, uint32_t out_width, const void *d_bias,
			   int bias_type, int activation, const void *d_residual, uint64_t residual_pitch, void *d_out, uint64_t out_pitch,
			   int out_type, float *d_out_scale, uint64_t out_scale_pitch, void *d_saved, uint64_t saved_pitch, int saved_type,
			   float *d_saved_scale, uint64_t saved_scale_pitch, void *stream)
{
	int rc = require_device();
	if (rc != 0) {
		return rc;
	}
	const uint32_t size = product_type_size(type), bias_size = d_bias ? row_type_size(bias_type) : 1;
	if (!size || !bias_size || !activation_ok(activation) || !types_fit(type, out_type) || (d_saved && !types_fit(type, saved_type)) ||
	    (reinterpret_cast<uintptr_t>(d_bias) % bias_size) || (d_residual && out_type == OFI_AMD_E4M3)) {
		return -EINVAL;
	}
	rc = check_experts(d_offset, n_experts, max_rows, width, out_width);
	if (rc != 0 || max_rows == 0) {
		return rc;
	}
	forward_t o = {};
	o.scale = d_scale;
	o.scale_pitch = scale_pitch;
	o.weight_scale = d_weight_scale;
	o.bias = matrix(const_cast<void *>(d_bias), 0, bias_type, nullptr, 0);
	o.activation = activation;
	o.out = matrix(d_out, out_pitch, out_type, d_out_scale, out_scale_pitch);
	o.saved = matrix(d_saved, saved_pitch, saved_type, d_saved_scale, saved_scale_pitch);
	o.residual = matrix(const_cast<void *>(d_residual), residual_pitch, out_type, nullptr, 0);
	if (!rows_ok(d_rows, rows_pitch, max_rows, (uint64_t)width * size, size) ||
	    !stack_ok(d_weight, weight_pitch, expert_pitch, n_experts, out_width, (uint64_t)width * size, size) ||
	    !output_ok(o.out, max_rows, out_width, 1) || (d_saved && !output_ok(o.saved, max_rows, out_width, 1)) ||
	    (d_residual && !output_ok(o.residual, max_rows, out_width, 1)) ||
	    (type == OFI_AMD_E4M3 && (!scales_ok(d_scale, scale_pitch, max_rows, blocks_of(width)) || !scales_ok(d_weight_scale, 4, 1, 1)))) {
		return -EINVAL;
	}
	return forward(d_rows, rows_pitch, type, d_offset, n_experts, max_rows, d_weight, weight_pitch, expert_pitch, width, out_width, o, stream);
}

} /* extern "C" */
