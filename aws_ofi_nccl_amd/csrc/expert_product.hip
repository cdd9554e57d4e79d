/*
 * Products of rows sorted by expert with their expert's weights:
 *   gated      h = act(x G^T) (x U^T), both projections in one kernel, and what the activation was taken of kept for the way back
 *   product    y = act(x W^T + b) + r
 * x and the weights run along the summed axis.  Rows of e4m3 and their weights have a scale for every 128 of it, which are what one
 * step sums: a step's sums are multiplied by both scales in 32 bits and added.
 */
#include "expert_forward.hpp"

namespace ofi_amd {
namespace {

template <typename T, uint32_t WM, uint32_t WN, uint32_t MF, bool DIRECT>
__global__ __launch_bounds__(64 * WM * WN) void expert_forward_kernel(const int32_t *offset, const uint8_t *x, const uint8_t *w, uint32_t n_experts,
								      uint32_t max_rows, uint32_t width, uint32_t n, uint32_t n_tiles,
								      uint32_t first_tile, uint64_t x_pitch, uint64_t w_pitch,
								      uint64_t expert_pitch, forward_t o)
{
	constexpr uint32_t BM = 16 * MF * WM, THREADS = 64 * WM * WN, G = 8 / WN;
	constexpr bool SCALED = sizeof(T) == 1;
	using rows_tile = along_t<T, BM, THREADS>;
	using part_tile = along_t<T, kBlock, THREADS>;
	constexpr uint32_t kTile = rows_tile::kBytes + 2 * part_tile::kBytes, kFills = rows_tile::kChunks + 2 * part_tile::kChunks;
	constexpr uint32_t kStages = DIRECT && !SCALED && WM < 4 ? 3 : 2;
	__shared__ __attribute__((aligned(1024))) uint8_t lds[kStages * kTile];

	const tile_t tile = tile_of<BM>(offset, n_experts, max_rows, n_tiles, first_tile + blockIdx.x);
	if (!tile.any) {
		return;
	}
	const uint32_t lane = threadIdx.x & 63u, wave = uniform(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
	/* column 0 of both parts, in the matrix of n columns; a gated block's parts are n rows of weights apart */
	const uint32_t c0 = tile.nt * (o.gated ? kBlock : 2 * kBlock), c1 = o.gated ? c0 : c0 + kBlock;
	const uint32_t there0 = n - c0 < kBlock ? n - c0 : kBlock, there1 = c1 >= n ? 0 : n - c1 < kBlock ? n - c1 : kBlock;
	const uint8_t *const weights = w + tile.expert * expert_pitch;
	const int64_t bytes = (int64_t)width * sizeof(T);
	rows_tile rows = { x + tile.from * x_pitch, x_pitch, tile.rows, bytes };
	part_tile part0 = { weights + c0 * w_pitch, w_pitch, there0, bytes };
	part_tile part1 = { weights + (there1 ? (o.gated ? (uint64_t)n : 0) + c1 : 0) * w_pitch, w_pitch, there1, bytes };

	f32x4_t sums[MF][2][G];
#pragma unroll
	for (int m = 0; m < (int)MF; m++) {
#pragma unroll
		for (int j = 0; j < (int)(2 * G); j++) {
			sums[m][j / G][j % G] = f32x4_t{ 0, 0, 0, 0 };
		}
	}
	const along_frag_t row_frag(wm * 16 * MF, lane), column_frag(wn * 16 * G, lane);
	const uint32_t steps = (width + kStepOf<T> - 1) / kStepOf<T>;
	auto fill = [&](uint32_t step, uint8_t *to) __attribute__((always_inline)) {
		rows.fill(step, to);
		part0.fill(step, to + rows_tile::kBytes);
		part1.fill(step, to + rows_tile::kBytes + part_tile::kBytes);
	};
	auto load = [&](uint32_t step) __attribute__((always_inline)) {
		rows.load(step);
		part0.load(step);
		part1.load(step);
	};
	auto store = [&](uint8_t *to) __attribute__((always_inline)) {
		rows.store(to);
		part0.store(to + rows_tile::kBytes);
		part1.store(to + rows_tile::kBytes + part_tile::kBytes);
	};
	if constexpr (!SCALED) {
		sum_steps<T, DIRECT, kStages, kFills>(sums, wm * 16 * MF < tile.rows, steps, lds, kTile, rows_tile::kBytes, row_frag, column_frag, fill, load, store,
				     [](const u32x4_t(&)[MF]) {});
	} else {
		/* a lane's row of each of its groups */
		const float *row_scale[MF], *weight_scale[2];
		const uint32_t k_blocks = blocks_of(width), n_blocks = blocks_of(n);
		const float *of_expert = o.weight_scale + (uint64_t)tile.expert * (o.gated ? 2 : 1) * n_blocks * k_blocks;
		weight_scale[0] = of_expert + (uint64_t)(c0 / kBlock) * k_blocks;
		weight_scale[1] = there1 ? of_expert + (uint64_t)((o.gated ? n_blocks : 0) + c1 / kBlock) * k_blocks : weight_scale[0];
#pragma unroll
		for (int m = 0; m < (int)MF; m++) {
			const uint32_t r = (wm * MF + m) * 16 + (lane & 15u);
			row_scale[m] = row_at(o.scale, o.scale_pitch, tile.from + (r < tile.rows ? r : tile.rows - 1));
		}
		if (DIRECT) {
			fill(0, lds);
		} else {
			load(0);
		}
		for (uint32_t step = 0; step < steps; step++) {
			uint8_t *const now = lds + (step & 1u) * kTile;
			if (DIRECT) {
				landed<0>();
			} else {
				store(now);
			}
			__syncthreads(); /* this tile is there, and the other one's readers are past it */
			if (step + 1 < steps) {
				if (DIRECT) {
					fill(step + 1, lds + (~step & 1u) * kTile);
				} else {
					load(step + 1);
				}
			}
			float by[MF][2];
			u32x4_t r[MF][4];
#pragma unroll
			for (int m = 0; m < (int)MF; m++) {
				const float s = row_scale[m][step];
				by[m][0] = s * weight_scale[0][step];
				by[m][1] = s * weight_scale[1][step];
#pragma unroll
				for (uint32_t half = 0; half < 2; half++) {
					const u32x4_t q = row_frag.get(now, m * 16, half);
					r[m][2 * half] = widened(q.x, q.y);
					r[m][2 * half + 1] = widened(q.z, q.w);
				}
			}
#pragma unroll
			for (int j = 0; j < (int)(2 * G); j++) {
				const uint8_t *const columns = now + rows_tile::kBytes;
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
	}

	const forward_rows_t out(o, tile, n, c0, c1, kBlock, (lane & 15u) * 8);
	for_rows<WM, WN, MF>(
		sums, lds, [&](uint32_t r) { return out.load(r); },
		[&](uint32_t r, f32x8_t a, f32x8_t b, const forward_rows_t::in_t &in) { out.finish(r, a, b, in); });
}


int forward(const void *d_rows, uint64_t rows_pitch, int type, const int32_t *d_offset, uint32_t n_experts, uint32_t max_rows,
	    const void *d_weight, uint64_t weight_pitch, uint64_t expert_pitch, uint32_t width, uint32_t n, const forward_t &o, void *stream)
{
	const uint64_t bytes = (uint64_t)width * product_type_size(type);
	const bool direct = in_chunks(d_rows, rows_pitch, bytes) && in_chunks(d_weight, weight_pitch, bytes) && expert_pitch % 16 == 0;
	const uint32_t n_tiles = (n + (o.gated ? kBlock : 2 * kBlock) - 1) / (o.gated ? kBlock : 2 * kBlock);
	const uint32_t bm = row_tile_for(max_rows, n_experts, n_tiles, direct);
	if (forward_is_few(max_rows, n_experts, n_tiles)) {
		return forward_few(d_rows, rows_pitch, type, d_offset, n_experts, max_rows, d_weight, weight_pitch, expert_pitch, width, n, o, stream);
	}
	const uint64_t tiles = most_row_tiles(max_rows, n_experts, bm) * n_tiles;
	if (tiles > 0x7fffffffull) {
		return -E2BIG;
	}
	auto with = [&](auto element) {
		using T = decltype(element);
		auto kernel = direct ? (bm == 256 ? expert_forward_kernel<T, 4, 2, 4, true>
						: bm == 128 ? expert_forward_kernel<T, 2, 4, 4, true> : expert_forward_kernel<T, 1, 8, 4, true>)
				     : bm == 128 ? expert_forward_kernel<T, 2, 4, 4, false> : expert_forward_kernel<T, 1, 8, 4, false>;
		launch_tiles(tiles, [&](uint32_t first, uint32_t count) {
			launch_kernel(kernel, dim3(count), dim3(512), 0, as_stream(stream), d_offset,
				      static_cast<const uint8_t *>(d_rows), static_cast<const uint8_t *>(d_weight), n_experts, max_rows, width, n,
				      n_tiles, first, rows_pitch, weight_pitch, expert_pitch, o);
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
