/*
 * The forward products for few rows an expert (a token or a few requests): each weight is used for a handful of rows, so that reading
 * the weights once is all the time there is.  They go from memory straight to the registers that feed the matrix cores, at any
 * alignment; rows come the same way, out of the caches.
 *
 * A wavefront has 16 columns of both parts (the gate's and the other's, or two neighbouring groups) and every KS-th step of 128 bytes of
 * their rows; what the KS have summed is added in LDS, in their order.  CG wavefronts side by side make a workgroup of 16 CG columns:
 * eight where a block of 128 shares an output's scale, else one, for as many workgroups as there can be.
 * 8 rows of 8 of 32 experts in 8 bits: product of 2048 to 4096 17.5 us (3.9 TB/s of weights with the launch), gated 4096 to 2048 32 us (4.2 TB/s) into
 * bfloat16 and 41 into 8 bits, as 16 blocks of 8 experts are half of the compute units; in bfloat16 31 and 55 us (4.3 and 4.9 TB/s).  128
 * rows of all 32, gated, bfloat16: 176 us, 6.0 TB/s.
 */
#include "expert_forward.hpp"

namespace ofi_amd {
namespace {

template <typename T, uint32_t MB, uint32_t CG, uint32_t KS>
__global__ __launch_bounds__(64 * CG * KS, MB == 1 ? 4 : 2) void expert_few_kernel(const int32_t *offset, const uint8_t *x, const uint8_t *w, uint32_t n_experts,
								  uint32_t max_rows, uint32_t width, uint32_t n, uint32_t n_tiles,
								  uint32_t first_tile, uint64_t x_pitch, uint64_t w_pitch, uint64_t expert_pitch,
								  forward_t o)
{
	constexpr uint32_t BM = 16 * MB, PART = 16 * CG, kAhead = MB > 1 ? 2 : sizeof(T) == 1 ? 3 : 4;
	constexpr bool SCALED = sizeof(T) == 1;
	__shared__ __attribute__((aligned(16))) float part[KS][BM][2][PART];

	const tile_t tile = find_tile<BM>({ offset, n_experts, max_rows, n_tiles }, first_tile + blockIdx.x);
	if (!tile.any) {
		return;
	}
	const uint32_t lane = threadIdx.x & 63u, wave = uniform(threadIdx.x >> 6), group = wave % CG, slice = wave / CG, q = lane >> 4;
	const uint32_t c0 = tile.nt * (o.gated ? PART : 2 * PART), c1 = o.gated ? c0 : c0 + PART;
	/* columns and rows that are not there are read as the last that is, and not written */
	const uint8_t *columns[2], *rows[MB];
	const uint8_t *const of_expert = w + tile.expert * expert_pitch;
#pragma unroll
	for (uint32_t p = 0; p < 2; p++) {
		const uint32_t c = (p ? c1 : c0) + group * 16 + (lane & 15u);
		columns[p] = of_expert + ((c < n ? c : n - 1) + (p && o.gated ? (uint64_t)n : 0)) * w_pitch + q * 16;
	}
	uint64_t row[MB];
#pragma unroll
	for (uint32_t m = 0; m < MB; m++) {
		const uint32_t r = m * 16 + (lane & 15u);
		row[m] = tile.from + (r < tile.rows ? r : tile.rows - 1);
		rows[m] = x + row[m] * x_pitch + q * 16;
	}
	const float *weight_scale[2] = {};
	const float *row_scale[MB] = {};
	if constexpr (SCALED) {
		const uint32_t k_blocks = blocks_of(width), n_blocks = blocks_of(n);
		const float *const scales = o.weight_scale + (uint64_t)tile.expert * (o.gated ? 2 : 1) * n_blocks * k_blocks;
#pragma unroll
		for (uint32_t p = 0; p < 2; p++) {
			const uint32_t c = (p ? c1 : c0) + group * 16;
			weight_scale[p] = scales + (uint64_t)((c < n ? c : n - 1) / kBlock + (p && o.gated ? n_blocks : 0)) * k_blocks;
		}
#pragma unroll
		for (uint32_t m = 0; m < MB; m++) {
			row_scale[m] = row_at(o.scale, o.scale_pitch, row[m]);
		}
	}

	struct step_t {
		u32x4_t c[2][2], r[MB][2];
		float by[MB], of[2];
	};
	f32x4_t sums[MB][2] = {};
	auto load = [&](uint32_t step, bool whole) __attribute__((always_inline)) {
		step_t s = {};
		const uint32_t at = step * kStepBytes;
		const int64_t left = (int64_t)width * sizeof(T) - at - q * 16;
#pragma unroll
		for (uint32_t half = 0; half < 2; half++) {
#pragma unroll
			for (uint32_t p = 0; p < 2; p++) {
				s.c[p][half] = whole ? *reinterpret_cast<const any16_t *>(columns[p] + at + half * 64)
						     : chunk_at<T>(columns[p] + at + half * 64, left - half * 64);
			}
#pragma unroll
			for (uint32_t m = 0; m < MB; m++) {
				s.r[m][half] = whole ? *reinterpret_cast<const any16_t *>(rows[m] + at + half * 64)
						     : chunk_at<T>(rows[m] + at + half * 64, left - half * 64);
			}
		}
		if constexpr (SCALED) {
			s.of[0] = weight_scale[0][step];
			s.of[1] = weight_scale[1][step];
#pragma unroll
			for (uint32_t m = 0; m < MB; m++) {
				s.by[m] = row_scale[m][step];
			}
		}
		return s;
	};
	auto add = [&](const step_t &s) __attribute__((always_inline)) {
		if constexpr (SCALED) {
#pragma unroll
			for (uint32_t p = 0; p < 2; p++) {
				const u32x4_t c[4] = { widened(s.c[p][0].x, s.c[p][0].y), widened(s.c[p][0].z, s.c[p][0].w),
						       widened(s.c[p][1].x, s.c[p][1].y), widened(s.c[p][1].z, s.c[p][1].w) };
#pragma unroll
				for (uint32_t m = 0; m < MB; m++) {
					f32x4_t of_step = { 0, 0, 0, 0 };
#pragma unroll
					for (uint32_t half = 0; half < 2; half++) {
						of_step = multiply<f16_t>(c[2 * half], widened(s.r[m][half].x, s.r[m][half].y), of_step);
						of_step = multiply<f16_t>(c[2 * half + 1], widened(s.r[m][half].z, s.r[m][half].w), of_step);
					}
					const float by = s.by[m] * s.of[p];
#pragma unroll
					for (int i = 0; i < 4; i++) {
						sums[m][p][i] = __builtin_fmaf(of_step[i], by, sums[m][p][i]);
					}
				}
			}
		} else {
#pragma unroll
			for (uint32_t half = 0; half < 2; half++) {
#pragma unroll
				for (uint32_t p = 0; p < 2; p++) {
#pragma unroll
					for (uint32_t m = 0; m < MB; m++) {
						sums[m][p] = multiply<T>(s.c[p][half], s.r[m][half], sums[m][p]);
					}
				}
			}
		}
	};
	/* whole steps, kAhead of them asked for; the rest of a row at the end */
	const uint32_t whole = width / kStepOf<T>, mine = whole > slice ? (whole - slice + KS - 1) / KS : 0;
	step_t ahead[kAhead];
#pragma unroll
	for (uint32_t i = 0; i < kAhead; i++) {
		if (i < mine) {
			ahead[i] = load(slice + i * KS, true);
		}
	}
	uint32_t s = 0;
	for (; s + 2 * kAhead <= mine; s += kAhead) {
#pragma unroll
		for (uint32_t i = 0; i < kAhead; i++) {
			add(ahead[i]);
			ahead[i] = load(slice + (s + i + kAhead) * KS, true);
			__builtin_amdgcn_sched_barrier(0); /* kAhead - 1 steps on their way at any time */
		}
	}
	for (; s < mine; s += kAhead) {
#pragma unroll
		for (uint32_t i = 0; i < kAhead; i++) {
			if (s + i < mine) {
				add(ahead[i]);
			}
			if (s + i + kAhead < mine) {
				ahead[i] = load(slice + (s + i + kAhead) * KS, true);
			}
		}
	}
	if (width % kStepOf<T> && whole % KS == slice) {
		add(load(whole, false));
	}

#pragma unroll
	for (uint32_t m = 0; m < MB; m++) {
#pragma unroll
		for (uint32_t p = 0; p < 2; p++) {
			*reinterpret_cast<f32x4_t *>(&part[slice][m * 16 + (lane & 15u)][p][group * 16 + 4 * q]) = sums[m][p];
		}
	}
	__syncthreads();
	const forward_tile_t place = { tile.from, tile.rows, c0, c1, n - c0 < PART ? n - c0 : PART, c1 >= n ? 0 : n - c1 < PART ? n - c1 : PART, n, tile.expert };
	constexpr uint32_t kOfRow = PART / 8; /* lanes that have a row */
	for (uint32_t r = threadIdx.x / kOfRow; r < BM; r += 64 * CG * KS / kOfRow) {
		const uint32_t c = threadIdx.x % kOfRow * 8;
		const forward_in_t in = forward_load<false>(o, place, r, c);
		f32x8_t a = {}, b = {};
#pragma unroll
		for (uint32_t s = 0; s < KS; s++) {
			a += *reinterpret_cast<const f32x8_t *>(&part[s][r][0][c]);
			b += *reinterpret_cast<const f32x8_t *>(&part[s][r][1][c]);
		}
		forward_finish<false>(o, place, r, c, a, b, in);
	}
}

} // namespace

int forward_few(const void *d_rows, uint64_t rows_pitch, int type, const int32_t *d_offset, uint32_t n_experts, uint32_t max_rows,
		const void *d_weight, uint64_t weight_pitch, uint64_t expert_pitch, uint32_t width, uint32_t n, const forward_t &o, void *stream)
{
	const bool blocks = o.out.type == OFI_AMD_E4M3 || (o.saved.p && o.saved.type == OFI_AMD_E4M3);
	const uint32_t columns = (blocks ? 128 : 16) * (o.gated ? 1 : 2), n_tiles = (n + columns - 1) / columns;
	const uint32_t of_expert = (max_rows + n_experts - 1) / n_experts;
	const uint32_t bm = of_expert <= 8 ? 16 : of_expert <= 20 ? 32 : 64;
	const uint64_t tiles = most_row_tiles(max_rows, n_experts, bm) * n_tiles;
	if (tiles > 0x7fffffffull) {
		return -E2BIG;
	}
	auto with = [&](auto element) {
		using T = decltype(element);
		auto kernel = blocks ? (bm == 16 ? expert_few_kernel<T, 1, 8, 2> : bm == 32 ? expert_few_kernel<T, 2, 8, 1> : expert_few_kernel<T, 4, 8, 1>)
				     : (bm == 16 ? expert_few_kernel<T, 1, 1, 8> : bm == 32 ? expert_few_kernel<T, 2, 1, 8> : expert_few_kernel<T, 4, 1, 8>);
		const uint32_t lanes = blocks && bm == 16 ? 1024 : 512;
		launch_tiles(tiles, lanes, [&](uint32_t first, uint32_t count) {
			return launch_kernel(kernel, dim3(count), dim3(lanes), 0, as_stream(stream), d_offset, static_cast<const uint8_t *>(d_rows),
					     static_cast<const uint8_t *>(d_weight), n_experts, max_rows, width, n, n_tiles, first, rows_pitch,
					     weight_pitch, expert_pitch, o);
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

} // namespace ofi_amd
