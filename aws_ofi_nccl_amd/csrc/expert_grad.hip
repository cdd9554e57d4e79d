/*
 * Gradients of the experts' products with respect to what went in:
 *   rows_grad     dx = dy W (+ add)
 *   hidden_grad   dh = dy W, and from it and what the forward product kept: dg = dh u act'(g), du = dh act(g), h = act(g) u
 * dy runs along the summed axis (the product's outputs), the weights run across it.  In the second the sums never leave the
 * registers: the checkpoint is read, in 8 bits or 16, where they are.
 */
#include "expert_tiles.hpp"

namespace ofi_amd {
namespace {

struct backward_t {
	matrix_t saved, dsaved, hidden; /* hidden_grad */
	matrix_t add, out;              /* rows_grad */
	int activation;
	bool gated;
};

/* k: the product's outputs, n: its columns */
template <typename T, uint32_t WM, uint32_t WN, uint32_t MF, bool HIDDEN, bool DIRECT>
__global__ __launch_bounds__(64 * WM * WN) void expert_backward_kernel(const int32_t *offset, const uint8_t *dout, const uint8_t *w,
								       uint32_t n_experts, uint32_t max_rows, uint32_t k, uint32_t n,
								       uint32_t n_tiles, uint32_t first_tile, uint64_t dout_pitch,
								       uint64_t w_pitch, uint64_t expert_pitch, backward_t o)
{
	constexpr uint32_t BM = 16 * MF * WM, BN = 2 * kBlock, THREADS = 64 * WM * WN, G = 8 / WN;
	using rows_tile = along_t<T, BM, THREADS>;
	using columns_tile = across_t<T, BN, THREADS>;
	constexpr uint32_t kTile = rows_tile::kBytes + columns_tile::kBytes, kFills = rows_tile::kChunks + columns_tile::kChunks;
	constexpr uint32_t kStages = DIRECT && WM < 4 ? 3 : 2;
	__shared__ __attribute__((aligned(1024))) uint8_t lds[kStages * kTile];

	const tile_t tile = tile_of<BM>(offset, n_experts, max_rows, n_tiles, first_tile + blockIdx.x);
	if (!tile.any) {
		return;
	}
	const uint32_t lane = threadIdx.x & 63u, wave = uniform(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
	const uint32_t c0 = tile.nt * BN, there = n - c0 < BN ? n - c0 : BN;
	rows_tile rows = { dout + tile.from * dout_pitch, dout_pitch, tile.rows, (int64_t)k * 2 };
	columns_tile columns = { w + tile.expert * expert_pitch + c0 * 2, w_pitch, k, (int64_t)there * 2 };

	f32x4_t sums[MF][2][G];
#pragma unroll
	for (int m = 0; m < (int)MF; m++) {
#pragma unroll
		for (int j = 0; j < (int)(2 * G); j++) {
			sums[m][j / G][j % G] = f32x4_t{ 0, 0, 0, 0 };
		}
	}
	const along_frag_t row_frag(wm * 16 * MF, lane);
	const across_frag_t<BN> column_frag(wn * 16 * G, lane);
	sum_steps<T, DIRECT, kStages, kFills>(
		sums, wm * 16 * MF < tile.rows, (k + kStepRows - 1) / kStepRows, lds, kTile, rows_tile::kBytes, row_frag, column_frag,
		[&](uint32_t step, uint8_t *to) __attribute__((always_inline)) {
			rows.fill(step, to);
			columns.fill(step, to + rows_tile::kBytes);
		},
		[&](uint32_t step) __attribute__((always_inline)) {
			rows.load(step);
			columns.load(step);
		},
		[&](uint8_t *to) __attribute__((always_inline)) {
			rows.store(to);
			columns.store(to + rows_tile::kBytes);
		},
		[](const u32x4_t(&)[MF]) {});

	const uint32_t c = (lane & 15u) * 8, blocks = blocks_of(n), block = c0 / kBlock;
	const uint32_t left[2] = { c < there ? there - c : 0, c + kBlock < there ? there - c - kBlock : 0 };
	struct in_t {
		eight_t g[2], u[2]; /* what was kept, or what is added */
	};
	for_rows<WM, WN, MF>(
		sums, lds,
		[&](uint32_t r) {
			in_t in = {};
			const uint64_t row = tile.from + r;
#pragma unroll
			for (int p = 0; p < 2; p++) {
				const uint32_t column = c0 + p * kBlock + c;
				if (r < tile.rows && left[p]) {
					if (!HIDDEN && o.add.p) {
						in.g[p] = load_eight(o.add, row, column, left[p], 0);
					} else if (HIDDEN) {
						in.g[p] = load_eight(o.saved, row, column, left[p], block + p);
						if (o.gated) {
							in.u[p] = load_eight(o.saved, row, (uint64_t)n + column, left[p], blocks + block + p);
						}
					}
				}
			}
			return in;
		},
		[&](uint32_t r, f32x8_t a, f32x8_t b, const in_t &in) {
			const uint64_t row = tile.from + r;
#pragma unroll
			for (int p = 0; p < 2; p++) {
				const uint32_t column = c0 + p * kBlock + c;
				f32x8_t v = p ? b : a;
				if (r >= tile.rows || left[p] == 0) {
					continue;
				}
				if constexpr (HIDDEN) {
					f32x8_t g = values_of(in.g[p], o.saved.type), u = {}, h;
					if (o.gated) {
						u = values_of(in.u[p], o.saved.type);
					}
					with_activation(o.activation, [&](auto activation) {
#pragma unroll
						for (int i = 0; i < 8; i++) {
							float value, slope;
							activated_with_slope<decltype(activation)::value>(g[i], value, slope);
							g[i] = o.gated ? v[i] * u[i] * slope : v[i] * slope;
							h[i] = o.gated ? value * u[i] : value;
							v[i] *= value;
						}
					});
					write_values(o.dsaved, row, column, left[p], g);
					if (o.gated) {
						write_values(o.dsaved, row, (uint64_t)n + column, left[p], v);
					}
					if (o.hidden.p) {
						write_values(o.hidden, row, column, left[p], h);
					}
				} else {
					if (o.add.p) {
						v += values_of(in.g[p], o.add.type);
					}
					write_values(o.out, row, column, left[p], v);
				}
			}
		});
}

template <bool HIDDEN>
int backward(const void *d_dout, uint64_t dout_pitch, int type, const int32_t *d_offset, uint32_t n_experts, uint32_t max_rows,
	     const void *d_weight, uint64_t weight_pitch, uint64_t expert_pitch, uint32_t k, uint32_t n, const backward_t &o, void *stream)
{
	const bool direct = in_chunks(d_dout, dout_pitch, 2ull * k) && in_chunks(d_weight, weight_pitch, 2ull * n) && expert_pitch % 16 == 0;
	const uint32_t n_tiles = (n + 2 * kBlock - 1) / (2 * kBlock), bm = row_tile_for(max_rows, n_experts, n_tiles, direct);
	const uint64_t tiles = most_row_tiles(max_rows, n_experts, bm) * n_tiles;
	if (tiles > 0x7fffffffull) {
		return -E2BIG;
	}
	auto with = [&](auto element) {
		using T = decltype(element);
		auto kernel = direct ? (bm == 256 ? expert_backward_kernel<T, 4, 2, 4, HIDDEN, true>
						: bm == 128 ? expert_backward_kernel<T, 2, 4, 4, HIDDEN, true>
							    : expert_backward_kernel<T, 1, 8, 4, HIDDEN, true>)
				     : bm == 128 ? expert_backward_kernel<T, 2, 4, 4, HIDDEN, false>
						 : expert_backward_kernel<T, 1, 8, 4, HIDDEN, false>;
		launch_tiles(tiles, [&](uint32_t first, uint32_t count) {
			launch_kernel(kernel, dim3(count), dim3(512), 0, as_stream(stream), d_offset,
				      static_cast<const uint8_t *>(d_dout), static_cast<const uint8_t *>(d_weight), n_experts, max_rows, k, n,
				      n_tiles, first, dout_pitch, weight_pitch, expert_pitch, o);
		});
	};
	if (type == OFI_AMD_BFLOAT16) {
		with(bf16_t{});
	} else {
		with(f16_t{});
	}
	OFI_AMD_HIP_TRY(hipGetLastError());
	return 0;
}

bool two_byte(int type) { return type == OFI_AMD_BFLOAT16 || type == OFI_AMD_FLOAT16; }

matrix_t matrix(const void *p, uint64_t pitch, int type, const float *scale = nullptr, uint64_t scale_pitch = 0)
{
	return { static_cast<uint8_t *>(const_cast<void *>(p)), pitch, type, const_cast<float *>(scale), scale_pitch };
}

} // namespace
} // namespace ofi_amd

using namespace ofi_amd;

extern "C" {

int ofi_amd_expert_hidden_grad(const void *d_dout, uint64_t dout_pitch, int type, const int32_t *d_offset, uint32_t n_experts, uint32_t max_rows,
			       const void *d_weight, uint64_t weight_pitch, uint64_t expert_pitch, uint32_t width, uint32_t inner, int gated,
			       int activation, const void *d_saved, uint64_t saved_pitch, int saved_type, const float *d_saved_scale,
			       uint64_t saved_scale_pitch, void *d_dsaved, uint64_t dsaved_pitch, void *d_hidden, uint64_t hidden_pitch,
			       void *stream)
{
	int rc = require_device();
	if (rc != 0) {
		return rc;
	}
	if (!two_byte(type) || !activation_ok(activation) || (saved_type != type && saved_type != OFI_AMD_E4M3) || (gated & ~1)) {
		return -EINVAL;
	}
	rc = check_experts(d_offset, n_experts, max_rows, width, inner);
	if (rc != 0 || max_rows == 0) {
		return rc;
	}
	const uint32_t parts = gated ? 2 : 1, size = product_type_size(saved_type);
	const uint64_t bytes = (uint64_t)parts * inner;
	if (!rows_ok(d_dout, dout_pitch, max_rows, 2ull * width, 2) ||
	    !stack_ok(d_weight, weight_pitch, expert_pitch, n_experts, width, 2ull * inner, 2) ||
	    !rows_ok(d_saved, saved_pitch, max_rows, bytes * size, size) || !rows_ok(d_dsaved, dsaved_pitch, max_rows, bytes * 2, 2) ||
	    (saved_type == OFI_AMD_E4M3 && !scales_ok(d_saved_scale, saved_scale_pitch, max_rows, parts * blocks_of(inner))) ||
	    (d_hidden && !rows_ok(d_hidden, hidden_pitch, max_rows, 2ull * inner, 2))) {
		return -EINVAL;
	}
	backward_t o = {};
	o.saved = matrix(d_saved, saved_pitch, saved_type, d_saved_scale, saved_scale_pitch);
	o.dsaved = matrix(d_dsaved, dsaved_pitch, type);
	o.hidden = matrix(d_hidden, hidden_pitch, type);
	o.activation = activation;
	o.gated = gated;
	return backward<true>(d_dout, dout_pitch, type, d_offset, n_experts, max_rows, d_weight, weight_pitch, expert_pitch, width, inner, o,
			      stream);
}

int ofi_amd_expert_rows_grad(const void *d_dout, uint64_t dout_pitch, int type, const int32_t *d_offset, uint32_t n_experts, uint32_t max_rows,
			     const void *d_weight, uint64_t weight_pitch, uint64_t expert_pitch, uint32_t width, uint32_t out_width,
			     const void *d_add, uint64_t add_pitch, void *d_drows, uint64_t drows_pitch, void *stream)
{
	int rc = require_device();
	if (rc != 0) {
		return rc;
	}
	if (!two_byte(type)) {
		return -EINVAL;
	}
	rc = check_experts(d_offset, n_experts, max_rows, width, out_width);
	if (rc != 0 || max_rows == 0) {
		return rc;
	}
	if (!rows_ok(d_dout, dout_pitch, max_rows, 2ull * out_width, 2) ||
	    !stack_ok(d_weight, weight_pitch, expert_pitch, n_experts, out_width, 2ull * width, 2) ||
	    (d_add && !rows_ok(d_add, add_pitch, max_rows, 2ull * width, 2)) || !rows_ok(d_drows, drows_pitch, max_rows, 2ull * width, 2)) {
		return -EINVAL;
	}
	backward_t o = {};
	o.add = matrix(d_add, add_pitch, type);
	o.out = matrix(d_drows, drows_pitch, type);
	return backward<false>(d_dout, dout_pitch, type, d_offset, n_experts, max_rows, d_weight, weight_pitch, expert_pitch, out_width, width, o,
			       stream);
}

} /* extern "C" */
