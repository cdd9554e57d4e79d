/*
 * Gradients of the experts' products with respect to what went in:
 *   rows_grad     dx = dy W (+ add)
 *   hidden_grad   dh = dy W, and from it and what the forward product kept: dg = dh u act'(g), du = dh act(g), h = act(g) u
 * dy runs along the summed axis (the product's outputs), the weights run across it.  In the second the checkpoint is read, in 8 bits or 16, by the
 * lanes that have the sums: dh is never written.
 * Bound by the matrix cores for many rows: 32,768 rows of 32 experts, bfloat16, rows_grad of 4096 to 4096 1005-1040 us (1,080 TFLOP/s), hidden_grad of
 * 4096 to 2048 from a checkpoint of 8 bits 645 (850, and 1.35 GB moved in the epilogues); by the weights for few: 8192 rows of 64 experts, 2048
 * to 4096, 245 us, 4.8 TB/s.  Odd widths come through registers at any alignment: 1331 rows of 5 experts, 999 to 1023, 41 us, a step's latency
 * sixteen times in half of the compute units; 700 rows of 60 experts, 1000 to 1408, 44 us, 3.9 TB/s of weights.
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
struct backward_args_t {
	rows_t of;
	const uint8_t *dout, *w;
	uint64_t dout_pitch, w_pitch, expert_pitch;
	uint32_t k, n, first_tile;
	backward_t o;
};

/* A tile, the same for all lanes: its rows from `from` on, `there` columns from c0 on of n */
struct backward_tile_t {
	uint64_t from;
	uint32_t rows, c0, there, n;
};

/* COLUMN_ROWS: of the summed axis in a tile of the columns, a step's or half a step's */
template <typename T, uint32_t BM, uint32_t THREADS, uint32_t COLUMN_ROWS> struct backward_operands_t {
	along_t<T, BM, THREADS> rows;
	across_t<T, 2 * kBlock, THREADS, COLUMN_ROWS> columns;
	backward_tile_t place;
	static constexpr uint32_t kRowsBytes = decltype(rows)::kBytes, kColumnsBytes = decltype(columns)::kBytes, kBytes = kRowsBytes + kColumnsBytes;
	static constexpr uint32_t kFills = decltype(rows)::kChunks + decltype(columns)::kChunks;

	__device__ __forceinline__ void set(const backward_args_t *a, const tile_t &tile)
	{
		const uint32_t n = a->n, c0 = tile.nt * 2 * kBlock, there = n - c0 < 2 * kBlock ? n - c0 : 2 * kBlock;
		place = { tile.from, tile.rows, c0, there, n };
		rows.set(a->dout + tile.from * a->dout_pitch, a->dout_pitch, tile.rows, (int64_t)a->k * 2);
		columns.set(a->w + tile.expert * a->expert_pitch + c0 * 2, a->w_pitch, a->k, (int64_t)there * 2);
	}
	__device__ __forceinline__ void load(uint32_t step)
	{
		rows.load(step);
		columns.load(step);
	}
	__device__ __forceinline__ void store(uint32_t step, uint8_t *to) const
	{
		rows.store(step, to);
		columns.store(step, to + kRowsBytes);
	}
	__device__ __forceinline__ void fill(uint32_t step, uint8_t *to) const
	{
		rows.fill(step, to);
		columns.fill(step, to + kRowsBytes);
	}
};

template <typename T, uint32_t WM, uint32_t WN, uint32_t MF, bool HIDDEN, bool DIRECT>
__global__ __launch_bounds__(64 * WM * WN, WM * WN == 4 ? 2 : 1) void expert_backward_kernel(backward_args_t)
{
	constexpr uint32_t BM = 16 * MF * WM, BN = 2 * kBlock, THREADS = 64 * WM * WN, G = 8 / WN;
	constexpr bool PAIR = WM * WN == 4; /* of workgroups on a compute unit */
	using operands_t = backward_operands_t<T, BM, THREADS, PAIR ? kStepRows / 2 : kStepRows>;
	constexpr uint32_t kStages = DIRECT ? 3 : 2;
	__shared__ __attribute__((aligned(1024))) uint8_t lds[PAIR ? 2 * operands_t::kRowsBytes + 3 * operands_t::kColumnsBytes : kStages * operands_t::kBytes];

	operands_t of;
	uint32_t steps;
	{
		const backward_args_t *const a = argument<backward_args_t>();
		steps = (a->k + kStepRows - 1) / kStepRows;
		const tile_t tile = find_tile<BM>(a->of, a->first_tile + blockIdx.x);
		if (!tile.any) {
			return;
		}
		of.set(a, tile);
	}
	const uint32_t lane = threadIdx.x & 63u, wave = uniform(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
	f32x4_t sums[MF][2][G] = {};
	if constexpr (PAIR) {
		sum_halves<T, decltype(of.rows)::kChunks, decltype(of.columns)::kChunks, operands_t::kRowsBytes, operands_t::kColumnsBytes>(
			sums, wm * 16 * MF < of.place.rows, steps, lds, along_frag_t(wm * 16 * MF, lane), across_frag_t<BN>(wn * 16 * G, lane),
			[&](uint32_t step, uint8_t *to) __attribute__((always_inline)) { of.rows.fill(step, to); },
			[&](uint32_t half, uint8_t *to) __attribute__((always_inline)) { of.columns.fill(half, to); }, [](const u32x4_t(&)[MF]) {});
	} else {
		sum_steps<T, DIRECT, kStages, operands_t::kFills>(
			sums, wm * 16 * MF < of.place.rows, steps, lds, operands_t::kBytes, operands_t::kRowsBytes, along_frag_t(wm * 16 * MF, lane),
			across_frag_t<BN>(wn * 16 * G, lane), [&](uint32_t step, uint8_t *to) __attribute__((always_inline)) { of.fill(step, to); },
			[&](uint32_t step) __attribute__((always_inline)) { of.load(step); },
			[&](uint32_t step, uint8_t *to) __attribute__((always_inline)) { of.store(step, to); }, [](const u32x4_t(&)[MF]) {});
	}

	struct in_t {
		eight_t g[2], u[2]; /* what was kept, or what is added */
	};
	const backward_tile_t place = of.place;
	auto left_at = [&](uint32_t column) { return column < place.there ? place.there - column : 0u; };
	for_rows<WM, WN, MF, false>(
		sums, lds, place.rows == BM && place.there == BN,
		[&](auto all, uint32_t r, uint32_t part_lane) __attribute__((always_inline)) {
			constexpr bool WHOLE = decltype(all)::value;
			const backward_t &o = argument<backward_args_t>()->o;
			in_t in = {};
			const uint32_t c = part_lane * 8, block = place.c0 / kBlock;
			const uint64_t row = place.from + r;
#pragma unroll
			for (int p = 0; p < 2; p++) {
				const uint32_t column = place.c0 + p * kBlock + c, some = WHOLE ? 8 : left_at(p * kBlock + c);
				if (WHOLE || (r < place.rows && some)) {
					if (!HIDDEN && o.add.p) {
						in.g[p] = load_eight(o.add, row, column, some, 0);
					} else if (HIDDEN) {
						in.g[p] = load_eight(o.saved, row, column, some, block + p);
						if (o.gated) {
							in.u[p] = load_eight(o.saved, row, (uint64_t)place.n + column, some, blocks_of(place.n) + block + p);
						}
					}
				}
			}
			return in;
		},
		[&](auto all, uint32_t r, uint32_t part_lane, f32x8_t p0, f32x8_t p1, const in_t &in) __attribute__((always_inline)) {
			constexpr bool WHOLE = decltype(all)::value;
			const backward_t &o = argument<backward_args_t>()->o;
			const uint32_t c = part_lane * 8;
#pragma unroll
			for (int p = 0; p < 2; p++) {
				const uint64_t column = place.c0 + p * kBlock + c;
				const uint32_t left = WHOLE ? 8 : left_at(p * kBlock + c);
				f32x8_t v = p ? p1 : p0;
				if constexpr (HIDDEN) {
					f32x8_t g = values_of(in.g[p], o.saved.type), h = { 1, 1, 1, 1, 1, 1, 1, 1 };
					if (o.gated) {
						h = values_of(in.u[p], o.saved.type);
					}
					with_activation(o.activation, [&](auto activation) __attribute__((always_inline)) {
#pragma unroll
						for (int i = 0; i < 8; i++) {
							float value, slope;
							activated_with_slope<decltype(activation)::value>(g[i], value, slope);
							g[i] = v[i] * h[i] * slope;
							h[i] *= value;
							v[i] *= value;
						}
					});
					write_row<WHOLE>(o.dsaved, place.from, column, 0, r, place.rows, left, g);
					if (o.gated) {
						write_row<WHOLE>(o.dsaved, place.from, (uint64_t)place.n + column, 0, r, place.rows, left, v);
					}
					if (o.hidden.p) {
						write_row<WHOLE>(o.hidden, place.from, column, 0, r, place.rows, left, h);
					}
				} else {
					if (o.add.p) {
						v += values_of(in.g[p], o.add.type);
					}
					write_row<WHOLE>(o.out, place.from, column, 0, r, place.rows, left, v);
				}
			}
		});
}

template <bool HIDDEN>
int backward(const void *d_dout, uint64_t dout_pitch, int type, const int32_t *d_offset, uint32_t n_experts, uint32_t max_rows,
	     const void *d_weight, uint64_t weight_pitch, uint64_t expert_pitch, uint32_t k, uint32_t n, const backward_t &o, void *stream)
{
	const bool direct = in_chunks(d_dout, dout_pitch, 2ull * k) && in_chunks(d_weight, weight_pitch, 2ull * n) && expert_pitch % 16 == 0;
	const uint32_t n_tiles = (n + 2 * kBlock - 1) / (2 * kBlock);
	const bool pairs = direct && pairs_fit(max_rows, n_experts, n_tiles);
	const uint32_t bm = pairs ? 128 : row_tile_for(max_rows, n_experts, n_tiles, false);
	const uint64_t tiles = most_row_tiles(max_rows, n_experts, bm) * n_tiles;
	if (tiles > 0x7fffffffull) {
		return -E2BIG;
	}
	backward_args_t args = { { d_offset, n_experts, max_rows, n_tiles }, static_cast<const uint8_t *>(d_dout), static_cast<const uint8_t *>(d_weight),
				 dout_pitch, weight_pitch, expert_pitch, k, n, 0, o };
	auto with = [&](auto element) {
		using T = decltype(element);
		auto kernel = direct ? (pairs ? expert_backward_kernel<T, 2, 2, 4, HIDDEN, true>
						   : bm == 128 ? expert_backward_kernel<T, 2, 4, 4, HIDDEN, true>
							    : expert_backward_kernel<T, 1, 8, 4, HIDDEN, true>)
				     : bm == 128 ? expert_backward_kernel<T, 2, 4, 4, HIDDEN, false>
						 : expert_backward_kernel<T, 1, 8, 4, HIDDEN, false>;
		const uint32_t lanes = pairs ? 256 : 512;
		launch_tiles(tiles, lanes, [&](uint32_t first, uint32_t count) {
			args.first_tile = first;
			return launch_kernel(kernel, dim3(count), dim3(lanes), 0, as_stream(stream), args);
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
