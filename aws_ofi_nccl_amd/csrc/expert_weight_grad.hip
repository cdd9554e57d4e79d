/*
 * Gradients of the experts' weights and biases: dW_e = add + sum over the expert's rows of dy[r]^T x[r], db_e = add + sum of dy[r].
 * Both operands run across the summed axis, which is as long as the expert has rows; a workgroup sums all of it for one tile of
 * one expert's matrix, so that every sum runs in the rows' order.  The bias is the product with a column of ones.
 * 32,768 rows of 32 experts, 4096 x 4096, bfloat16, us: bfloat16 out 1170 (940 TFLOP/s), float32 out 1280, float32 added to float32 1390 (4.8 GB at 3.5
 * TB/s, 790 TFLOP/s): the matrix cores and, for float32, the memory's share that two workgroups on a compute unit do not hide.  1331 rows of 60
 * experts, 777 x 1023: 60 us, of 776 x 1024 33, where most of a tile's time is its beginning and its epilogue.
 */
#include "expert_tiles.hpp"

namespace ofi_amd {
namespace {

struct weight_grad_args_t {
	const int32_t *offset;
	const uint8_t *dout, *x;
	uint64_t dout_pitch, x_pitch;
	uint32_t max_rows, m, n; /* rows of the result are dout's columns, m of them; its columns are x's */
	uint32_t n_experts, m_tiles, n_tiles, first_tile;
	matrix_t add, out;
	uint64_t expert_pitch; /* of both */
	const float *bias_add;
	float *dbias;
};

template <typename T> constexpr uint32_t kTwoOnes = 0x3f803f80u; /* bfloat16 */
template <> constexpr uint32_t kTwoOnes<f16_t> = 0x3c003c00u;

/* A tile, the same for all lanes */
struct weight_tile_t {
	uint32_t expert, m0, n0, m_there, n_there, summed;
	bool bias; /* of one column tile, in a loop of its own */
};

/* COLUMN_ROWS: of the summed axis in a tile of the columns, a step's or half a step's */
template <typename T, uint32_t BM, uint32_t THREADS, uint32_t COLUMN_ROWS> struct weight_operands_t {
	static constexpr uint32_t BN = 2 * kBlock;
	across_t<T, BM, THREADS> rows;
	across_t<T, BN, THREADS, COLUMN_ROWS> columns;
	weight_tile_t place;
	static constexpr uint32_t kRowsBytes = decltype(rows)::kBytes, kColumnsBytes = decltype(columns)::kBytes, kBytes = kRowsBytes + kColumnsBytes;
	static constexpr uint32_t kFills = decltype(rows)::kChunks + decltype(columns)::kChunks;

	/* Workgroups go to the eight XCDs in turn: each XCD has an eighth of every expert's tiles, in one piece, as the experts have unlike numbers of
	 * rows to sum (with whole experts to an XCD 1662 us for 1412 of 32,768 rows of 32 experts); one on for each expert, as the last piece may be
	 * short or none (777 x 1023 of 60 experts has seven: 74.6 us, so 61.7).  In an expert, bands of eight row tiles.  False: `id` has none */
	__device__ __forceinline__ bool set(const weight_grad_args_t *a, uint32_t id)
	{
		const uint32_t n_tiles = a->n_tiles, m_tiles = a->m_tiles, share = (m_tiles * n_tiles + 7) / 8, at = id >> 3, expert = at / share;
		const uint32_t in_expert = ((id + expert) & 7u) * share + at - expert * share;
		if (expert >= a->n_experts || in_expert >= m_tiles * n_tiles) {
			return false;
		}
		const uint32_t band = in_expert / (8 * n_tiles), in_band = in_expert - band * 8 * n_tiles;
		const uint32_t height = m_tiles - band * 8 < 8 ? m_tiles - band * 8 : 8, nt = in_band / height;
		const uint32_t m0 = (band * 8 + in_band - nt * height) * BM, n0 = nt * BN;
		uint32_t lo, hi;
		run_of(a->offset, expert, a->max_rows, lo, hi);
		lo = uniform(lo);
		hi = uniform(hi);
		place = { expert, m0, n0, a->m - m0 < BM ? a->m - m0 : BM, a->n - n0 < BN ? a->n - n0 : BN, hi - lo, a->dbias && n0 == 0 };
		rows.set(a->dout + lo * a->dout_pitch + m0 * 2, a->dout_pitch, hi - lo, (int64_t)place.m_there * 2);
		columns.set(a->x + lo * a->x_pitch + n0 * 2, a->x_pitch, hi - lo, (int64_t)place.n_there * 2);
		return true;
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

/* F32: float32 out, else T */
template <typename T, uint32_t WM, uint32_t WN, uint32_t MF, bool DIRECT, bool F32>
__global__ __launch_bounds__(64 * WM * WN, WM * WN == 4 ? 2 : 1) void expert_weight_grad_kernel(weight_grad_args_t)
{
	constexpr uint32_t BM = 16 * MF * WM, BN = 2 * kBlock, THREADS = 64 * WM * WN, G = 8 / WN, kStages = 2;
	constexpr bool PAIR = WM * WN == 4; /* of workgroups on a compute unit */
	using operands_t = weight_operands_t<T, BM, THREADS, PAIR ? kStepRows / 2 : kStepRows>;
	__shared__ __attribute__((aligned(1024))) uint8_t lds[PAIR ? 2 * operands_t::kRowsBytes + 3 * operands_t::kColumnsBytes : kStages * operands_t::kBytes];

	operands_t of;
	{
		const weight_grad_args_t *const a = argument<weight_grad_args_t>();
		if (!of.set(a, a->first_tile + blockIdx.x)) {
			return;
		}
	}
	const uint32_t lane = threadIdx.x & 63u, wave = uniform(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
	const weight_tile_t place = of.place;
	const uint32_t steps = (place.summed + kStepRows - 1) / kStepRows;
	const bool busy = wm * 16 * MF < place.m_there;
	f32x4_t sums[MF][2][G] = {};
	auto sum = [&](auto also) __attribute__((always_inline)) {
		if constexpr (PAIR) {
			sum_halves<T, decltype(of.rows)::kChunks, decltype(of.columns)::kChunks, operands_t::kRowsBytes, operands_t::kColumnsBytes>(
				sums, busy, steps, lds, across_frag_t<BM>(wm * 16 * MF, lane), across_frag_t<BN>(wn * 16 * G, lane),
				[&](uint32_t step, uint8_t *to) __attribute__((always_inline)) { of.rows.fill(step, to); },
				[&](uint32_t half, uint8_t *to) __attribute__((always_inline)) { of.columns.fill(half, to); }, also);
		} else {
			sum_steps<T, DIRECT, kStages, operands_t::kFills>(
				sums, busy, steps, lds, operands_t::kBytes, operands_t::kRowsBytes, across_frag_t<BM>(wm * 16 * MF, lane),
				across_frag_t<BN>(wn * 16 * G, lane), [&](uint32_t step, uint8_t *to) __attribute__((always_inline)) { of.fill(step, to); },
				[&](uint32_t step) __attribute__((always_inline)) { of.load(step); },
				[&](uint32_t step, uint8_t *to) __attribute__((always_inline)) { of.store(step, to); }, also);
		}
	};
	if (place.bias) {
		f32x4_t bias[MF] = {};
		sum([&](const u32x4_t(&r)[MF]) __attribute__((always_inline)) {
			const u32x4_t ones = { kTwoOnes<T>, kTwoOnes<T>, kTwoOnes<T>, kTwoOnes<T> };
#pragma unroll
			for (int m = 0; m < (int)MF; m++) {
				bias[m] = multiply<T>(ones, r[m], bias[m]);
			}
		});
		const weight_grad_args_t *const a = argument<weight_grad_args_t>();
		if (wn == 0 && lane < 16) {
#pragma unroll
			for (int m = 0; m < (int)MF; m++) {
				const uint32_t r = (wm * MF + m) * 16 + lane;
				if (r < place.m_there) {
					const uint64_t i = (uint64_t)place.expert * a->m + place.m0 + r;
					a->dbias[i] = bias[m][0] + (a->bias_add ? a->bias_add[i] : 0.0f);
				}
			}
		}
	} else {
		sum([](const u32x4_t(&)[MF]) {});
	}

	/* Written past the caches, which are for the operands (float32 added to float32 1448 -> 1399 us, 776 x 1024 of 60 experts 36.3 -> 33.4).
	 * A lane's columns of each part: of float32 four, and four 64 further, so that sixteen lanes have 256 bytes of a row both times; of 16 bits eight */
	struct in_t {
		eight_t eight[F32 ? 1 : 2];
		f32x4_t four[F32 ? 4 : 1];
	};
	auto left_of = [&](uint32_t column) { return column < place.n_there ? place.n_there - column : 0u; };
	for_rows<WM, WN, MF, F32>(
		sums, lds, place.m_there == BM && place.n_there == BN,
		[&](auto all, uint32_t r, uint32_t part_lane) __attribute__((always_inline)) {
			constexpr bool WHOLE = decltype(all)::value;
			const weight_grad_args_t *const a = argument<weight_grad_args_t>();
			in_t in = {};
			if (a->add.p && (WHOLE || r < place.m_there)) {
				const matrix_t add = { a->add.p + place.expert * a->expert_pitch, a->add.pitch, a->add.type, nullptr, 0 };
				if constexpr (F32) {
					const float *const p = reinterpret_cast<const float *>(add.p + (uint64_t)(place.m0 + r) * add.pitch);
#pragma unroll
					for (uint32_t i = 0; i < 4; i++) {
						const uint32_t c = i * 64 + part_lane * 4;
						in.four[i] = read_four(p + place.n0 + c, WHOLE ? 4 : left_of(c));
					}
				} else {
#pragma unroll
					for (uint32_t i = 0; i < 2; i++) {
						const uint32_t c = i * kBlock + part_lane * 8;
						in.eight[i] = load_eight(add, place.m0 + r, place.n0 + c, WHOLE ? 8 : left_of(c), 0);
					}
				}
			}
			return in;
		},
		[&](auto all, uint32_t r, uint32_t part_lane, f32x8_t p0, f32x8_t p1, const in_t &in) __attribute__((always_inline)) {
			constexpr bool WHOLE = decltype(all)::value;
			const weight_grad_args_t *const a = argument<weight_grad_args_t>();
			const matrix_t out = { a->out.p + place.expert * a->expert_pitch, a->out.pitch, a->out.type, nullptr, 0 };
			if constexpr (F32) {
				if (WHOLE || r < place.m_there) {
					float *const p = reinterpret_cast<float *>(out.p + (uint64_t)(place.m0 + r) * out.pitch);
#pragma unroll
					for (uint32_t i = 0; i < 4; i++) {
						const f32x4_t v = i == 0 ? p0.lo : i == 1 ? p0.hi : i == 2 ? p1.lo : p1.hi;
						const uint32_t c = i * 64 + part_lane * 4;
						write_four(p + place.n0 + c, WHOLE ? 4 : left_of(c), v + in.four[i]);
					}
				}
			} else {
#pragma unroll
				for (uint32_t i = 0; i < 2; i++) {
					const uint32_t c = i * kBlock + part_lane * 8;
					f32x8_t v = i ? p1 : p0;
					if (a->add.p) {
						v += floats_of<T>(in.eight[i].words);
					}
					write_row_as<WHOLE, T, true>(out, place.m0, place.n0 + c, r, place.m_there, WHOLE ? 8 : left_of(c), v);
				}
			}
		});
}

} // namespace
} // namespace ofi_amd

using namespace ofi_amd;

extern "C" {

int ofi_amd_expert_weight_grad(const void *d_dout, uint64_t dout_pitch, const void *d_rows, uint64_t rows_pitch, int type,
			       const int32_t *d_offset, uint32_t n_experts, uint32_t max_rows, uint32_t width, uint32_t out_width,
			       const void *d_add, void *d_dweight, uint64_t dweight_pitch, uint64_t expert_pitch, int dweight_type,
			       const float *d_bias_add, float *d_dbias, void *stream)
{
	int rc = require_device();
	if (rc != 0) {
		return rc;
	}
	if ((type != OFI_AMD_BFLOAT16 && type != OFI_AMD_FLOAT16) || (dweight_type != type && dweight_type != OFI_AMD_FLOAT32)) {
		return -EINVAL;
	}
	rc = check_experts(d_offset, n_experts, max_rows, width, out_width);
	if (rc != 0) {
		return rc;
	}
	const uint32_t size = row_type_size(dweight_type);
	if ((max_rows != 0 && (!rows_ok(d_dout, dout_pitch, max_rows, 2ull * out_width, 2) ||
			       !rows_ok(d_rows, rows_pitch, max_rows, 2ull * width, 2))) ||
	    !stack_ok(d_dweight, dweight_pitch, expert_pitch, n_experts, out_width, (uint64_t)width * size, size) ||
	    (reinterpret_cast<uintptr_t>(d_add) % size) || ((reinterpret_cast<uintptr_t>(d_dbias) | reinterpret_cast<uintptr_t>(d_bias_add)) & 3u)) {
		return -EINVAL;
	}
	if (max_rows == 1) { /* may be apart by anything; rows behind it have to lie behind its bytes, where zeros are read */
		dout_pitch = 2ull * out_width;
		rows_pitch = 2ull * width;
	}
	/* tiles of 128 x 256, two workgroups to a compute unit where they are enough for that */
	const uint32_t n_tiles = (width + 255) / 256, m_tiles = (out_width + 127) / 128;
	const bool direct = in_chunks(d_dout, dout_pitch, 2ull * out_width) && in_chunks(d_rows, rows_pitch, 2ull * width);
	const bool pairs = direct && (uint64_t)n_experts * m_tiles * n_tiles >= 2 * kComputeUnits;
	const uint64_t tiles = (uint64_t)n_experts * (((uint64_t)m_tiles * n_tiles + 7) / 8) * 8;
	if (tiles > 0x7fffffffull) {
		return -E2BIG;
	}
	const matrix_t out = { static_cast<uint8_t *>(d_dweight), dweight_pitch, dweight_type, nullptr, 0 };
	const matrix_t add = { static_cast<uint8_t *>(const_cast<void *>(d_add)), dweight_pitch, dweight_type, nullptr, 0 };
	weight_grad_args_t args = { d_offset, static_cast<const uint8_t *>(d_dout), static_cast<const uint8_t *>(d_rows), dout_pitch, rows_pitch, max_rows,
				    out_width, width, n_experts, m_tiles, n_tiles, 0, add, out, expert_pitch, d_bias_add, d_dbias };
	auto with = [&](auto element) {
		using T = decltype(element);
		auto of = [&](auto f32) {
			constexpr bool F = decltype(f32)::value;
			return direct ? (pairs ? expert_weight_grad_kernel<T, 2, 2, 4, true, F> : expert_weight_grad_kernel<T, 2, 4, 4, true, F>)
				      : expert_weight_grad_kernel<T, 2, 4, 4, false, F>;
		};
		auto kernel = dweight_type == OFI_AMD_FLOAT32 ? of(std::true_type{}) : of(std::false_type{});
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

} /* extern "C" */
