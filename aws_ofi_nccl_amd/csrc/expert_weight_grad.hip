/*
 * Gradients of the experts' weights and biases: dW_e = add + sum over the expert's rows of dy[r]^T x[r], db_e = add + sum of dy[r].
 * Both operands run across the summed axis, which is as long as the expert has rows; a workgroup sums all of it for one tile of
 * one expert's matrix, so that every sum runs in the rows' order.  The bias is the product with a column of ones.
 */
#include "expert_tiles.hpp"

namespace ofi_amd {
namespace {

struct weight_grad_t {
	matrix_t add, out;
	uint64_t expert_pitch; /* of both */
	const float *bias_add;
	float *dbias;
};

template <typename T> constexpr uint32_t kTwoOnes = 0x3f803f80u; /* bfloat16 */
template <> constexpr uint32_t kTwoOnes<f16_t> = 0x3c003c00u;

/* rows of the result: m (dout's columns); columns: n (x's) */
template <typename T, uint32_t WM, uint32_t WN, uint32_t MF, bool DIRECT>
__global__ __launch_bounds__(64 * WM * WN) void expert_weight_grad_kernel(const int32_t *offset, const uint8_t *dout, const uint8_t *x,
									  uint32_t max_rows, uint32_t m_width, uint32_t n_width,
									  uint32_t m_tiles, uint32_t n_tiles, uint32_t tiles, uint32_t first_tile,
									  uint64_t dout_pitch, uint64_t x_pitch, weight_grad_t o)
{
	constexpr uint32_t BM = 16 * MF * WM, BN = 2 * kBlock, THREADS = 64 * WM * WN, G = 8 / WN;
	using rows_tile = across_t<T, BM, THREADS>;
	using columns_tile = across_t<T, BN, THREADS>;
	constexpr uint32_t kTile = rows_tile::kBytes + columns_tile::kBytes, kFills = rows_tile::kChunks + columns_tile::kChunks;
	constexpr uint32_t kStages = DIRECT && WM < 4 ? 3 : 2;
	__shared__ __attribute__((aligned(1024))) uint8_t lds[kStages * kTile];

	/* an eighth of the tiles in one piece for each XCD; in an expert, bands of eight row tiles */
	const uint32_t id = first_tile + blockIdx.x, share = (tiles + 7) / 8, at = (id & 7u) * share + (id >> 3);
	if ((id >> 3) >= share || at >= tiles) {
		return;
	}
	const uint32_t expert = at / (m_tiles * n_tiles), in_expert = at % (m_tiles * n_tiles);
	const uint32_t band = in_expert / (8 * n_tiles), in_band = in_expert - band * 8 * n_tiles;
	const uint32_t height = m_tiles - band * 8 < 8 ? m_tiles - band * 8 : 8;
	const uint32_t m0 = (band * 8 + in_band % height) * BM, n0 = in_band / height * BN;
	uint32_t lo, hi;
	run_of(offset, expert, max_rows, lo, hi);
	lo = uniform(lo);
	hi = uniform(hi);

	const uint32_t lane = threadIdx.x & 63u, wave = uniform(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
	const uint32_t m_there = m_width - m0 < BM ? m_width - m0 : BM, n_there = n_width - n0 < BN ? n_width - n0 : BN;
	rows_tile rows = { dout + lo * dout_pitch + m0 * 2, dout_pitch, hi - lo, (int64_t)m_there * 2 };
	columns_tile columns = { x + lo * x_pitch + n0 * 2, x_pitch, hi - lo, (int64_t)n_there * 2 };
	const bool with_bias = o.dbias && n0 == 0; /* of one column tile, in a loop of its own */

	f32x4_t sums[MF][2][G], bias[MF];
#pragma unroll
	for (int m = 0; m < (int)MF; m++) {
		bias[m] = f32x4_t{ 0, 0, 0, 0 };
#pragma unroll
		for (int j = 0; j < (int)(2 * G); j++) {
			sums[m][j / G][j % G] = f32x4_t{ 0, 0, 0, 0 };
		}
	}
	const across_frag_t<BM> row_frag(wm * 16 * MF, lane);
	const across_frag_t<BN> column_frag(wn * 16 * G, lane);
	auto sum = [&](auto also) __attribute__((always_inline)) {
		sum_steps<T, DIRECT, kStages, kFills>(
			sums, wm * 16 * MF < m_there, (hi - lo + kStepRows - 1) / kStepRows, lds, kTile, rows_tile::kBytes, row_frag, column_frag,
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
			also);
	};
	if (with_bias) {
		sum([&](const u32x4_t(&r)[MF]) __attribute__((always_inline)) {
			const u32x4_t ones = { kTwoOnes<T>, kTwoOnes<T>, kTwoOnes<T>, kTwoOnes<T> };
#pragma unroll
			for (int m = 0; m < (int)MF; m++) {
				bias[m] = multiply<T>(ones, r[m], bias[m]);
			}
		});
	} else {
		sum([](const u32x4_t(&)[MF]) {});
	}

	if (with_bias && wn == 0 && lane < 16) {
#pragma unroll
		for (int m = 0; m < (int)MF; m++) {
			const uint32_t r = (wm * MF + m) * 16 + lane;
			if (r < m_there) {
				const uint64_t i = (uint64_t)expert * m_width + m0 + r;
				o.dbias[i] = bias[m][0] + (o.bias_add ? o.bias_add[i] : 0.0f);
			}
		}
	}
	const matrix_t out = { o.out.p + expert * o.expert_pitch, o.out.pitch, o.out.type, nullptr, 0 };
	const matrix_t add = { o.add.p ? o.add.p + expert * o.expert_pitch : nullptr, o.add.pitch, o.add.type, nullptr, 0 };
	const uint32_t c = (lane & 15u) * 8;
	const uint32_t left[2] = { c < n_there ? n_there - c : 0, c + kBlock < n_there ? n_there - c - kBlock : 0 };
	struct in_t {
		f32x8_t was[2]; /* float32, or eight values of 16 bits */
	};
	for_rows<WM, WN, MF>(
		sums, lds,
		[&](uint32_t r) {
			in_t in = {};
#pragma unroll
			for (int p = 0; p < 2; p++) {
				if (add.p && r < m_there && left[p]) {
					const uint64_t column = n0 + p * kBlock + c;
					if (add.type == OFI_AMD_FLOAT32) {
						in.was[p] = read_floats(add.p + (m0 + r) * add.pitch + column * 4, left[p]);
					} else {
						in.was[p].lo = __builtin_bit_cast(f32x4_t, load_eight(add, m0 + r, column, left[p], 0).words);
					}
				}
			}
			return in;
		},
		[&](uint32_t r, f32x8_t a, f32x8_t b, const in_t &in) {
#pragma unroll
			for (int p = 0; p < 2; p++) {
				f32x8_t v = p ? b : a;
				if (r < m_there && left[p]) {
					if (add.p) {
						const f32x4_t low = in.was[p].lo;
						v += add.type == OFI_AMD_FLOAT32 ? in.was[p] : floats_of<T>(__builtin_bit_cast(u32x4_t, low));
					}
					write_values(out, m0 + r, n0 + p * kBlock + c, left[p], v);
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
	/* tiles of 256 x 256 where they are enough for the GPU, else of 128 x 256 */
	const uint32_t n_tiles = (width + 255) / 256;
	const bool direct = in_chunks(d_dout, dout_pitch, 2ull * out_width) && in_chunks(d_rows, rows_pitch, 2ull * width);
	const bool wide = direct && (uint64_t)n_experts * ((out_width + 255) / 256) * n_tiles >= 256;
	const uint32_t bm = wide ? 256 : 128, m_tiles = (out_width + bm - 1) / bm;
	const uint64_t tiles = (uint64_t)n_experts * m_tiles * n_tiles;
	if (tiles > 0x7fffffffull) {
		return -E2BIG;
	}
	weight_grad_t o = {};
	o.out = { static_cast<uint8_t *>(d_dweight), dweight_pitch, dweight_type, nullptr, 0 };
	o.add = { static_cast<uint8_t *>(const_cast<void *>(d_add)), dweight_pitch, dweight_type, nullptr, 0 };
	o.expert_pitch = expert_pitch;
	o.bias_add = d_bias_add;
	o.dbias = d_dbias;
	auto with = [&](auto element) {
		using T = decltype(element);
		auto kernel = direct ? (wide ? expert_weight_grad_kernel<T, 4, 2, 4, true> : expert_weight_grad_kernel<T, 2, 4, 4, true>)
				     : expert_weight_grad_kernel<T, 2, 4, 4, false>;
		launch_tiles(tiles, [&](uint32_t first, uint32_t count) {
			launch_kernel(kernel, dim3(count), dim3(512), 0, as_stream(stream), d_offset, static_cast<const uint8_t *>(d_dout),
				      static_cast<const uint8_t *>(d_rows), max_rows, out_width, width, m_tiles, n_tiles, (uint32_t)tiles, first,
				      dout_pitch, rows_pitch, o);
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
