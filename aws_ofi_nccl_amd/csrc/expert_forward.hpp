/*
 * What leaves an expert's forward product: bias, what is kept for the way back, activation, the gate's product, residual, and rounding,
 * for a lane's eight columns of both parts of a row.
 */
#ifndef OFI_AMD_EXPERT_FORWARD_HPP_
#define OFI_AMD_EXPERT_FORWARD_HPP_

#include "expert_tiles.hpp"

namespace ofi_amd {

struct forward_t {
	const float *scale, *weight_scale;
	uint64_t scale_pitch;
	matrix_t bias, residual, out, saved;
	int activation;
	bool gated;
};

struct forward_rows_t {
	struct in_t {
		eight_t add0, add1;
	};
	const forward_t &o;
	uint64_t from, n;
	uint32_t rows, column0, column1, left0, left1, block0, block1, blocks;
	f32x8_t bias0, bias1;

	/* c0, c1: the parts' first columns, each of `part` columns at most; c: the lane's first in them */
	__device__ __forceinline__ forward_rows_t(const forward_t &with, const tile_t &tile, uint32_t width, uint32_t c0, uint32_t c1, uint32_t part,
						  uint32_t c)
		: o(with), from(tile.from), n(width), rows(tile.rows), column0(c0 + c), column1(c1 + c), block0(c0 / kBlock), block1(c1 / kBlock),
		  blocks(blocks_of(width)), bias0{}, bias1{}
	{
		const uint32_t end0 = c0 + part < width ? c0 + part : width, end1 = c1 + part < width ? c1 + part : width;
		left0 = column0 < end0 ? end0 - column0 : 0;
		left1 = column1 < end1 ? end1 - column1 : 0;
		if (o.bias.p) {
			auto bias_at = [&](uint32_t column, uint32_t left) {
				const uint64_t at = (uint64_t)tile.expert * n + column;
				return o.bias.type == OFI_AMD_FLOAT32 ? read_floats(o.bias.p + at * 4, left)
								      : values_of(load_eight(o.bias, 0, at, left, 0), o.bias.type);
			};
			bias0 = bias_at(column0, left0);
			bias1 = bias_at(column1, left1);
		}
	}
	__device__ __forceinline__ in_t load(uint32_t r) const
	{
		in_t in = {};
		if (o.residual.p && r < rows) {
			in.add0 = load_eight(o.residual, from + r, column0, left0, 0);
			in.add1 = load_eight(o.residual, from + r, column1, left1, 0);
		}
		return in;
	}
	/* All sixteen lanes of a block call */
	__device__ __forceinline__ void finish(uint32_t r, f32x8_t a, f32x8_t b, const in_t &in) const
	{
		const uint64_t row = from + r;
		const bool write = r < rows;
		if (o.bias.p) {
			a += bias0;
			b += bias1;
		}
		if (o.saved.p) {
			write_any(o.saved, row, column0, left0, block0, a, write);
			write_any(o.saved, row, (o.gated ? n : 0) + column1, left1, (o.gated ? blocks : 0) + block1, b, write);
		}
		with_activation(o.activation, [&](auto activation) {
#pragma unroll
			for (int i = 0; i < 8; i++) {
				a[i] = activated<decltype(activation)::value>(a[i]);
				b[i] = o.gated ? b[i] : activated<decltype(activation)::value>(b[i]);
			}
		});
		if (o.gated) {
			a *= b;
		} else {
			if (o.residual.p) {
				a += values_of(in.add0, o.residual.type);
				b += values_of(in.add1, o.residual.type);
			}
			write_any(o.out, row, column1, left1, block1, b, write);
		}
		write_any(o.out, row, column0, left0, block0, a, write);
	}
};

/* Few rows an expert: expert_few.hip.  Few are up to 8, and up to 64 where tiles of 64 x 256 would leave compute units without any.
 * Both sides, us (width 4096 to 2048 in 8 bits, 32 experts): 128 rows 98 in streams and 127 in tiles, 256 rows 115 and 136, 512 183 and
 * 143; one expert of 4096 x 4096 in bfloat16: 1 row 12 and 46, 64 rows 25 and 49. */
inline bool forward_is_few(uint32_t max_rows, uint32_t n_experts, uint32_t n_tiles)
{
	const uint32_t experts = n_experts < max_rows ? n_experts : max_rows, of_expert = (max_rows + experts - 1) / experts;
	return max_rows <= 8ull * n_experts || (of_expert <= 64 && (uint64_t)experts * n_tiles < kComputeUnits);
}
int forward_few(const void *d_rows, uint64_t rows_pitch, int type, const int32_t *d_offset, uint32_t n_experts, uint32_t max_rows,
		const void *d_weight, uint64_t weight_pitch, uint64_t expert_pitch, uint32_t width, uint32_t n, const forward_t &o, void *stream);

} // namespace ofi_amd

#endif
