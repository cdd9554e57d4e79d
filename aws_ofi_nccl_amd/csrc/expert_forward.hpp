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

/* A tile of both parts of a forward product, the same for all lanes: its rows from `from` on, the parts' columns from c0 and c1 on, of which
 * there0 and there1 are there; n: columns of the matrix */
struct forward_tile_t {
	uint64_t from;
	uint32_t rows, c0, c1, there0, there1, n, expert;
};
struct forward_in_t {
	eight_t add0, add1;
};

__device__ __forceinline__ uint32_t left_of(uint32_t there, uint32_t c) { return c < there ? there - c : 0u; }

/* c: the lane's first column in its part */
template <bool WHOLE> __device__ __forceinline__ forward_in_t forward_load(const forward_t &o, forward_tile_t t, uint32_t r, uint32_t c)
{
	forward_in_t in = {};
	if (o.residual.p && (WHOLE || r < t.rows)) {
		in.add0 = load_eight(o.residual, t.from + r, t.c0 + c, WHOLE ? 8 : left_of(t.there0, c), 0);
		in.add1 = load_eight(o.residual, t.from + r, t.c1 + c, WHOLE ? 8 : left_of(t.there1, c), 0);
	}
	return in;
}

__device__ __forceinline__ f32x8_t bias_at(const matrix_t &bias, uint64_t at, uint32_t left)
{
	return bias.type == OFI_AMD_FLOAT32 ? read_floats(bias.p + at * 4, left) : values_of(load_eight(bias, 0, at, left, 0), bias.type);
}

/* All sixteen lanes of a block call */
template <bool WHOLE>
__device__ __forceinline__ void forward_finish(const forward_t &o, forward_tile_t t, uint32_t r, uint32_t c, f32x8_t a, f32x8_t b,
					       const forward_in_t &in)
{
	const uint32_t left0 = WHOLE ? 8 : left_of(t.there0, c), left1 = WHOLE ? 8 : left_of(t.there1, c), blocks = blocks_of(t.n);
	const uint32_t block0 = t.c0 / kBlock, block1 = t.c1 / kBlock;
	if (o.bias.p) { /* out of the caches: held, it would be sixteen registers of the whole epilogue */
		const uint64_t at = (uint64_t)t.expert * t.n + c;
		a += bias_at(o.bias, at + t.c0, left0);
		b += bias_at(o.bias, at + t.c1, left1);
	}
	if (o.saved.p) {
		write_row<WHOLE>(o.saved, t.from, t.c0 + c, block0, r, t.rows, left0, a);
		write_row<WHOLE>(o.saved, t.from, (o.gated ? (uint64_t)t.n : 0) + t.c1 + c, (o.gated ? blocks : 0) + block1, r, t.rows, left1, b);
	}
	if (o.gated) {
		with_activation(o.activation, [&](auto activation) __attribute__((always_inline)) {
#pragma unroll
			for (int i = 0; i < 8; i++) {
				a[i] = activated<decltype(activation)::value>(a[i]) * b[i];
			}
		});
	} else {
		with_activation(o.activation, [&](auto activation) __attribute__((always_inline)) {
#pragma unroll
			for (int i = 0; i < 8; i++) {
				a[i] = activated<decltype(activation)::value>(a[i]);
				b[i] = activated<decltype(activation)::value>(b[i]);
			}
		});
		if (o.residual.p) {
			a += values_of(in.add0, o.residual.type);
			b += values_of(in.add1, o.residual.type);
		}
		write_row<WHOLE>(o.out, t.from, t.c1 + c, block1, r, t.rows, left1, b);
	}
	write_row<WHOLE>(o.out, t.from, t.c0 + c, block0, r, t.rows, left0, a);
}

/* Few rows an expert: expert_few.hip.  Few are up to 8, and up to 64 where tiles of 64 x 256 would leave compute units without any.
 * Both sides, us (width 4096 to 2048 in 8 bits into bfloat16, 32 experts): 128 rows 98-105 in streams and 127-129 in tiles, 256 rows 115 and 137,
 * 512 183 and 138-143; into 8 bits, whose blocks of columns are workgroups of 128: 128 rows 115 and 130, 256 rows 161 and 138; one expert of
 * 4096 x 4096 in bfloat16: 1 row 12 and 46, 64 rows 25 and 49.  What counts is the room for rows: 8 rows with room for 16,384 take 114 where
 * those with room for 8 take 42. */
inline bool forward_is_few(uint32_t max_rows, uint32_t n_experts, uint32_t n_tiles)
{
	const uint32_t experts = n_experts < max_rows ? n_experts : max_rows, of_expert = (max_rows + experts - 1) / experts;
	return max_rows <= 8ull * n_experts || (of_expert <= 64 && (uint64_t)experts * n_tiles < kComputeUnits);
}
int forward_few(const void *d_rows, uint64_t rows_pitch, int type, const int32_t *d_offset, uint32_t n_experts, uint32_t max_rows,
		const void *d_weight, uint64_t weight_pitch, uint64_t expert_pitch, uint32_t width, uint32_t n, const forward_t &o, void *stream);

} // namespace ofi_amd

#endif
