/*
 * What the kernels on rows of numbers share: pieces of a row as floats, and sums and maxima over lanes.
 *
 * A row is cut into chunks of V elements, one per lane: 16 bytes, at whatever address the row starts (the global memory path
 * takes any alignment).  The last chunk of a row whose width is no whole number of chunks is read and computed as the 16 bytes
 * that end with the row, so that no load is conditional: its first `skip` elements are its neighbour's, which stores them.
 * Lanes beyond the row read those last 16 bytes too and skip all of them.  Rows narrower than a chunk are cut into single
 * elements (V = 1).
 */
#ifndef OFI_AMD_ROW_TYPES_HPP_
#define OFI_AMD_ROW_TYPES_HPP_

#include <cerrno>
#include <cstdint>
#include <type_traits>

#include <hip/hip_runtime.h>

#include "ofi_amd_hotpath.h"
#include "row_places.hpp"

namespace ofi_amd {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

template <typename T> constexpr uint32_t kChunk = 16 / sizeof(T); /* elements of a chunk */

template <typename T, uint32_t V> struct piece_t {
	typedef T raw __attribute__((ext_vector_type(V)));
	typedef T anywhere __attribute__((ext_vector_type(V), aligned(sizeof(T)))); /* at an address of the element's alignment */
};
template <typename T, uint32_t V> using raw_t = typename piece_t<T, V>::raw;
typedef uint32_t any16_t __attribute__((ext_vector_type(4), aligned(1))); /* 16 bytes of anything at any address */

/* What a kernel reads and writes past the caches */
enum flow_t { STREAM_NONE, STREAM_LOADS, STREAM_BOTH };

/* STREAM: read once, not to be kept in the caches */
template <bool STREAM, typename T, uint32_t V> __device__ __forceinline__ raw_t<T, V> load_raw(const T *p)
{
	const auto *q = reinterpret_cast<const typename piece_t<T, V>::anywhere *>(p);
	return STREAM ? __builtin_nontemporal_load(q) : *q;
}

/* The chunk's own elements, 0 in place of the skipped ones */
template <typename T, uint32_t V> __device__ __forceinline__ void to_floats(raw_t<T, V> c, uint32_t skip, float (&f)[V])
{
#pragma unroll
	for (uint32_t i = 0; i < V; i++) {
		f[i] = (float)c[i];
	}
	if (skip) {
#pragma unroll
		for (uint32_t i = 0; i < V; i++) {
			f[i] = i < skip ? 0.0f : f[i];
		}
	}
}

/* The chunk's own elements go to the row's place `from`, each rounded to the row's type once, to nearest even */
template <bool STREAM, typename T, uint32_t V> __device__ __forceinline__ void store_piece(T *p, uint32_t skip, const float (&f)[V])
{
	float all __attribute__((ext_vector_type(V)));
#pragma unroll
	for (uint32_t i = 0; i < V; i++) {
		all[i] = f[i];
	}
	const raw_t<T, V> c = __builtin_convertvector(all, raw_t<T, V>);
	if (skip == 0) {
		auto *q = reinterpret_cast<typename piece_t<T, V>::anywhere *>(p);
		if (STREAM) {
			__builtin_nontemporal_store(c, q);
		} else {
			*q = c;
		}
	} else {
#pragma unroll
		for (uint32_t i = 0; i < V; i++) {
			if (i >= skip) {
				p[i] = c[i];
			}
		}
	}
}

template <typename T> __host__ __device__ __forceinline__ T *row_at(T *base, uint64_t pitch, uint64_t row)
{
	using byte_t = typename std::conditional<std::is_const<T>::value, const uint8_t, uint8_t>::type;
	return reinterpret_cast<T *>(reinterpret_cast<byte_t *>(base) + row * pitch);
}

/* The value of the lane that is `CTRL` away within the row of 16 (data-parallel primitives: no LDS) */
template <int CTRL> __device__ __forceinline__ uint32_t dpp(uint32_t v)
{
	return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}

template <uint32_t V, typename T> __device__ __forceinline__ uint32_t lag_of(const T *row)
{
	return lag_at<V>(reinterpret_cast<uintptr_t>(row), sizeof(T));
}

/* LANES of a row in a wavefront; chunk: where the lane's chunk lies, at: its column */
template <typename T, uint32_t V, uint32_t LANES>
__device__ __forceinline__ uint32_t load_rest(const T *chunk, uint32_t lag, uint32_t at, uint32_t width)
{
	const bool lone = is_lone<V, LANES>(threadIdx.x, at, width);
	return V > 1 && lag && lone ? *reinterpret_cast<const rest_t *>(chunk + kRestAt<V>) : 0u;
}

/* All lanes of the wavefront call */
template <typename T, uint32_t V, uint32_t LANES>
__device__ __forceinline__ void catch_up(raw_t<T, V> &c, uint32_t rest, uint32_t lag, uint32_t at, uint32_t width)
{
	if constexpr (sizeof(T) == 2 && V > 1) {
		u32x4_t w = __builtin_bit_cast(u32x4_t, c);
		const uint32_t next = dpp<0x130>(w.x); /* wave_shl:1 */
		const uint32_t end = is_lone<V, LANES>(threadIdx.x, at, width) ? rest : next; /* its lower half */
		if (lag) {
			w = u32x4_t{ __builtin_amdgcn_alignbit(w.y, w.x, 16), __builtin_amdgcn_alignbit(w.z, w.y, 16),
				     __builtin_amdgcn_alignbit(w.w, w.z, 16), __builtin_amdgcn_alignbit(end, w.w, 16) };
			c = __builtin_bit_cast(raw_t<T, V>, w);
		}
	}
}

/* Rows of 16 lanes exchanged: {a0, b0, a2, b2} and {a1, b1, a3, b3} */
__device__ __forceinline__ void swap_rows16(uint32_t &a, uint32_t &b)
{
	const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
	a = r[0];
	b = r[1];
}

/* Halves exchanged: {a low, b low} and {a high, b high} */
__device__ __forceinline__ void swap_halves(uint32_t &a, uint32_t &b)
{
	const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
	a = r[0];
	b = r[1];
}

/* op over each group of LANES neighbouring lanes (a power of two), the result in all of them.  The order of the operations
 * depends on the lane number alone. */
template <int LANES, typename Op> __device__ __forceinline__ uint32_t over_lanes(uint32_t v, Op op)
{
	if (LANES >= 2) {
		v = op(v, dpp<0xB1>(v)); /* quad_perm [1,0,3,2] */
	}
	if (LANES >= 4) {
		v = op(v, dpp<0x4E>(v)); /* quad_perm [2,3,0,1] */
	}
	if (LANES >= 8) {
		v = op(v, dpp<0x141>(v)); /* row_half_mirror */
	}
	if (LANES >= 16) {
		v = op(v, dpp<0x140>(v)); /* row_mirror */
	}
	if (LANES >= 32) {
		uint32_t w = v;
		swap_rows16(v, w);
		v = op(v, w);
	}
	if (LANES >= 64) {
		uint32_t w = v;
		swap_halves(v, w);
		v = op(v, w);
	}
	return v;
}

template <int LANES> __device__ __forceinline__ float sum_over(float v)
{
	return __uint_as_float(over_lanes<LANES>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
		return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
	}));
}

__device__ __forceinline__ float sum_of_halves(float a, float b)
{
	uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
	swap_halves(x, y);
	return __uint_as_float(x) + __uint_as_float(y);
}

__device__ __forceinline__ float sum_of_rows16(float a, float b)
{
	uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
	swap_rows16(x, y);
	return __uint_as_float(x) + __uint_as_float(y);
}

/* Eight sums over the wavefront at once: the one of v[lane / 8], in all eight of those lanes.  Half of what is added is another value
 * at each of the first three steps, so that there are ten additions instead of 48. */
__device__ __forceinline__ float eight_sums(const float (&v)[8], uint32_t lane)
{
	float four[4], two[2];
#pragma unroll
	for (int i = 0; i < 4; i++) {
		four[i] = sum_of_halves(v[i], v[i + 4]);
	}
#pragma unroll
	for (int i = 0; i < 2; i++) {
		two[i] = sum_of_rows16(four[i], four[i + 2]);
	}
	const bool odd = lane & 8u;
	const float keep = odd ? two[1] : two[0], give = odd ? two[0] : two[1];
	return sum_over<8>(keep + __uint_as_float(dpp<0x140>(__float_as_uint(give)))); /* row_mirror */
}

/* Maximum of absolute values given as their bits: a NaN's are above an infinity's, so that a NaN comes out */
template <int LANES> __device__ __forceinline__ uint32_t max_bits_over(uint32_t v)
{
	return over_lanes<LANES>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

__device__ __forceinline__ uint32_t abs_bits(float f) { return __float_as_uint(f) & 0x7fffffffu; }

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

/* The scale of a group's values from the largest one's bits */
__device__ __forceinline__ float scale_of(uint32_t amax_bits)
{
	/* __builtin_fmaxf would drop a NaN, which every value of its group is then to show */
	const float s = __uint_as_float(amax_bits) / 448.0f;
	return s < 0x1p-126f ? 0x1p-126f : s;
}

/* The value of every wavefront of a row's put together by op, in all of their lanes.  s: a word for each of up to 16 wavefronts, which
 * nothing else uses meanwhile.  All wavefronts of the workgroup call. */
template <typename Op> __device__ __forceinline__ uint32_t over_waves(uint32_t v, uint32_t *s, uint32_t waves, uint32_t none, Op op)
{
	if (waves == 1) {
		return v;
	}
	const uint32_t lane = threadIdx.x & 63u;
	if (lane == 0) {
		s[threadIdx.x >> 6] = v;
	}
	__syncthreads();
	return over_lanes<16>((lane & 15u) < waves ? s[lane & 15u] : none, op);
}

__device__ __forceinline__ float block_sum(float v, uint32_t *s, uint32_t waves)
{
	return __uint_as_float(over_waves(__float_as_uint(sum_over<64>(v)), s, waves, 0u, [](uint32_t a, uint32_t b) {
		return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
	}));
}

__device__ __forceinline__ uint32_t block_max_bits(uint32_t v, uint32_t *s, uint32_t waves)
{
	return over_waves(max_bits_over<64>(v), s, waves, 0u, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

/* Wavefronts that take a row of `chunks` in the fewest rounds of at most `most`, as even as they can be */
inline uint32_t even_waves(uint32_t chunks, uint32_t most)
{
	const uint32_t all = (chunks + 63) / 64, rounds = (all + most - 1) / most;
	return (all + rounds - 1) / rounds;
}

/* Bytes of an element of a row's type, 0 for a type that rows do not have */
inline uint32_t row_type_size(int type)
{
	return type == OFI_AMD_FLOAT32 ? 4u : type == OFI_AMD_BFLOAT16 || type == OFI_AMD_FLOAT16 ? 2u : 0u;
}

/* Calls f with a value of the row's type (checked before) and the elements of its chunks */
template <typename F> inline void with_row_type(int type, uint32_t width, F f)
{
	auto with = [&](auto element) {
		constexpr uint32_t V = kChunk<decltype(element)>;
		if (width >= V) {
			f(element, std::integral_constant<uint32_t, V>{});
		} else {
			f(element, std::integral_constant<uint32_t, 1>{});
		}
	};
	if (type == OFI_AMD_BFLOAT16) {
		with(bf16_t{});
	} else if (type == OFI_AMD_FLOAT16) {
		with(f16_t{});
	} else {
		with(float{});
	}
}

/*
 * By what a call reads and writes.  Inputs that fill much of the memory-side cache of 256 MB have not stayed there since they were
 * made, and read past the caches they come faster; outputs of a call that overflows it will not be found there either.  Measured on
 * three sets of tensors by turns, us with neither / streaming loads / both:
 *   sums of 8 rows of 8 KiB        84 MB 14.3 15.9 -      168 MB 34.3 31.1 29.7    672 MB 131.2 115.5 117.3   1343 MB 263 249 238
 *   their gradient                 71 MB 14.8 17.3 16.4   143 MB 32.9 27.2 29.9    571 MB 118.1 118.3 113.4   2283 MB 454 460 444
 *   norms of 8192 values to e4m3   59 MB 13.7 14.1 14.1   236 MB 46.1 43.8 42.6    472 MB 84.4 82.8 80.3      944 MB 164.9 164.3 157.5
 *   gradients of norms of 4096     67 MB 17.4 19.1 -      134 MB 32.2 29.1 29.9    268 MB 54.9 48.4 50.9      537 MB 102.4 96.8 94.4
 * Rows that do not start on chunks go the same way (sums of rows of 8190 bytes, 1343 MB, 262 268 247; their norms' gradient, 537 MB, 131 132
 * 122), although what lies across two lines is fetched twice where the caches would have had it (43 MB of rows of 4092 bytes 8.3 15.9 -).
 */
inline flow_t flow_of(uint64_t moved)
{
	return moved <= (100u << 20) ? STREAM_NONE : moved <= (256u << 20) ? STREAM_LOADS : STREAM_BOTH;
}

/* The kernel of a flow */
template <typename K> inline K by_flow(flow_t flow, K none, K loads, K both)
{
	return flow == STREAM_NONE ? none : flow == STREAM_LOADS ? loads : both;
}

/* n rows of `bytes` at p, a pitch apart, each element on its own boundary */
inline bool rows_ok(const void *p, uint64_t pitch, uint64_t n, uint64_t bytes, uint32_t element)
{
	return p && (reinterpret_cast<uintptr_t>(p) % element) == 0 && pitch % element == 0 && (n <= 1 || pitch >= bytes) &&
	       pitch < (1ull << 40);
}

} // namespace ofi_amd

#endif
