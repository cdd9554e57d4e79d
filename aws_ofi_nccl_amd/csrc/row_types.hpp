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

/* Where the chunk at column `at` is read, and how many of its elements are not its own */
struct place_t {
	uint32_t from, skip;
};
template <uint32_t V> __device__ __forceinline__ place_t place_of(uint32_t at, uint32_t width)
{
	const uint32_t from = min(at, width - V);
	return { from, at - from };
}

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
	raw_t<T, V> c;
#pragma unroll
	for (uint32_t i = 0; i < V; i++) {
		c[i] = (T)f[i];
	}
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
		v = op(v, (uint32_t)__shfl_xor((int)v, 16));
	}
	if (LANES >= 64) {
		v = op(v, (uint32_t)__shfl_xor((int)v, 32));
	}
	return v;
}

template <int LANES> __device__ __forceinline__ float sum_over(float v)
{
	return __uint_as_float(over_lanes<LANES>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
		return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
	}));
}

/* Maximum of absolute values given as their bits: a NaN's are above an infinity's, so that a NaN comes out */
template <int LANES> __device__ __forceinline__ uint32_t max_bits_over(uint32_t v)
{
	return over_lanes<LANES>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

__device__ __forceinline__ uint32_t abs_bits(float f) { return __float_as_uint(f) & 0x7fffffffu; }

/* The same in every wavefront of a workgroup of WAVES of them; s: WAVES words of LDS that nothing else uses meanwhile */
template <int WAVES> __device__ __forceinline__ float block_sum(float v, float *s)
{
	v = sum_over<64>(v);
	if (WAVES == 1) {
		return v;
	}
	if ((threadIdx.x & 63u) == 0) {
		s[threadIdx.x >> 6] = v;
	}
	__syncthreads();
	float total = s[0];
#pragma unroll
	for (int w = 1; w < WAVES; w++) {
		total += s[w];
	}
	return total;
}

template <int WAVES> __device__ __forceinline__ uint32_t block_max_bits(uint32_t v, uint32_t *s)
{
	v = max_bits_over<64>(v);
	if (WAVES == 1) {
		return v;
	}
	if ((threadIdx.x & 63u) == 0) {
		s[threadIdx.x >> 6] = v;
	}
	__syncthreads();
	uint32_t most = s[0];
#pragma unroll
	for (int w = 1; w < WAVES; w++) {
		most = s[w] > most ? s[w] : most;
	}
	return most;
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

/* Whether every chunk of the rows lies within a line: rows that are read past the caches (STREAM) have to.  A chunk across two
 * lines would fetch both again for its neighbour. */
inline bool on_chunks(const void *p, uint64_t pitch)
{
	return ((reinterpret_cast<uintptr_t>(p) | pitch) & 15u) == 0;
}

/* n rows of `bytes` at p, a pitch apart, each element on its own boundary */
inline bool rows_ok(const void *p, uint64_t pitch, uint64_t n, uint64_t bytes, uint32_t element)
{
	return p && (reinterpret_cast<uintptr_t>(p) % element) == 0 && pitch % element == 0 && (n <= 1 || pitch >= bytes) &&
	       pitch < (1ull << 40);
}

} // namespace ofi_amd

#endif
