/*
 * What the kernels on rows of numbers share: 16-byte pieces of a row as floats, and sums and maxima over lanes.
 *
 * A row is cut into chunks of 16 bytes, one per lane.  Chunks are accessed as 16-byte words at whatever address the
 * row starts (the global memory path takes any alignment); only the last chunk of a row whose width is no whole number of
 * chunks goes element by element.
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

template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) chunk_t {
	T v __attribute__((ext_vector_type(16 / sizeof(T))));
};
/* 16 bytes of anything at any address */
struct __attribute__((packed, aligned(1))) any16_t {
	u32x4_t v;
};

/* `left` elements of the row remain at p, at least one; those beyond read as 0 */
template <typename T> __device__ __forceinline__ void load_chunk(const T *__restrict__ p, uint32_t left, float (&f)[kChunk<T>])
{
	constexpr uint32_t V = kChunk<T>;
	if (left >= V) {
		const auto c = reinterpret_cast<const chunk_t<T> *>(p)->v;
#pragma unroll
		for (uint32_t i = 0; i < V; i++) {
			f[i] = (float)c[i];
		}
	} else {
#pragma unroll
		for (uint32_t i = 0; i < V; i++) {
			f[i] = i < left ? (float)p[i] : 0.0f;
		}
	}
}

/* Each element is rounded to the row's type once, to nearest even */
template <typename T> __device__ __forceinline__ void store_chunk(T *__restrict__ p, uint32_t left, const float (&f)[kChunk<T>])
{
	constexpr uint32_t V = kChunk<T>;
	if (left >= V) {
		chunk_t<T> c;
#pragma unroll
		for (uint32_t i = 0; i < V; i++) {
			c.v[i] = (T)f[i];
		}
		*reinterpret_cast<chunk_t<T> *>(p) = c;
	} else {
#pragma unroll
		for (uint32_t i = 0; i < V; i++) {
			if (i < left) {
				p[i] = (T)f[i];
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

/* Calls f with a value of the row's type (checked before) */
template <typename F> inline void with_row_type(int type, F f)
{
	if (type == OFI_AMD_BFLOAT16) {
		f(bf16_t{});
	} else if (type == OFI_AMD_FLOAT16) {
		f(f16_t{});
	} else {
		f(float{});
	}
}

/* n rows of `bytes` at p, a pitch apart, each element on its own boundary */
inline bool rows_ok(const void *p, uint64_t pitch, uint64_t n, uint64_t bytes, uint32_t element)
{
	return p && (reinterpret_cast<uintptr_t>(p) % element) == 0 && pitch % element == 0 && (n <= 1 || pitch >= bytes) &&
	       pitch < (1ull << 40);
}

} // namespace ofi_amd

#endif
