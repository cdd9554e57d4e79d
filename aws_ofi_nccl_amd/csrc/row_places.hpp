/*
 * Where the lanes of a kernel on rows read: plain arithmetic, for the kernels and for the host alike.
 */
#ifndef OFI_AMD_ROW_PLACES_HPP_
#define OFI_AMD_ROW_PLACES_HPP_

#include <cstdint>

namespace ofi_amd {

/* Where the chunk at column `at` is read, and how many of its elements are not its own */
struct place_t {
	uint32_t from, skip;
};
template <uint32_t V> constexpr place_t place_of(uint32_t at, uint32_t width)
{
	const uint32_t from = at < width - V ? at : width - V;
	return { from, at - from };
}

/*
 * Rows of two-byte elements that start between two words.  Loads there run at little over half the rate, so that a chunk is read from
 * the word in front of it (lag elements earlier).  Its last element is then the next lane's first; where the next lane is another
 * wavefront's or another row's, or ends with the row, a load of its own brings that element (for few lanes).  Nothing is read behind the
 * row, and in front of it nothing beyond the word that holds its start.
 */
template <uint32_t V> constexpr uint32_t lag_at(uint64_t row, uint32_t element_size)
{
	return element_size == 2 && V > 1 ? (uint32_t)(row >> 1) & 1u : 0u;
}

/* Of LANES lanes of a row in a wavefront, whether this one, at column `at`, loads the last element itself */
template <uint32_t V, uint32_t LANES> constexpr bool is_lone(uint32_t lane, uint32_t at, uint32_t width)
{
	return (lane & (LANES - 1)) == LANES - 1 || at + 2 * V > width;
}

/* What it loads, at element kRestAt<V> of its chunk: with a word, a row of odd width would end inside what is read */
typedef uint16_t rest_t;
template <uint32_t V> constexpr uint32_t kRestAt = V - 1;

} // namespace ofi_amd

#endif
