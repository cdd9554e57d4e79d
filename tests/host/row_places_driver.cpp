/*
 * The addresses that the lanes of the norms read (csrc/row_places.hpp), for rows of every parity of start, pitch and width: no byte behind
 * a row, in front of it none beyond the word that holds its start, and every element of the row in some lane that is not to pass it over.
 */
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "row_places.hpp"

using namespace ofi_amd;

namespace {

#define CHECK(cond)                                                                                                        \
	do {                                                                                                               \
		if (!(cond)) {                                                                                             \
			std::printf("%s: width %u, pitch %u, row %u of %u at %u, lane %u of %u: bytes %lld..%lld of %lld\n", #cond, width, \
				    pitch, row, rows, (unsigned)start, lane, LANES, (long long)lo, (long long)hi, (long long)(2ll * width)); \
			std::exit(1);                                                                                      \
		}                                                                                                          \
	} while (0)

const uint32_t V = 8; /* two-byte elements of a chunk */
long checked = 0;

/* `lanes` lanes with `chunks` chunks each to a row, LANES of them in a wavefront's part */
template <uint32_t LANES> void rows_of(uint32_t width, uint32_t pitch, uint32_t rows, uint32_t lanes, uint32_t chunks)
{
	for (uint32_t row = 0; row < rows; row++) {
		for (uint32_t first = 0; first < 2; first++) { /* where the first row starts, in elements from a word */
			const uint64_t start = 4096 + 2ull * (first + (uint64_t)row * pitch);
			const uint32_t lag = lag_at<V>(start, 2);
			std::vector<char> seen(width, 0);
			for (uint32_t k = 0; k < chunks; k++) {
				for (uint32_t lane = 0; lane < lanes; lane++) {
					const uint32_t at = (k * lanes + lane) * V;
					const place_t here = place_of<V>(at, width);
					/* bytes from the row's start */
					long long lo = 2ll * here.from - 2ll * lag, hi = lo + 2 * V;
					CHECK(((start + lo) & ~3ull) >= (start & ~3ull) && hi <= 2ll * width);
					if (lag && is_lone<V, LANES>(lane, at, width)) {
						lo = 2ll * (here.from + kRestAt<V>), hi = lo + (long long)sizeof(rest_t);
						CHECK(lo >= 0 && hi <= 2ll * width && lo == 2ll * (here.from + V - 1));
					} else if (lag) { /* the next lane's first word has it */
						const uint32_t theirs = at + V;
						CHECK(lane + 1 < lanes && place_of<V>(theirs, width).from == here.from + V);
					}
					for (uint32_t i = here.skip; i < V; i++) {
						seen[here.from + i]++;
					}
					checked++;
				}
			}
			for (uint32_t c = 0; c < width; c++) {
				if (seen[c] != 1) {
					std::printf("width %u: column %u %d times\n", width, c, seen[c]);
					std::exit(1);
				}
			}
		}
	}
}

} // namespace

int main()
{
	for (uint32_t width = V; width <= 32768; width = width < 1100 ? width + 1 : width * 3 / 2 + (width & 1 ? 0 : 1)) {
		for (uint32_t w = width; w <= width + (width < 1100 ? 0 : 3) && w <= 32768; w++) {
			const uint32_t all = (w + V - 1) / V;
			for (uint32_t pad = 0; pad < 4; pad++) {
				for (uint32_t rows = 1; rows <= 3; rows++) {
					if (all <= 16) {
						rows_of<16>(w, w + pad, rows, 16, 1);
					}
					if (all <= 32) {
						rows_of<32>(w, w + pad, rows, 32, 1);
					}
					for (uint32_t chunks = 1; chunks <= 4; chunks *= 2) {
						const uint32_t lanes = (all + 64 * chunks - 1) / (64 * chunks) * 64;
						if (lanes <= 1024) {
							rows_of<64>(w, w + pad, rows, lanes, chunks);
						}
					}
				}
			}
		}
	}
	std::printf("%ld loads: ok\n", checked);
	return 0;
}
