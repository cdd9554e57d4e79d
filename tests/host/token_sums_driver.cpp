/*
 * The launches of the table of many pairs, seen by the stand-in for the HIP runtime: with more than 128 tiles their counts are summed up by
 * a launch of its own, so that no tile of the table has to look at all the others'.
 */
#define main launch_driver_main
#include "launch_driver.cpp"
#undef main

int main()
{
	static char buffer[4096] __attribute__((aligned(4096)));
	void *const p = buffer;
	int32_t *const i = reinterpret_cast<int32_t *>(p);
	CHECK(ofi_amd_gpu_init() == 0);
	for (const uint32_t n : { 1u, 8192u, 8193u, 1u << 18, 128u << 13, (128u << 13) + 1, 1u << 24, 1u << 28, 0x7fffffffu }) {
		for (const uint32_t experts : { 1u, 16u, 17u, 1000u, 1024u }) {
			std::vector<uint32_t> tiles; /* of each launch of counts: 0, or those that are summed up */
			uint32_t of_table = 0;
			on_launch = [&](const launch_t &l) {
				CHECK((uint64_t)l.grid.x * l.block.x < 1ull << 32 && l.block.x == 1024);
				if (l.kernel.find("token_count_kernel") != std::string::npos) {
					CHECK(of_table == 0);
					tiles.push_back(l.arg<uint32_t>(4));
					CHECK(tiles.back() == 0 || (tiles.back() == l.grid.x && l.grid.x * 16 >= experts));
				} else {
					of_table = l.arg<uint32_t>(3);
				}
			};
			CHECK(ofi_amd_token_dispatch(p, OFI_AMD_INT64, n, 1, experts, n, i, i, i, nullptr, 0, nullptr, 0, 0, nullptr, 0, nullptr, 0, 0, p,
						     ~0ull, nullptr) == 0);
			CHECK(of_table >= 1 && tiles.size() == (of_table > 128 ? 2u : of_table > 1 ? 1u : 0u));
			CHECK(tiles.empty() || tiles[0] == 0);
			CHECK(tiles.size() < 2 || tiles[1] == of_table);
		}
	}
	std::printf("sums: ok\n");
	return 0;
}
