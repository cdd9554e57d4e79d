/*
 * Calls with room for far more rows than they have pairs, seen by the stand-in for the HIP runtime: the rows that no pair can have are
 * shared by workgroups of their own, so that no lane has more than a few of them as long as the chip is not full.
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
	for (const uint32_t n : { 0u, 1u, 8u, 200u, 1000u, 3000u, 40000u }) {
		for (const uint32_t rows : { 0u, 1u, 1u << 10, 1u << 16, (1u << 20) + 3, 1u << 24, 0x7fffffffu }) {
			for (const bool copies : { false, true }) {
				const uint32_t pairs = n * 2;
				uint64_t lanes = 0; /* that fill */
				uint32_t launches = 0;
				on_launch = [&](const launch_t &l) {
					const bool few = l.kernel.find("token_few_kernel") != std::string::npos;
					if (few || l.kernel.find("token_place_kernel") != std::string::npos) {
						const uint32_t others = few ? n + 1 : l.arg<uint32_t>(3);
						CHECK(l.grid.x >= others && (rows > pairs || l.grid.x == others));
						CHECK((uint64_t)l.grid.x * l.block.x < 1ull << 32);
						lanes = (uint64_t)(l.grid.x - others) * l.block.x;
						launches++;
					}
				};
				CHECK(ofi_amd_token_dispatch(p, OFI_AMD_INT64, n, 2, 60, rows, i, i, i, copies ? p : nullptr, 64, copies ? p : nullptr, 64, 64,
							     nullptr, 0, nullptr, 0, 0, p, ~0ull, nullptr) == 0);
				const uint64_t left = rows > pairs ? rows - pairs : 0;
				CHECK(launches == 1 && (lanes * 16 >= left || lanes >= 2048 * 64));
			}
		}
	}
	std::printf("room: ok\n");
	return 0;
}
