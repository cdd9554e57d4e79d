/*
 * Batches without tokens and buffers without rows, as the pointers of empty tensors are (NULL), against the stand-in for the HIP runtime.
 */
#define main launch_driver_main
#include "launch_driver.cpp"
#undef main

int main()
{
	static char buffer[4096] __attribute__((aligned(4096)));
	void *const p = buffer;
	float *const f = reinterpret_cast<float *>(p);
	int32_t *const i = reinterpret_cast<int32_t *>(p);
	const int bf = OFI_AMD_BFLOAT16;
	CHECK(ofi_amd_gpu_init() == 0);
	uint32_t rows_copied = 0;
	on_launch = [&](const launch_t &l) {
		rows_copied += l.kernel.find("token_rows_kernel") != std::string::npos || l.kernel.find("token_few_kernel") != std::string::npos;
	};
	auto dispatch = [&](uint32_t tokens, uint32_t most, void *x, void *rows, void *s, void *s_rows) {
		return ofi_amd_token_dispatch(tokens ? p : nullptr, OFI_AMD_INT32, tokens, 2, 8, most, i, tokens ? i : nullptr, most ? i : nullptr, x, 64,
					      rows, 64, 64, s, 16, s_rows, 16, 16, p, ~0ull, nullptr);
	};
	/* no tokens, into buffers of many rows and of none */
	CHECK(dispatch(0, 16, nullptr, p, nullptr, p) == 0 && dispatch(0, 16, nullptr, p, nullptr, nullptr) == 0);
	CHECK(dispatch(0, 0, nullptr, nullptr, nullptr, nullptr) == 0 && dispatch(0, 16, p, p, p, p) == 0);
	/* tokens, but no room for a row */
	CHECK(dispatch(4, 0, p, nullptr, p, nullptr) == 0 && dispatch(5000, 0, p, nullptr, p, nullptr) == 0 && rows_copied == 0);
	/* room and tokens: nothing may be missing */
	CHECK(dispatch(4, 16, nullptr, p, nullptr, nullptr) == -EINVAL && dispatch(4, 16, p, nullptr, nullptr, nullptr) == -EINVAL);
	CHECK(dispatch(4, 16, p, p, nullptr, p) == -EINVAL && dispatch(4, 16, p, p, p, nullptr) == -EINVAL);
	CHECK(rows_copied == 0 && dispatch(4, 16, p, p, p, p) == 0 && rows_copied == 1);
	/* sums and their gradients */
	CHECK(ofi_amd_token_combine(nullptr, 0, 0, i, f, 4, 2, 32, bf, nullptr, 0, p, 64, nullptr) == 0);
	CHECK(ofi_amd_token_combine(nullptr, 0, 0, nullptr, nullptr, 0, 2, 32, bf, nullptr, 0, nullptr, 0, nullptr) == 0);
	CHECK(ofi_amd_token_combine_grad(p, 64, nullptr, 64, 0, i, f, 4, 2, 32, bf, nullptr, 64, f, nullptr) == 0);
	CHECK(ofi_amd_token_combine_grad(p, 64, nullptr, 64, 0, i, f, 4, 2, 32, bf, nullptr, 64, nullptr, nullptr) == 0);
	CHECK(ofi_amd_token_combine_grad(nullptr, 64, p, 64, 16, nullptr, nullptr, 0, 2, 32, bf, p, 64, nullptr, nullptr) == 0);
	CHECK(ofi_amd_token_combine_grad(p, 64, p, 64, 16, i, f, 4, 2, 32, bf, nullptr, 64, nullptr, nullptr) == -EINVAL);
	CHECK(ofi_amd_token_combine_grad(nullptr, 64, nullptr, 64, 0, i, f, 4, 2, 32, bf, nullptr, 64, nullptr, nullptr) == -EINVAL);
	/* norms */
	CHECK(ofi_amd_rms_norm(nullptr, 64, nullptr, 64, p, bf, 0, 32, bf, 0.0f, nullptr, 64, nullptr, 64, nullptr, 32, nullptr, 4, 0, nullptr, nullptr) == 0);
	CHECK(ofi_amd_rms_norm_grad(nullptr, 64, nullptr, 64, nullptr, p, bf, 0, 32, bf, nullptr, 64, nullptr, 64, f, nullptr, 0, nullptr) == 0);
	std::printf("empty: ok\n");
	return 0;
}
