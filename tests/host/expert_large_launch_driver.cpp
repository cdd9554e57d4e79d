/*
 * The largest launches of the experts' products, seen by the stand-in for the HIP runtime: more tiles than one launch can have, with
 * workgroups of every size, and a runtime that refuses one of several launches.
 */
#define main launch_driver_main
#define hipLaunchKernel launch_as_asked
#include "launch_driver.cpp"
#undef hipLaunchKernel
#undef main

namespace {

char buffer[4096] __attribute__((aligned(4096)));
void *const p = buffer;
float *const f = reinterpret_cast<float *>(buffer);
int32_t *const offset = reinterpret_cast<int32_t *>(buffer);
const int bf = OFI_AMD_BFLOAT16, f16 = OFI_AMD_FLOAT16, f32 = OFI_AMD_FLOAT32, e4m3 = OFI_AMD_E4M3;

struct call_t {
	uint32_t rows, experts, width, n; /* from `width` to n columns */
};

/* Rows and weights without room between them */
int gated(const call_t &c, int type, int out, int saved = 0)
{
	const uint64_t size = type == e4m3 ? 1 : 2;
	return ofi_amd_expert_gated(p, c.width * size, f, 1 << 20, type, offset, c.experts, c.rows, p, c.width * size, 1ull << 45, f, c.width, c.n,
				    OFI_AMD_SILU, p, 1 << 24, out, f, 1 << 20, saved ? p : nullptr, 1 << 24, saved, f, 1 << 20, nullptr);
}

int product(const call_t &c)
{
	return ofi_amd_expert_product(p, c.width * 2, nullptr, 0, f16, offset, c.experts, c.rows, p, c.width * 2, 1ull << 45, nullptr, c.width, c.n, nullptr, 0,
				      0, nullptr, 0, p, 1 << 24, f16, nullptr, 0, nullptr, 0, 0, nullptr, 0, nullptr);
}

int back(const call_t &c, bool hidden)
{
	return hidden ? ofi_amd_expert_hidden_grad(p, c.width * 2, f16, offset, c.experts, c.rows, p, c.n * 2, 1ull << 45, c.width, c.n, 0, OFI_AMD_SILU, p,
						   1 << 24, f16, nullptr, 0, p, 1 << 24, nullptr, 0, nullptr)
		      : ofi_amd_expert_rows_grad(p, c.width * 2, f16, offset, c.experts, c.rows, p, c.n * 2, 1ull << 45, c.n, c.width, nullptr, 0, p, 1 << 24,
						 nullptr);
}

int weights(const call_t &c)
{
	return ofi_amd_expert_weight_grad(p, c.width * 2, p, c.n * 2, f16, offset, c.experts, c.rows, c.n, c.width, nullptr, p, 1 << 24, 1ull << 45, f32, nullptr,
					  f, nullptr);
}

int calls, refused_at = -1;

struct seen_t {
	uint64_t workgroups = 0, next = 0;
	uint32_t lanes = 0;
	int launches = 0;
	bool whole = true;
};

/* What a call launches: every launch is taken, of whole eighths, the same number of lanes, and begins where the one before ended */
template <typename F> seen_t seen(F call, int want = 0)
{
	seen_t s;
	bool sane = true;
	on_launch = [&](const launch_t &l) {
		sane = sane && (uint64_t)l.grid.x * l.block.x < (1ull << 32) && l.grid.x % 8 == 0 && (s.lanes == 0 || s.lanes == l.block.x);
		s.lanes = l.block.x;
		s.workgroups += l.grid.x;
		s.launches++;
	};
	calls = 0;
	s.whole = call() == want && sane && calls == s.launches + (refused_at >= 0);
	return s;
}

int large()
{
	/* 8 rows an expert and 128 columns that share a scale: workgroups of 1024 lanes */
	const call_t exact = { 512, 512, 16, 1u << 20 }, most = { 8192, 1024, 16, 1u << 20 };
	for (const int type : { f16, e4m3 }) {
		for (const call_t &c : { exact, most }) {
			const uint64_t row_tiles = (c.rows - c.experts) / 16 + c.experts, tiles = row_tiles * ((1u << 20) / 128);
			const seen_t s = seen([&] { return gated(c, type, e4m3); });
			CHECK(s.whole && s.lanes == 1024 && s.workgroups == tiles && s.launches == (int)((tiles * 1024 + (1ull << 31) - 1) >> 31));
			const seen_t kept = seen([&] { return gated(c, type, type == f16 ? f16 : bf, e4m3); });
			CHECK(kept.whole && kept.lanes == 1024 && kept.workgroups == tiles);
		}
	}
	/* 512 lanes and 256: products of more rows, and their gradients */
	const call_t rows = { 0x7fffffffu, 1, 64, 4096 };
	for (int what = 0; what < 3; what++) {
		const seen_t s = seen([&] { return what == 0 ? product(rows) : back(rows, what == 1); });
		const uint64_t high = what == 0 ? 256 : 128;
		CHECK(s.whole && s.lanes == (what == 0 ? 512u : 256u) && s.launches > 1 && s.workgroups >= 16 * ((0x7fffffffull + high - 1) / high));
	}
	const call_t wide = { 64, 1024, 1u << 13, 1u << 17 };
	const seen_t s = seen([&] { return weights(wide); });
	CHECK(s.whole && s.lanes == 256 && s.launches > 1 && s.workgroups == 1024ull * (wide.width / 128) * (wide.n / 256));
	return 0;
}

/* A launch that the runtime refuses is the call's last, and the call says so */
int refused()
{
	const call_t c = { 8192, 1024, 16, 1u << 20 };
	const int all = seen([&] { return gated(c, f16, e4m3); }).launches;
	CHECK(all > 2);
	for (refused_at = 0; refused_at < all; refused_at++) {
		const seen_t s = seen([&] { return gated(c, f16, e4m3); }, -EIO);
		CHECK(s.whole && s.launches == refused_at);
	}
	refused_at = -1;
	CHECK(seen([&] { return gated(c, f16, e4m3); }).whole); /* and nothing of it is left */
	return 0;
}

} // namespace

extern "C" hipError_t hipLaunchKernel(const void *f, dim3 grid, dim3 block, void **args, size_t shared, hipStream_t stream)
{
	const int call = calls++;
	return call == refused_at ? last_error = hipErrorInvalidConfiguration : launch_as_asked(f, grid, block, args, shared, stream);
}

int main(int argc, char **argv)
{
	const std::map<std::string, int (*)()> parts = { { "large", large }, { "refused", refused } };
	CHECK(argc == 2 && parts.count(argv[1]) && ofi_amd_gpu_init() == 0);
	const int rc = parts.at(argv[1])();
	std::printf("%s: %s\n", argv[1], rc == 0 ? "ok" : "failed");
	return rc;
}
