/*
 * The launches of the experts' products, seen by the stand-in for the HIP runtime: there is a workgroup for every tile that the experts'
 * rows can make, however they are spread, and no launch is larger than the runtime numbers.  What the calls refuse is here too, as it
 * needs no GPU.
 */
#include <random>
#include <regex>

#define main launch_driver_main
#include "launch_driver.cpp"
#undef main

namespace {

char buffer[4096] __attribute__((aligned(4096)));
void *const p = buffer;
float *const f = reinterpret_cast<float *>(buffer);
int32_t *const offset = reinterpret_cast<int32_t *>(buffer);
const int bf = OFI_AMD_BFLOAT16, f16 = OFI_AMD_FLOAT16, f32 = OFI_AMD_FLOAT32, e4m3 = OFI_AMD_E4M3;

/* The k-th last whole number among a kernel's template arguments.  (The demangler misreads bfloat16 and what follows it: float16 here.) */
uint32_t parameter(const std::string &name, size_t k)
{
	std::vector<uint32_t> all;
	const std::string in = name.substr(0, name.find(">("));
	static const std::regex mangled("Lj([0-9]+)E"), plain("[<, ]([0-9]+)u(?=,|$)");
	const std::regex &number = name.compare(0, 2, "_Z") == 0 ? mangled : plain;
	for (std::sregex_iterator i(in.begin(), in.end(), number), end; i != end; ++i) {
		all.push_back((uint32_t)std::atoi((*i)[1].str().c_str()));
	}
	if (k >= all.size()) {
		std::fprintf(stderr, "%s\n", name.c_str());
		return 0;
	}
	return all[all.size() - 1 - k];
}

bool is(const launch_t &l, const char *kernel) { return l.kernel.find(kernel) != std::string::npos; }

struct call_t {
	uint32_t rows, experts, width, n;
	uint64_t pitch;
};

int gated(const call_t &c, int type = f16, int out = f16, int saved = 0, int act = OFI_AMD_SILU)
{
	return ofi_amd_expert_gated(p, c.pitch, f, 1 << 20, type, offset, c.experts, c.rows, p, c.pitch, 1ull << 45, f, c.width, c.n, act, p, 1 << 24, out, f,
				    1 << 20, saved ? p : nullptr, 1 << 24, saved, f, 1 << 20, nullptr);
}

int product(const call_t &c, int type = f16, int out = f16, const void *residual = nullptr)
{
	return ofi_amd_expert_product(p, c.pitch, f, 1 << 20, type, offset, c.experts, c.rows, p, c.pitch, 1ull << 45, f, c.width, c.n, nullptr, 0, 0, residual,
				      1 << 24, p, 1 << 24, out, f, 1 << 20, nullptr, 0, 0, nullptr, 0, nullptr);
}

int back(const call_t &c, bool hidden)
{
	return hidden ? ofi_amd_expert_hidden_grad(p, c.pitch, f16, offset, c.experts, c.rows, p, 1 << 24, 1ull << 45, c.width, c.n, 1, OFI_AMD_SILU, p,
						   1 << 24, f16, nullptr, 0, p, 1 << 24, p, 1 << 24, nullptr)
		      : ofi_amd_expert_rows_grad(p, c.pitch, f16, offset, c.experts, c.rows, p, 1 << 24, 1ull << 45, c.n, c.width, nullptr, 0, p, 1 << 24, nullptr);
}

int weights(const call_t &c)
{
	return ofi_amd_expert_weight_grad(p, c.pitch, p, 1 << 24, f16, offset, c.experts, c.rows, c.n, c.width, nullptr, p, 1 << 24, 1ull << 45, f32, nullptr, f,
					  nullptr);
}

int spreads()
{
	std::mt19937_64 rng(5);
	uint64_t workgroups = 0;
	uint32_t bm = 0, bn = 0;
	bool sane = true;
	on_launch = [&](const launch_t &l) {
		sane = sane && l.grid.x >= 1 && l.grid.y == 1 && l.grid.z == 1 && l.block.x <= 1024 && l.block.x % 64 == 0 && l.grid.x % 8 == 0 &&
		       (uint64_t)l.grid.x * l.block.x < (1ull << 32);
		const uint32_t last = parameter(l.kernel, 0), middle = parameter(l.kernel, 1), first = parameter(l.kernel, 2);
		if (is(l, "expert_few_kernel")) {
			bm = 16 * first;
			bn = 2 * 16 * middle;
			sane = sane && l.block.x == 64 * middle * last;
		} else {
			bm = 16 * first * last;
			bn = 256;
			sane = sane && l.block.x == 64 * first * middle;
		}
		workgroups += l.grid.x;
	};
	const uint32_t sizes[] = { 1, 2, 7, 8, 9, 16, 63, 64, 65, 200, 255, 256, 257, 1000, 4096, 40000, 1u << 20 };
	for (const uint32_t experts : { 1u, 2u, 5u, 32u, 64u, 65u, 1024u }) {
		for (const uint32_t rows : sizes) {
			for (const uint32_t n : { 1u, 8u, 128u, 136u, 1000u, 4096u, 16384u }) {
				for (const uint64_t pitch : { 4096ull, 4098ull }) {
					const call_t c = { rows, experts, 2048, n, pitch };
					for (int what = 0; what < 5; what++) {
						workgroups = 0;
						const int rc = what == 0   ? gated(c, f16, rows % 2 ? f16 : e4m3)
							       : what == 1 ? product(c)
							       : what == 2 ? back(c, true)
							       : what == 3 ? back(c, false)
									   : weights(c);
						CHECK(rc == 0 && sane && workgroups > 0);
						const uint64_t n_tiles = what == 0 ? (n + bn / 2 - 1) / (bn / 2) : (n + bn - 1) / bn;
						if (what == 4) {
							CHECK(workgroups >= experts * n_tiles * ((2048 + bm - 1) / bm));
							continue;
						}
						/* the worst spread: as many experts as there can be with one row, the rest in one; and some others */
						const uint64_t used = experts < rows ? experts : rows;
						CHECK(workgroups >= n_tiles * (used - 1 + (rows - used + 1 + bm - 1) / bm));
						for (int k = 0; k < 4; k++) {
							uint64_t need = 0, left = rows;
							for (uint32_t e = 0; e < experts; e++) {
								const uint64_t mine = e + 1 == experts ? left : left ? rng() % (k < 2 ? left + 1 : 2 * rows / experts + 2) : 0;
								const uint64_t m = mine < left ? mine : left;
								need += (m + bm - 1) / bm;
								left -= m;
							}
							CHECK(workgroups >= n_tiles * need);
						}
					}
				}
			}
		}
	}
	/* several launches */
	workgroups = 0;
	CHECK(product({ 0x7fffffffu, 1, 64, 4096, 128 }) == 0 && sane && workgroups >= 16ull * 0x7fffffffull / 256);
	return 0;
}

int refusals()
{
	int launches = 0;
	on_launch = [&](const launch_t &) { launches++; };
	const call_t good = { 100, 4, 64, 48, 128 };
	auto with = [&](uint32_t rows, uint32_t experts, uint32_t width, uint32_t n, uint64_t pitch) { return call_t{ rows, experts, width, n, pitch }; };
	for (int what = 0; what < 5; what++) {
		auto call = [&](const call_t &c) {
			return what == 0 ? gated(c) : what == 1 ? product(c) : what == 2 ? back(c, true) : what == 3 ? back(c, false) : weights(c);
		};
		CHECK(call(with(100, 0, 64, 48, 128)) == -EINVAL && call(with(100, 4, 0, 48, 128)) == -EINVAL && call(with(100, 4, 64, 0, 128)) == -EINVAL);
		CHECK(call(with(100, 1025, 64, 48, 128)) == -E2BIG && call(with(1u << 31, 4, 64, 48, 128)) == -E2BIG);
		CHECK(call(with(100, 4, (1u << 20) + 1, 48, 1 << 24)) == -E2BIG && call(with(100, 4, 64, (1u << 20) + 1, 128)) == -E2BIG);
		CHECK(call(with(100, 4, 64, 48, 126)) == -EINVAL && call(with(100, 4, 64, 48, 129)) == -EINVAL && call(with(100, 4, 64, 48, 1ull << 40)) == -EINVAL);
		CHECK(launches == 0 && call(good) == 0 && launches == 1);
		launches = 0;
	}
	CHECK(product(with(0x7fffffffu, 1, 64, 1u << 20, 128)) == -E2BIG); /* more tiles than are numbered */
	/* types and activations */
	for (const int type : { f32, OFI_AMD_INT32, 0 }) {
		CHECK(gated(good, type) == -EINVAL && gated(good, bf, type) == -EINVAL && (type == 0 || gated(good, bf, bf, type) == -EINVAL));
		CHECK(product(good, type) == -EINVAL && product(good, bf, type) == -EINVAL);
	}
	CHECK(gated(good, bf, f16) == -EINVAL && gated(good, f16, bf) == -EINVAL && gated(good, bf, bf, f16) == -EINVAL);
	CHECK(gated(good, bf, bf, 0, 4) == -EINVAL && gated(good, bf, bf, 0, -1) == -EINVAL);
	CHECK(product(good, bf, e4m3, p) == -EINVAL); /* a residual beside an 8-bit output */
	CHECK(launches == 0 && gated(good, e4m3, e4m3, e4m3) == 0 && product(good, bf, e4m3) == 0 && product(good, bf, bf, p) == 0 && launches == 3);
	launches = 0;
	/* what may not be missing, and where it has to lie */
	auto gate = [&](const void *rows, const float *scale, int type, const int32_t *at, uint32_t experts, uint32_t max_rows, const void *w, uint64_t w_pitch,
			uint64_t e_pitch, const float *w_scale, void *out, uint64_t out_pitch, int out_type, float *out_scale) {
		return ofi_amd_expert_gated(rows, 128, scale, 4, type, at, experts, max_rows, w, w_pitch, e_pitch, w_scale, 64, 48, OFI_AMD_SILU, out, out_pitch,
					    out_type, out_scale, 4, nullptr, 0, 0, nullptr, 0, nullptr);
	};
	CHECK(gate(nullptr, f, bf, offset, 4, 10, p, 128, 128 * 96, f, p, 96, bf, f) == -EINVAL);
	CHECK(gate(p, f, bf, nullptr, 4, 10, p, 128, 128 * 96, f, p, 96, bf, f) == -EINVAL); /* one expert without offsets, not four */
	CHECK(gate(p, f, bf, reinterpret_cast<int32_t *>(buffer + 2), 4, 10, p, 128, 128 * 96, f, p, 96, bf, f) == -EINVAL);
	CHECK(gate(p, f, bf, offset, 4, 10, nullptr, 128, 128 * 96, f, p, 96, bf, f) == -EINVAL);
	CHECK(gate(p, f, bf, offset, 4, 10, p, 126, 128 * 96, f, p, 96, bf, f) == -EINVAL);
	CHECK(gate(p, f, bf, offset, 4, 10, p, 128, 128 * 96 - 2, f, p, 96, bf, f) == -EINVAL); /* experts that overlap */
	CHECK(gate(p, f, bf, offset, 4, 10, p, 128, 128 * 96 + 1, f, p, 96, bf, f) == -EINVAL);
	CHECK(gate(p, f, bf, offset, 4, 10, buffer + 1, 128, 128 * 96, f, p, 96, bf, f) == -EINVAL);
	CHECK(gate(p, f, bf, offset, 4, 10, p, 128, 128 * 96, f, nullptr, 96, bf, f) == -EINVAL);
	CHECK(gate(p, f, bf, offset, 4, 10, p, 128, 128 * 96, f, p, 94, bf, f) == -EINVAL);
	CHECK(gate(p, f, bf, offset, 4, 10, p, 128, 128 * 96, f, p, 96, e4m3, nullptr) == -EINVAL);
	CHECK(gate(p, nullptr, e4m3, offset, 4, 10, p, 128, 128 * 96, f, p, 96, bf, f) == -EINVAL);
	CHECK(gate(p, f, e4m3, offset, 4, 10, p, 128, 128 * 96, nullptr, p, 96, bf, f) == -EINVAL);
	CHECK(launches == 0);
	CHECK(gate(p, nullptr, bf, offset, 4, 10, p, 128, 128 * 96, nullptr, p, 96, bf, nullptr) == 0 && launches == 1);
	CHECK(gate(p, nullptr, bf, nullptr, 1, 10, p, 128, 0, nullptr, p, 96, bf, nullptr) == 0 && launches == 2);
	/* no rows: nothing to do, and nothing has to be there */
	CHECK(gate(nullptr, nullptr, bf, offset, 4, 0, nullptr, 0, 0, nullptr, nullptr, 0, bf, nullptr) == 0 && launches == 2);
	auto hidden = [&](int gated_, int saved_type, const void *saved, const float *scale, void *dsaved, uint64_t dsaved_pitch, void *h) {
		return ofi_amd_expert_hidden_grad(p, 128, bf, offset, 4, 10, p, 96, 96 * 64, 64, 48, gated_, OFI_AMD_GELU, saved, 192, saved_type, scale, 8, dsaved,
						  dsaved_pitch, h, 96, nullptr);
	};
	CHECK(hidden(2, bf, p, f, p, 192, p) == -EINVAL && hidden(1, f16, p, f, p, 192, p) == -EINVAL && hidden(1, bf, nullptr, f, p, 192, p) == -EINVAL);
	CHECK(hidden(1, e4m3, p, nullptr, p, 192, p) == -EINVAL && hidden(1, bf, p, f, nullptr, 192, p) == -EINVAL && hidden(1, bf, p, f, p, 190, p) == -EINVAL);
	CHECK(hidden(1, bf, p, f, p, 192, buffer + 1) == -EINVAL && launches == 2);
	CHECK(hidden(1, e4m3, p, f, p, 192, nullptr) == 0 && hidden(0, bf, p, nullptr, p, 96, p) == 0 && launches == 4);
	auto weight = [&](const void *dout, const void *rows, uint32_t max_rows, const void *add, void *dw, int type, const float *badd, float *db) {
		return ofi_amd_expert_weight_grad(dout, 96, rows, 128, bf, offset, 4, max_rows, 64, 48, add, dw, 256, 256 * 48, type, badd, db, nullptr);
	};
	CHECK(weight(nullptr, p, 10, nullptr, p, f32, nullptr, nullptr) == -EINVAL && weight(p, nullptr, 10, nullptr, p, f32, nullptr, nullptr) == -EINVAL);
	CHECK(weight(p, p, 10, nullptr, nullptr, f32, nullptr, nullptr) == -EINVAL && weight(p, p, 10, nullptr, p, f16, nullptr, nullptr) == -EINVAL);
	CHECK(weight(p, p, 10, buffer + 2, p, f32, nullptr, nullptr) == -EINVAL && weight(p, p, 10, nullptr, p, e4m3, nullptr, nullptr) == -EINVAL);
	CHECK(weight(p, p, 10, nullptr, p, f32, nullptr, reinterpret_cast<float *>(buffer + 2)) == -EINVAL && launches == 4);
	CHECK(weight(nullptr, nullptr, 0, nullptr, p, f32, nullptr, f) == 0 && weight(p, p, 10, p, p, bf, f, f) == 0 && launches == 6);
	return 0;
}

} // namespace

int main(int argc, char **argv)
{
	const std::map<std::string, int (*)()> parts = { { "spreads", spreads }, { "refusals", refusals } };
	CHECK(argc == 2 && parts.count(argv[1]) && ofi_amd_gpu_init() == 0);
	const int rc = parts.at(argv[1])();
	std::printf("%s: %s\n", argv[1], rc == 0 ? "ok" : "failed");
	return rc;
}
