/*
 * The launches of norms and token exchanges, seen by the stand-in for the HIP runtime: at sizes from nothing to the largest that is
 * taken, every row, token and pair is in exactly one launch, rows fit the lanes they are given, and no launch is larger than the
 * runtime numbers.  What the calls refuse is here too, as it needs no GPU.
 */
#include <regex>

#define main launch_driver_main
#include "launch_driver.cpp"
#undef main

namespace {

char buffer[4096] __attribute__((aligned(4096)));
void *const p = buffer;
const uint64_t pitch = 1 << 20; /* no row is longer than what is tried here; nothing is read */

/* The k-th last whole number among a kernel's template arguments.  (The demangler misreads bfloat16 and what
 * follows it, or leaves the name as it is.) */
int parameter(const std::string &name, size_t k)
{
	static std::map<std::string, std::vector<int>> known;
	std::vector<int> &all = known[name];
	const std::string in = all.empty() ? name.substr(0, name.find(">(")) : std::string();
	static const std::regex mangled("L[ij]([0-9]+)E"), plain("[<, ]([0-9]+)u?(?=,|$)");
	const std::regex &number = name.compare(0, 2, "_Z") == 0 ? mangled : plain;
	for (std::sregex_iterator i(in.begin(), in.end(), number), end; i != end; ++i) {
		all.push_back(std::atoi((*i)[1].str().c_str()));
	}
	if (k >= all.size()) {
		std::printf("%s\n", name.c_str());
	}
	CHECK(k < all.size());
	return all[all.size() - 1 - k];
}

bool is(const launch_t &l, const char *kernel) { return l.kernel.find(kernel) != std::string::npos; }

void sane(const launch_t &l)
{
	CHECK(l.grid.x >= 1 && l.grid.y == 1 && l.grid.z == 1 && l.block.x % 64 == 0);
	CHECK(l.block.x * l.block.y * l.block.z <= 1024 && l.shared <= 160 * 1024 - 8192);
}

const struct {
	int type;
	uint32_t size;
} kTypes[] = { { OFI_AMD_BFLOAT16, 2 }, { OFI_AMD_FLOAT16, 2 }, { OFI_AMD_FLOAT32, 4 } };
const uint32_t kWidths[] = { 1, 3, 4, 7, 8, 9, 63, 64, 127, 128, 129, 255, 256, 257, 512, 513, 1024, 2047, 4095, 4096, 4097, 8192, 8193,
			     16384, 16385, 24000, 32768 };
const uint32_t kMany[] = { 1, 2, 15, 16, 17, 255, 256, 257, 1023, 4097, 1u << 19, (1u << 21) - 1, 1u << 21, (1u << 21) + 1, (1u << 22) + 1,
			   0x7fffffffu };

int norms()
{
	for (const auto &t : kTypes) {
		for (const uint32_t width : kWidths) {
			for (const uint32_t n : kMany) {
				uint64_t next = 0;
				const uint32_t chunk = width >= 16 / t.size ? 16 / t.size : 1;
				on_launch = [&](const launch_t &l) {
					sane(l);
					CHECK(is(l, "rms_norm_kernel") && l.arg<uint32_t>(6) == n && l.arg<uint32_t>(7) == width);
					const int lanes = parameter(l.kernel, 0), chunks = parameter(l.kernel, 1);
					const uint64_t rows = lanes < 64 ? l.block.x / (uint32_t)lanes : 1;
					CHECK((uint64_t)(lanes < 64 ? (uint32_t)lanes : l.block.x) * (uint32_t)chunks * chunk >= width);
					CHECK(l.arg<uint32_t>(5) == next); /* where the last one ended */
					next += l.grid.x * rows;
				};
				CHECK(ofi_amd_rms_norm(p, pitch, p, pitch, p, t.type, n, width, t.type, 1e-6f, p, pitch, nullptr, 0, p, pitch,
						       reinterpret_cast<float *>(p), pitch, 128, nullptr, nullptr) == 0);
				CHECK(next >= n && next < (uint64_t)n + 16);
				if (n > 5000 && width > 300) {
					continue; /* the gradient is the same for all of those */
				}
				int gains = 0, rows = 0;
				on_launch = [&](const launch_t &l) {
					sane(l);
					gains += is(l, "gain_kernel");
					if (is(l, "gain_kernel")) {
						CHECK((uint64_t)l.grid.x * 32 >= width && l.arg<uint32_t>(2) <= 512);
						return;
					}
					rows++;
					CHECK(l.block.x >= 64 && l.arg<uint32_t>(8) == n && l.arg<uint32_t>(9) == width);
					if (is(l, "few_kernel")) {
						CHECK(n <= 256 && l.grid.x == n + (width + 63) / 64 && (uint64_t)l.block.x * chunk >= width);
						gains++;
					} else {
						const uint64_t held = is(l, "wide_kernel") ? (uint64_t)parameter(l.kernel, 0) : 1;
						CHECK(l.grid.x == (n < 512 ? n : 512) && l.block.x * held * chunk >= width);
						CHECK(is(l, "wide_kernel") || l.block.x * l.block.y <= 64u * (uint32_t)parameter(l.kernel, 0));
					}
				};
				const uint64_t need = ofi_amd_rms_norm_grad_work_bytes(n, width);
				CHECK(need == (uint64_t)(n < 512 ? n : 512) * width * 4);
				for (void *dx : { p, static_cast<void *>(buffer + 1024) }) {
					gains = rows = 0;
					CHECK(ofi_amd_rms_norm_grad(p, pitch, p, pitch, reinterpret_cast<float *>(p), p, t.type, n, width, t.type,
								    nullptr, 0, dx, pitch, reinterpret_cast<float *>(p), p, need, nullptr) == 0);
					CHECK(gains == 1 && rows == 1);
				}
			}
		}
	}
	return 0;
}

int tokens()
{
	const uint32_t choices[] = { 1, 2, 7, 8, 9, 64 };
	for (const uint32_t top_k : choices) {
		for (const uint32_t n : kMany) {
			if ((uint64_t)n * top_k > 0x7fffffffu) {
				continue;
			}
			const uint32_t pairs = n * top_k, experts = 1 + n % 1024;
			for (const uint32_t bytes : { 1u, 100u, 4096u, 14336u, 16384u, 1u << 20 }) {
				/* scales by their place, by token, too long for the former */
				const uint32_t scale = bytes == 100 ? 252 : bytes == 16384 ? 256 : 4;
				const bool apart = bytes != 1 && scale < 256;
				const uint64_t per = scale == 252 ? 16 : 1024; /* short rows of a wavefront */
				uint64_t placed = 0, copied = 0, counted = 0, short_rows = 0;
				bool few = false;
				on_launch = [&](const launch_t &l) {
					sane(l);
					if (is(l, "token_few_kernel")) {
						few = true;
						CHECK(pairs <= 2048 && n <= 1024 && l.grid.x == n + 1 && l.block.x <= 512);
						placed = counted = pairs, copied = n;
					} else if (is(l, "token_count_kernel")) {
						counted = (uint64_t)l.grid.x * 1024 * (uint32_t)parameter(l.kernel, 0);
					} else if (is(l, "token_place_kernel")) {
						placed = (uint64_t)l.grid.x * 1024 * (uint32_t)parameter(l.kernel, 0);
						CHECK(l.shared == 64u * (experts + 1) && l.arg<uint32_t>(3) == l.grid.x);
						CHECK(counted == (l.grid.x > 1 ? placed : 0));
					} else {
						const uint32_t waves = l.arg<uint32_t>(5), shorts = l.arg<uint32_t>(7), end = l.arg<uint32_t>(3);
						CHECK(is(l, "token_rows_kernel") && placed >= pairs && l.arg<uint32_t>(2) == copied && end <= n);
						CHECK(l.block.x * l.block.y <= 512 && l.arg<uint32_t>(8) == short_rows / (l.block.x / 64 * l.block.y * per));
						CHECK(l.block.x == 64 * (waves + (apart ? 0 : 1)) && (apart || shorts == 0));
						CHECK((uint64_t)(l.grid.x - shorts) * l.block.y >= end - copied);
						copied = end;
						short_rows += (uint64_t)shorts * (l.block.x / 64) * l.block.y * per;
					}
				};
				const uint64_t need = ofi_amd_token_dispatch_work_bytes(n, top_k, experts);
				CHECK(ofi_amd_token_dispatch(p, OFI_AMD_INT64, n, top_k, experts, pairs, reinterpret_cast<int32_t *>(p),
							     reinterpret_cast<int32_t *>(p), bytes == 1 ? nullptr : reinterpret_cast<int32_t *>(p), p,
							     pitch, p, pitch, bytes, p, pitch, p, pitch, scale, p, need, nullptr) == 0);
				CHECK(copied == n && placed >= pairs && (few || !apart || short_rows >= pairs));
				CHECK(few || need == (placed > 8192 ? placed / 1024 / (pairs <= 65536 ? 1 : pairs <= 131072 ? 2 : pairs <= 262144 ? 4 : 8) *
									      experts * 4
								    : 0));
			}
			int rows_copied = 0; /* the table alone */
			on_launch = [&](const launch_t &l) { rows_copied += !is(l, "token_count_kernel") && !is(l, "token_place_kernel"); };
			CHECK(ofi_amd_token_dispatch(p, OFI_AMD_INT32, n, top_k, experts, 7, reinterpret_cast<int32_t *>(p), reinterpret_cast<int32_t *>(p),
						     nullptr, nullptr, 0, nullptr, 0, 0, nullptr, 0, nullptr, 0, 0, p, ~0ull, nullptr) == 0);
			CHECK(rows_copied == 0);
			for (const auto &t : kTypes) {
				for (const uint32_t width : { 1u, 8u, 60u, 257u, 4096u, 5000u, 1u << 18 }) {
					uint64_t at = 0;
					const uint32_t chunk = width >= 16 / t.size ? 16 / t.size : 1;
					on_launch = [&](const launch_t &l) {
						sane(l);
						CHECK(is(l, "token_combine_kernel") && l.block.x <= 512 && l.block.x * l.block.y <= 512);
						const uint32_t here = l.arg<uint32_t>(8);
						CHECK((uint64_t)l.grid.x * l.block.y >= here && (uint64_t)(l.grid.x - 1) * l.block.y < here);
						CHECK(l.arg<const int32_t *>(0) == reinterpret_cast<int32_t *>(p) + at * top_k);
						const uint32_t each = chunk > 1 && top_k <= 2 ? 4 : 1; /* chunks of a lane */
						CHECK((uint64_t)l.block.x * each * chunk >= width || l.block.x > 256);
						at += here;
					};
					CHECK(ofi_amd_token_combine(p, pitch, pairs, reinterpret_cast<int32_t *>(p), nullptr, n, top_k, width, t.type, nullptr, 0, p,
								    pitch, nullptr) == 0);
					CHECK(at == n);
					at = 0;
					on_launch = [&](const launch_t &l) {
						sane(l);
						CHECK(is(l, "token_combine_grad_kernel") && l.block.x <= 512 && l.block.y == 1);
						CHECK(l.arg<const int32_t *>(0) == reinterpret_cast<int32_t *>(p) + at * top_k);
						at += l.grid.x;
					};
					CHECK(ofi_amd_token_combine_grad(p, pitch, p, pitch, pairs, reinterpret_cast<int32_t *>(p), nullptr, n, top_k, width, t.type,
									 p, pitch, reinterpret_cast<float *>(p), nullptr) == 0);
					CHECK(at == n);
				}
			}
		}
	}
	return 0;
}

int refusals()
{
	int launches = 0;
	on_launch = [&](const launch_t &) { launches++; };
	float *const f = reinterpret_cast<float *>(p);
	int32_t *const i = reinterpret_cast<int32_t *>(p);
	const int bf = OFI_AMD_BFLOAT16, f16 = OFI_AMD_FLOAT16, f32 = OFI_AMD_FLOAT32;
	auto norm = [&](void *x, uint64_t xp, void *gain, int gain_type, uint32_t n, uint32_t width, int type, float eps, void *sum, void *q,
			float *scale, uint32_t group) {
		return ofi_amd_rms_norm(x, xp, nullptr, 0, gain, gain_type, n, width, type, eps, sum, 256, nullptr, 0, q, 256, scale, 256, group,
					nullptr, nullptr);
	};
	CHECK(norm(nullptr, 256, p, bf, 4, 64, bf, 0, p, nullptr, nullptr, 0) == -EINVAL);
	CHECK(norm(p, 256, nullptr, bf, 4, 64, bf, 0, p, nullptr, nullptr, 0) == -EINVAL);
	CHECK(norm(p, 126, p, bf, 4, 64, bf, 0, p, nullptr, nullptr, 0) == -EINVAL); /* below a row */
	CHECK(norm(p, 257, p, bf, 4, 64, bf, 0, p, nullptr, nullptr, 0) == -EINVAL);
	CHECK(norm(buffer + 1, 256, p, bf, 4, 64, bf, 0, p, nullptr, nullptr, 0) == -EINVAL);
	CHECK(norm(p, 256, p, f16, 4, 64, bf, 0, p, nullptr, nullptr, 0) == -EINVAL);
	CHECK(norm(p, 256, p, OFI_AMD_INT32, 4, 64, OFI_AMD_INT32, 0, p, nullptr, nullptr, 0) == -EINVAL);
	CHECK(norm(p, 256, p, bf, 4, 0, bf, 0, p, nullptr, nullptr, 0) == -EINVAL);
	CHECK(norm(p, 1 << 20, p, bf, 4, 32769, bf, 0, p, nullptr, nullptr, 0) == -E2BIG);
	CHECK(norm(p, 256, p, bf, 1u << 31, 64, bf, 0, p, nullptr, nullptr, 0) == -E2BIG);
	CHECK(norm(p, 256, p, bf, 4, 64, bf, -1, p, nullptr, nullptr, 0) == -EINVAL);
	CHECK(norm(p, 256, p, bf, 4, 64, bf, 0.0f / 0.0f, p, nullptr, nullptr, 0) == -EINVAL);
	CHECK(norm(p, 256, p, bf, 4, 64, bf, 0, nullptr, nullptr, nullptr, 0) == -EINVAL); /* nothing asked for */
	CHECK(norm(p, 256, p, bf, 4, 64, bf, 0, p, p, nullptr, 0) == -EINVAL);
	CHECK(norm(p, 256, p, bf, 4, 64, bf, 0, p, nullptr, f, 0) == -EINVAL);
	for (const uint32_t group : { 1u, 16u, 48u, 100u, 512u }) {
		CHECK(norm(p, 256, p, bf, 4, 64, bf, 0, p, p, f, group) == -EINVAL);
	}
	/* nothing to do, or next to nothing */
	CHECK(ofi_amd_token_dispatch(nullptr, OFI_AMD_INT32, 0, 2, 8, 0, i, nullptr, nullptr, nullptr, 0, nullptr, 0, 0, nullptr, 0, nullptr, 0, 0,
				     nullptr, 0, nullptr) == 0);
	CHECK(ofi_amd_token_dispatch(nullptr, OFI_AMD_INT32, 0, 2, 8, 0, i, nullptr, nullptr, p, 64, p, 64, 64, nullptr, 0, nullptr, 0, 0, nullptr, 0,
				     nullptr) == 0);
	CHECK(launches == 2);
	launches = 0;
	CHECK(norm(nullptr, 0, nullptr, bf, 0, 64, bf, 0, p, nullptr, nullptr, 0) == 0 && launches == 0); /* no rows */
	auto grad = [&](void *dout, float *rstd, uint32_t n, uint32_t width, void *dx, float *dgain, void *work, uint64_t bytes) {
		return ofi_amd_rms_norm_grad(dout, 256, p, 256, rstd, p, f32, n, width, bf, nullptr, 0, dx, 256, dgain, work, bytes, nullptr);
	};
	CHECK(grad(nullptr, f, 4, 64, p, f, p, 1024) == -EINVAL && grad(p, nullptr, 4, 64, p, f, p, 1024) == -EINVAL);
	CHECK(grad(p, f, 4, 64, nullptr, f, p, 1024) == -EINVAL && grad(p, f, 4, 64, p, f, nullptr, 1024) == -EINVAL);
	CHECK(grad(p, f, 4, 64, p, f, p, 1023) == -EINVAL && grad(p, f, 4, 64, p, f, buffer + 2, 1024) == -EINVAL);
	CHECK(grad(p, f, 4, 0, p, f, p, 1024) == -EINVAL && grad(p, f, 1u << 31, 64, p, f, p, ~0ull) == -E2BIG);
	auto dispatch = [&](void *ids, int type, uint32_t n, uint32_t k, uint32_t e, uint32_t rows, void *offset, void *row_of, void *x, void *to,
			    uint32_t bytes, void *s, void *st, uint32_t s_bytes) {
		return ofi_amd_token_dispatch(ids, type, n, k, e, rows, static_cast<int32_t *>(offset), static_cast<int32_t *>(row_of), nullptr, x, 64, to,
					      64, bytes, s, 64, st, 64, s_bytes, nullptr, 0, nullptr);
	};
	const int i32 = OFI_AMD_INT32, i64 = OFI_AMD_INT64;
	CHECK(dispatch(p, bf, 4, 2, 8, 8, p, p, p, p, 64, nullptr, nullptr, 0) == -EINVAL);
	CHECK(dispatch(p, i32, 4, 0, 8, 8, p, p, p, p, 64, nullptr, nullptr, 0) == -EINVAL);
	CHECK(dispatch(p, i32, 4, 2, 0, 8, p, p, p, p, 64, nullptr, nullptr, 0) == -EINVAL);
	CHECK(dispatch(p, i32, 4, 2, 8, 8, nullptr, p, p, p, 64, nullptr, nullptr, 0) == -EINVAL);
	CHECK(dispatch(p, i32, 4, 2, 8, 8, p, nullptr, p, p, 64, nullptr, nullptr, 0) == -EINVAL);
	CHECK(dispatch(buffer + 4, i64, 4, 2, 8, 8, p, p, p, p, 64, nullptr, nullptr, 0) == -EINVAL);
	CHECK(dispatch(p, i32, 4, 2, 8, 8, p, p, p, nullptr, 64, nullptr, nullptr, 0) == -EINVAL);
	CHECK(dispatch(p, i32, 4, 2, 8, 8, p, p, p, p, 0, nullptr, nullptr, 0) == -EINVAL);
	CHECK(dispatch(p, i32, 4, 2, 8, 8, p, p, p, p, 65, nullptr, nullptr, 0) == -EINVAL); /* a pitch below a row */
	CHECK(dispatch(p, i32, 4, 2, 8, 8, p, p, nullptr, nullptr, 0, p, p, 4) == -EINVAL);  /* scales without rows */
	CHECK(dispatch(p, i32, 4, 2, 8, 8, p, p, p, p, 64, p, nullptr, 4) == -EINVAL);
	CHECK(dispatch(p, i32, 4, 65, 8, 8, p, p, p, p, 64, nullptr, nullptr, 0) == -E2BIG);
	CHECK(dispatch(p, i32, 4, 2, 1025, 8, p, p, p, p, 64, nullptr, nullptr, 0) == -E2BIG);
	CHECK(dispatch(p, i32, 1u << 30, 2, 8, 8, p, p, p, p, 64, nullptr, nullptr, 0) == -E2BIG);
	CHECK(dispatch(p, i32, 4, 2, 8, 1u << 31, p, p, p, p, 64, nullptr, nullptr, 0) == -E2BIG);
	CHECK(dispatch(p, i32, 5000, 2, 8, 8, p, p, p, p, 64, nullptr, nullptr, 0) == -EINVAL); /* no workspace */
	auto sum = [&](void *rows, const int32_t *row_of, const float *w, uint32_t n, uint32_t k, uint32_t width, int type, void *out) {
		return ofi_amd_token_combine(rows, 256, 16, row_of, w, n, k, width, type, nullptr, 0, out, 256, nullptr);
	};
	CHECK(sum(nullptr, i, f, 4, 2, 64, bf, p) == -EINVAL && sum(p, nullptr, f, 4, 2, 64, bf, p) == -EINVAL);
	CHECK(sum(p, i, f, 4, 2, 64, bf, nullptr) == -EINVAL && sum(p, i, f, 4, 2, 129, bf, p) == -EINVAL);
	CHECK(sum(p, i, f, 4, 0, 64, bf, p) == -EINVAL && sum(p, i, f, 4, 2, 0, bf, p) == -EINVAL && sum(p, i, f, 4, 2, 64, i32, p) == -EINVAL);
	CHECK(sum(p, i, f, 4, 65, 64, bf, p) == -E2BIG && sum(p, i, f, 4, 2, (1u << 20) + 1, bf, p) == -E2BIG);
	CHECK(sum(p, i, f, 1u << 31, 2, 64, bf, p) == -E2BIG && sum(buffer + 1, i, f, 4, 2, 64, bf, p) == -EINVAL);
	CHECK(sum(nullptr, nullptr, nullptr, 0, 2, 64, bf, nullptr) == 0);
	auto back = [&](void *dout, void *rows, void *drows, float *dw) {
		return ofi_amd_token_combine_grad(dout, 256, rows, 256, 16, i, f, 4, 2, 64, bf, drows, 256, dw, nullptr);
	};
	CHECK(back(nullptr, p, p, f) == -EINVAL && back(p, nullptr, p, f) == -EINVAL && back(p, p, nullptr, nullptr) == -EINVAL);
	CHECK(back(p, p, buffer + 1, f) == -EINVAL && launches == 0);
	CHECK(back(p, nullptr, p, nullptr) == 0 && back(p, p, nullptr, f) == 0 && launches == 2);
	return 0;
}

} // namespace

int main(int argc, char **argv)
{
	const std::map<std::string, int (*)()> parts = { { "norms", norms }, { "tokens", tokens }, { "refusals", refusals } };
	CHECK(argc == 2 && parts.count(argv[1]) && ofi_amd_gpu_init() == 0);
	const int rc = parts.at(argv[1])();
	std::printf("%s: %s\n", argv[1], rc == 0 ? "ok" : "failed");
	return rc;
}
