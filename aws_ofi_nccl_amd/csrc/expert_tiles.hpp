/*
 * What the experts' products share: which rows of which expert a workgroup takes, how tiles of both operands come into LDS and
 * from there to the matrix cores, and how sums leave in rows.
 *
 * A workgroup of WM x WN wavefronts computes 64 WM rows (of the result) by two parts of 128 columns: a part is the gate's or the
 * other projection's share of a gated block, or half of 256 neighbouring columns.  A wavefront has 64 rows and 128 / WN columns of both
 * parts, so that a gate's sums and those they are multiplied with lie in the same lane, and each part is one block of 128 columns that
 * shares an 8-bit scale.
 *
 * The summed axis is taken in steps: 128 bytes of a row where the operand's rows run along it ("along"), 64 rows where they run
 * across it ("across").  Two or three tiles of LDS take turns: while one is computed on, the others are filled (sum_steps, sum_halves).
 *   along    16-byte chunk c of row r lies at slot c ^ (r & 7) of the row: eight rows' same chunk, which eight lanes read at once,
 *            are in eight different groups of banks
 *   across   row k's chunk c lies at slot c ^ 2 (k & 3 | (k >> 3 & 1) << 2): four rows' same 32 bytes, which sixteen lanes read and
 *            exchange (ds_read_b64_tr_b16: lane l of sixteen gets column l of four rows), are in different groups too
 * The matrix instruction's first operand is the column tile, so that a lane's four sums are neighbouring columns of one row (columns
 * 4 (lane / 16) + i of a group of 16, row lane % 16).
 */
#ifndef OFI_AMD_EXPERT_TILES_HPP_
#define OFI_AMD_EXPERT_TILES_HPP_

#include "common.hpp"
#include "row_types.hpp"

namespace ofi_amd {

struct e4m3_t {
	uint8_t bits;
};

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x8_t __attribute__((ext_vector_type(8)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void lds_void_t;
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;

constexpr uint32_t kBlock = 128;       /* columns that share a scale, and columns of a part */
constexpr uint32_t kStepBytes = 128;   /* of a row along the summed axis, in a step */
constexpr uint32_t kStepRows = 64;     /* rows across it */
constexpr uint32_t kComputeUnits = 256;
constexpr uint32_t kMostExperts = 1024, kMostExpertWidth = 1u << 20;

template <typename T> constexpr uint32_t kStepOf = kStepBytes / sizeof(T); /* elements of the summed axis in a step */

__host__ __device__ inline uint32_t blocks_of(uint32_t width) { return (width + kBlock - 1) / kBlock; }

/* ---- rows of experts ---------------------------------------------------------------------------------------- */

/* from: the tile's first row, rows: those it has; nt: which of the column tiles */
struct tile_t {
	uint32_t expert, from, rows, nt;
	bool any;
};

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }

/* Rows [lo, hi) of expert e, whatever the offsets are: within the rows there are */
__device__ __forceinline__ void run_of(const int32_t *offset, uint32_t e, uint32_t max_rows, uint32_t &lo, uint32_t &hi)
{
	const int32_t a = offset ? offset[e] : 0, b = offset ? offset[e + 1] : (int32_t)max_rows;
	lo = a < 0 ? 0u : (uint32_t)a < max_rows ? (uint32_t)a : max_rows;
	hi = b < 0 ? 0u : (uint32_t)b < max_rows ? (uint32_t)b : max_rows;
	hi = hi < lo ? lo : hi;
}

/* Sum over the lanes up to this one */
__device__ __forceinline__ uint32_t running_sum(uint32_t v, uint32_t lane)
{
#pragma unroll
	for (uint32_t d = 1; d < 64; d *= 2) {
		const uint32_t up = (uint32_t)__shfl_up((int)v, d, 64);
		v += lane >= d ? up : 0u;
	}
	return v;
}

/*
 * The tiles of a launch.  They are numbered expert by expert, an expert's in bands of eight row tiles, a band's column by column: what an
 * XCD's 32 compute units work on at once is about eight row tiles by four column tiles, which its L2 holds a step of.  Workgroups go to
 * the eight XCDs in turn, so each XCD gets an eighth of the numbers in one piece.  Each lane has one of 64 experts.
 */
struct rows_t {
	const int32_t *offset;
	uint32_t n_experts, max_rows, n_tiles;
};

/* Of one of 64 experts, in a lane: its rows, its row tiles, and those of the experts before it */
struct seen_t {
	uint32_t lo, hi, mine, before;
};

/* Experts e to e + 63, behind `before` row tiles, which is then all up to them */
template <uint32_t BM> __device__ __forceinline__ seen_t look_at_experts(rows_t rows, uint32_t e, uint32_t &before)
{
	const uint32_t lane = threadIdx.x & 63u;
	seen_t s = {};
	if (e + lane < rows.n_experts) {
		run_of(rows.offset, e + lane, rows.max_rows, s.lo, s.hi);
	}
	s.mine = (s.hi - s.lo + BM - 1) / BM;
	const uint32_t sum = running_sum(s.mine, lane);
	s.before = before + sum - s.mine;
	before += (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
	return s;
}

/* The tile of workgroup `id` */
template <uint32_t BM> __device__ __forceinline__ tile_t find_tile(rows_t rows, uint32_t id)
{
	tile_t t = {};
	uint32_t total = 0, first = 0;
	seen_t seen = look_at_experts<BM>(rows, 0, total);
	for (uint32_t e = 64; e < rows.n_experts; e += 64) {
		(void)look_at_experts<BM>(rows, e, total);
	}
	const uint32_t n_tiles = rows.n_tiles, tiles = total * n_tiles, share = (tiles + 7) / 8;
	uint32_t at = uniform((id & 7u) * share + (id >> 3));
	if ((id >> 3) >= share || at >= tiles) {
		return t;
	}
	if (rows.n_experts > 64) { /* again, up to the expert that has the tile */
		uint32_t before = 0;
		for (uint32_t e = 0; e < rows.n_experts && at >= before * n_tiles; e += 64) {
			first = e;
			seen = look_at_experts<BM>(rows, e, before);
		}
	}
	const uint64_t has = __ballot(seen.mine != 0 && at >= seen.before * n_tiles && at < (seen.before + seen.mine) * n_tiles);
	if (!has) {
		return t;
	}
	const int who = (int)__builtin_ctzll(has);
	const uint32_t begin = (uint32_t)__builtin_amdgcn_readlane((int)seen.lo, who), end = (uint32_t)__builtin_amdgcn_readlane((int)seen.hi, who);
	const uint32_t row_tiles = (uint32_t)__builtin_amdgcn_readlane((int)seen.mine, who);
	at -= (uint32_t)__builtin_amdgcn_readlane((int)seen.before, who) * n_tiles;
	const uint32_t band = at / (8 * n_tiles), in_band = at - band * 8 * n_tiles;
	const uint32_t height = row_tiles - band * 8 < 8 ? row_tiles - band * 8 : 8;
	t.expert = first + (uint32_t)who;
	t.nt = in_band / height;
	t.from = begin + (band * 8 + in_band - t.nt * height) * BM;
	t.rows = end - t.from < BM ? end - t.from : BM;
	t.any = true;
	return t;
}

/*
 * The kernel's argument, a single A.  Each call is another pointer to the compiler: what one part of a kernel needs of it is loaded there, and
 * does not lie in scalar registers from the beginning on (200 of them were spilled into the registers of the sums).
 */
template <typename A> __device__ __forceinline__ const A *argument()
{
	auto p = __builtin_amdgcn_kernarg_segment_ptr();
	asm volatile("" : "+s"(p));
	return (const A *)p;
}

/* ---- operands ----------------------------------------------------------------------------------------------- */

/* Up to 16 bytes of a row's `left` bytes from p on, zeros behind them; any alignment */
template <typename T> __device__ __forceinline__ u32x4_t chunk_at(const uint8_t *p, int64_t left)
{
	if (left >= 16) {
		return *reinterpret_cast<const any16_t *>(p);
	}
	u32x4_t v = { 0, 0, 0, 0 };
	if (left > 0) {
#pragma unroll
		for (uint32_t i = 0; i < 16 / sizeof(T); i++) {
			if ((int64_t)(i * sizeof(T)) < left) {
				if constexpr (sizeof(T) == 2) {
					v[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t *>(p)[i] << (16 * (i & 1));
				} else {
					v[i / 4] |= (uint32_t)p[i] << (8 * (i & 3));
				}
			}
		}
	}
	return v;
}

/*
 * 16 bytes for each lane of the wavefront from a buffer of `bytes` at p, to LDS at `lds` (of the wavefront) and 16 more for each lane;
 * zeros from beyond the buffer.  Written as the instruction, because the compiler waits for the builtin's bytes before the next
 * exchanging read of LDS, whichever part of it that reads: the wait is landed()'s.  What the compiler sees to in front of its own loads is done
 * here too: a scalar register that a vector instruction wrote (uniform(), or a spilled one's return) is not there for a load before five wait
 * states, which s_nop 4 is, and M0, from which the place is taken, not before one.
 */
typedef int i32x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void to_lds(const uint8_t *p, int bytes, uint32_t offset, uint8_t *lds)
{
	const uint64_t at = reinterpret_cast<uint64_t>(p);
	const i32x4_t buffer = { (int)uniform((uint32_t)at), (int)uniform((uint32_t)(at >> 32) & 0xffffu), (int)uniform((uint32_t)bytes), 0x00020000 };
	const uint32_t to = uniform((uint32_t)reinterpret_cast<uintptr_t>((lds_void_t *)lds));
	asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"{m0}"(to), "v"(offset), "s"(buffer) : "memory");
}
/* The same of 4 bytes for each lane */
__device__ __forceinline__ void words_to_lds(const uint8_t *p, int bytes, uint32_t offset, uint8_t *lds)
{
	const uint64_t at = reinterpret_cast<uint64_t>(p);
	const i32x4_t buffer = { (int)uniform((uint32_t)at), (int)uniform((uint32_t)(at >> 32) & 0xffffu), (int)uniform((uint32_t)bytes), 0x00020000 };
	const uint32_t to = uniform((uint32_t)reinterpret_cast<uintptr_t>((lds_void_t *)lds));
	asm volatile("s_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"{m0}"(to), "v"(offset), "s"(buffer) : "memory");
}
/* All but the last N of the wavefront's to_lds have landed */
template <uint32_t N> __device__ __forceinline__ void landed()
{
	static_assert(N < 64, "the counter has six bits");
	asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
/* A barrier at which every wavefront's reads of LDS are done.  What to_lds has on its way stays on its way (__syncthreads would wait for
 * it); what comes through registers is stored by then. */
template <bool DIRECT> __device__ __forceinline__ void workgroup_meets()
{
	if (DIRECT) {
		asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
		__builtin_amdgcn_s_barrier();
		asm volatile("" ::: "memory");
	} else {
		__syncthreads();
	}
	__builtin_amdgcn_sched_barrier(0);
}
constexpr uint32_t kBeyond = 0x80000000u; /* of any buffer */

/* The chunk whose last `over` bytes lie behind the row, read as the 16 bytes that end with it: its own bytes, and zeros */
__device__ __forceinline__ u32x4_t shifted(u32x4_t v, uint32_t over)
{
	const uint64_t lo = v.x | (uint64_t)v.y << 32, hi = v.z | (uint64_t)v.w << 32;
	const uint32_t bits = 8 * over;
	const uint64_t low = bits >= 64 ? hi >> (bits - 64) : bits ? lo >> bits | hi << (64 - bits) : lo, high = bits >= 64 ? 0 : hi >> bits;
	return u32x4_t{ (uint32_t)low, (uint32_t)(low >> 32), (uint32_t)high, (uint32_t)(high >> 32) };
}

/*
 * ROWS rows of an operand whose rows run along the summed axis.  base: the first row's start; rows of them are there, each of `bytes`;
 * what is not there of the summed axis is zeros.
 */
template <typename T, uint32_t ROWS, uint32_t THREADS> struct along_t {
	static constexpr uint32_t kChunks = ROWS * 8 / THREADS, kRowsOfRound = THREADS / 8, kBytes = ROWS * kStepBytes;
	const uint8_t *base;
	uint64_t pitch;
	uint32_t rows;
	int64_t bytes;
	u32x4_t held[kChunks];

	__device__ __forceinline__ void set(const uint8_t *p, uint64_t apart, uint32_t n, int64_t size)
	{
		base = p;
		pitch = apart;
		rows = n;
		bytes = size;
	}
	/* Rows that are not there are read as the last that is (no result of theirs is written), chunks behind the row as its last 16 bytes: no load
	 * is conditional where a row has 16 bytes */
	__device__ __forceinline__ void load(uint32_t step)
	{
		const uint32_t row = threadIdx.x / 8, chunk = (threadIdx.x & 7u) ^ (row & 7u);
		const int64_t at = (int64_t)step * kStepBytes + chunk * 16;
#pragma unroll
		for (uint32_t t = 0; t < kChunks; t++) {
			const uint32_t r = t * kRowsOfRound + row;
			const uint8_t *const p = base + (uint64_t)(r < rows ? r : rows - 1) * pitch;
			held[t] = bytes >= 16 ? *reinterpret_cast<const any16_t *>(p + (at + 16 <= bytes ? at : bytes - 16)) : chunk_at<T>(p + at, bytes - at);
		}
	}
	__device__ __forceinline__ void store(uint32_t step, uint8_t *lds) const
	{
		const uint32_t row = threadIdx.x / 8, chunk = (threadIdx.x & 7u) ^ (row & 7u);
		const int64_t at = (int64_t)step * kStepBytes + chunk * 16;
		const bool rest = (int64_t)(step + 1) * kStepBytes > bytes && bytes >= 16;
#pragma unroll
		for (uint32_t t = 0; t < kChunks; t++) {
			u32x4_t v = held[t];
			if (rest) { /* of all rows alike */
				const u32x4_t s = shifted(v, (uint32_t)(16 - bytes % 16) % 16);
				v = at + 16 <= bytes ? v : at < bytes ? s : u32x4_t{ 0, 0, 0, 0 };
			}
			*reinterpret_cast<u32x4_t *>(lds + (t * THREADS + threadIdx.x) * 16) = v;
		}
	}
	/* Both at once, past the registers: rows in whole chunks (in_chunks), so that a tile is within 31 bits */
	__device__ __forceinline__ void fill(uint32_t step, uint8_t *lds) const
	{
		const uint32_t row = threadIdx.x / 8, chunk = (threadIdx.x & 7u) ^ (row & 7u), wave = uniform(threadIdx.x >> 6);
		const uint32_t at = step * kStepBytes, apart = (uint32_t)pitch * kRowsOfRound;
		const uint32_t place = (row * (uint32_t)pitch + chunk * 16) | (at + chunk * 16 < (uint32_t)bytes ? 0 : kBeyond);
		const int left = (int)((rows - 1) * (uint32_t)pitch + (uint32_t)bytes) - (int)at - (rows ? 0 : 0x40000000); /* no rows: nothing */
#pragma unroll
		for (uint32_t t = 0; t < kChunks; t++) {
			const int n = left - (int)(t * apart);
			to_lds(base + at + (uint64_t)(t * apart), n > 0 ? n : 0, place, lds + (t * THREADS + wave * 64) * 16);
		}
	}
};

/* The rows of `along` that a lane feeds to a matrix instruction: 16 bytes of each half of a step */
struct along_frag_t {
	static constexpr int kReads = 1;
	uint32_t at[2];
	__device__ __forceinline__ along_frag_t(uint32_t first_row, uint32_t lane)
	{
		at[0] = (first_row + (lane & 15u)) * kStepBytes + (((lane >> 4) ^ (lane & 7u)) << 4);
		at[1] = at[0] ^ 64u;
	}
	/* row: the first of 16, behind first_row */
	__device__ __forceinline__ u32x4_t get(const uint8_t *lds, uint32_t row, uint32_t half) const
	{
		return *reinterpret_cast<const u32x4_t *>(lds + at[half] + row * kStepBytes);
	}
};

template <uint32_t W> __device__ __forceinline__ uint32_t across_slot(uint32_t k)
{
	return (((k & 3u) | ((k >> 3) & 1u) << 2) << 1) & (W / 8 - 1);
}

/* W columns of an operand whose rows run across the summed axis; two-byte elements.  base: column 0 of the first row */
template <typename T, uint32_t W, uint32_t THREADS, uint32_t ROWS = kStepRows> struct across_t {
	static constexpr uint32_t kOfRow = W / 8, kChunks = ROWS * kOfRow / THREADS, kBytes = ROWS * W * 2;
	const uint8_t *base;
	uint64_t pitch;
	uint32_t rows;  /* of the summed axis */
	int64_t bytes;  /* of the columns there are, at most W's */
	u32x4_t held[kChunks];

	__device__ __forceinline__ void set(const uint8_t *p, uint64_t apart, uint32_t n, int64_t size)
	{
		base = p;
		pitch = apart;
		rows = n;
		bytes = size;
	}
	__device__ __forceinline__ void load(uint32_t step)
	{
#pragma unroll
		for (uint32_t t = 0; t < kChunks; t++) {
			const uint32_t slot = t * THREADS + threadIdx.x, k = slot / kOfRow, r = step * ROWS + k;
			const int64_t at = (slot % kOfRow ^ across_slot<W>(k)) * 16;
			const uint8_t *const p = base + (uint64_t)(r < rows ? r : rows - 1) * pitch;
			held[t] = bytes >= 16 ? *reinterpret_cast<const any16_t *>(p + (at + 16 <= bytes ? at : bytes - 16)) : chunk_at<T>(p + at, bytes - at);
		}
	}
	__device__ __forceinline__ void store(uint32_t step, uint8_t *lds) const
	{
		const uint32_t over = (uint32_t)(16 - bytes % 16) % 16;
		const bool some = over && bytes >= 16, rest = (step + 1) * ROWS > rows;
#pragma unroll
		for (uint32_t t = 0; t < kChunks; t++) {
			const uint32_t slot = t * THREADS + threadIdx.x, k = slot / kOfRow, r = step * ROWS + k;
			u32x4_t v = held[t];
			if (some) {
				const int64_t at = (slot % kOfRow ^ across_slot<W>(k)) * 16;
				const u32x4_t s = shifted(v, over);
				v = at < bytes && at + 16 > bytes ? s : v;
			}
			if (rest) {
				v = r < rows ? v : u32x4_t{ 0, 0, 0, 0 };
			}
			*reinterpret_cast<u32x4_t *>(lds + (t * THREADS + threadIdx.x) * 16) = v;
		}
	}
	__device__ __forceinline__ void fill(uint32_t step, uint8_t *lds) const
	{
		constexpr uint32_t kRowsOfRound = THREADS / kOfRow;
		const uint64_t at = (uint64_t)step * ROWS * pitch;
		const int64_t left = (int64_t)((rows - 1) * pitch + bytes - at) - (rows ? 0 : 1ll << 60); /* no rows: nothing */
		const uint32_t apart = (uint32_t)pitch * kRowsOfRound, row = threadIdx.x / kOfRow, wave = uniform(threadIdx.x >> 6);
		const int some = left <= 0 ? 0 : left < 0x7fffffff ? (int)left : 0x7fffffff;
#pragma unroll
		for (uint32_t t = 0; t < kChunks; t++) {
			const uint32_t chunk = (threadIdx.x % kOfRow) ^ across_slot<W>(t * kRowsOfRound + row);
			const uint32_t place = (row * (uint32_t)pitch + chunk * 16) | (chunk * 16 < (uint32_t)bytes ? 0 : kBeyond);
			const int n = some - (int)(t * apart);
			to_lds(base + at + (uint64_t)(t * apart), n > 0 ? n : 0, place, lds + (t * THREADS + wave * 64) * 16);
		}
	}
};

/* The columns of `across` that a lane feeds to a matrix instruction: eight of the summed axis, four at a time */
template <uint32_t W> struct across_frag_t {
	static constexpr int kReads = 2;
	uint32_t at[4]; /* of four groups of 16 columns in a row; those of the other part are 256 bytes on */
	__device__ __forceinline__ across_frag_t(uint32_t first_column, uint32_t lane)
	{
		const uint32_t k = (lane >> 4) * 8 + ((lane & 15u) >> 2);
#pragma unroll
		for (uint32_t g = 0; g < 4; g++) {
			at[g] = k * W * 2 + (lane & 1u) * 8 + ((((first_column / 8 + 2 * g) ^ across_slot<W>(k)) + ((lane & 3u) >> 1)) << 4);
		}
	}
	/* column: the first of 16, behind first_column: of the first four groups, or of those 128 columns on */
	__device__ __forceinline__ u32x4_t get(uint8_t *lds, uint32_t column, uint32_t half) const
	{
		uint8_t *const p = lds + at[column / 16 & 3u] + (column & 128u ? 256u : 0u) + half * 32 * W * 2;
		const s16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)p);
		const s16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)(p + 4 * W * 2));
		const u32x2_t lo = __builtin_bit_cast(u32x2_t, a), hi = __builtin_bit_cast(u32x2_t, b);
		return u32x4_t{ lo.x, lo.y, hi.x, hi.y };
	}
};

/* sums[i] += column tile x row tile, 32 of the summed axis */
template <typename T> __device__ __forceinline__ f32x4_t multiply(u32x4_t columns, u32x4_t rows, f32x4_t sums)
{
	if constexpr (std::is_same<T, bf16_t>::value) {
		return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, columns), __builtin_bit_cast(bf16x8_t, rows), sums, 0,
							       0, 0);
	} else {
		return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, columns), __builtin_bit_cast(f16x8_t, rows), sums, 0,
							      0, 0);
	}
}

/* Eight values of e4m3 as float16, which holds each of them */
__device__ __forceinline__ u32x4_t widened(uint32_t a, uint32_t b)
{
	const auto w0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false), w1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true);
	const auto w2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false), w3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true);
	return u32x4_t{ __builtin_bit_cast(uint32_t, w0), __builtin_bit_cast(uint32_t, w1), __builtin_bit_cast(uint32_t, w2),
			__builtin_bit_cast(uint32_t, w3) };
}

/* READS of LDS among PAIRS pairs of matrix instructions, so that they are done when their half begins */
template <int READS, int PAIRS> __device__ __forceinline__ void spread_reads()
{
	constexpr int kEach = (READS + PAIRS - 1) / PAIRS;
#pragma unroll
	for (int i = 0; i < PAIRS; i++) {
		__builtin_amdgcn_sched_group_barrier(0x100, kEach, 0);
		__builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
	}
	__builtin_amdgcn_sched_barrier(0);
}

/*
 * sums[m][p][j] += all steps.  Fragments of half a step are read while the other half's are multiplied.  When all of a step's are in
 * registers, a barrier: the next step's tile is there (it was asked for STAGES - 1 steps before), and this one's place is free for the
 * step STAGES on.  fill: both operands' tiles of a step to LDS, kFills instructions of a wavefront; or (not DIRECT, two stages) load: to
 * registers, and store: from there.  Fills behind the last step write zeros.  busy: whether the wavefront has rows; the matrix
 * cores are another's where it has none, so that an expert's last tile costs the quarters of it that there are.
 */
template <typename T, bool DIRECT, uint32_t STAGES, uint32_t FILLS, uint32_t MF, uint32_t G, typename RowFrag, typename ColumnFrag, typename Fill,
	  typename Load, typename Store, typename Also>
__device__ __forceinline__ void sum_steps(f32x4_t (&sums)[MF][2][G], bool busy, uint32_t steps, uint8_t *lds, uint32_t tile_bytes,
					  uint32_t rows_bytes, const RowFrag &row_frag, const ColumnFrag &column_frag, Fill fill, Load load, Store store,
					  Also also)
{
	static_assert(DIRECT || STAGES == 2, "what comes through registers has two stages");
	static_assert(MF <= 4 && G <= 4, "groups of columns that a fragment has places for");
	u32x4_t r[2][MF], c[2][2 * G];
	auto read = [&](uint8_t *tile, uint32_t half, u32x4_t(&rows)[MF], u32x4_t(&columns)[2 * G]) __attribute__((always_inline)) {
#pragma unroll
		for (uint32_t m = 0; m < MF; m++) {
			rows[m] = row_frag.get(tile, m * 16, half);
		}
#pragma unroll
		for (uint32_t j = 0; j < 2 * G; j++) {
			columns[j] = column_frag.get(tile + rows_bytes, j / G * kBlock + j % G * 16, half);
		}
	};
	auto mul = [&](const u32x4_t(&rows)[MF], const u32x4_t(&columns)[2 * G]) __attribute__((always_inline)) {
#pragma unroll
		for (uint32_t j = 0; j < 2 * G; j++) {
#pragma unroll
			for (uint32_t m = 0; m < MF; m++) {
				sums[m][j / G][j % G] = multiply<T>(columns[j], rows[m], sums[m][j / G][j % G]);
			}
		}
		also(rows);
	};
	auto spread = [&]() __attribute__((always_inline)) { spread_reads<MF * RowFrag::kReads + 2 * G * ColumnFrag::kReads, MF * G>(); };
	if (steps == 0) {
		return;
	}
	if (DIRECT) {
#pragma unroll
		for (uint32_t s = 0; s < STAGES; s++) {
			fill(s, lds + s * tile_bytes);
		}
		landed<(STAGES - 1) * FILLS>();
		workgroup_meets<true>();
	} else {
		load(0);
		store(0, lds);
		__syncthreads();
		load(1);
	}
	auto loop = [&](auto has_rows) __attribute__((always_inline)) {
		constexpr bool kBusy = decltype(has_rows)::value;
		uint32_t at = 0;
		if (kBusy) {
			read(lds, 0, r[0], c[0]);
		}
		for (uint32_t step = 0; step < steps; step++) {
			uint8_t *const now = lds + at;
			at = at + tile_bytes < STAGES * tile_bytes ? at + tile_bytes : 0;
			uint8_t *const next = lds + at;
			if (kBusy) {
				read(now, 1, r[1], c[1]);
				mul(r[0], c[0]);
				spread();
			}
			if (DIRECT) {
				landed<(STAGES - 2) * FILLS>();
			} else {
				store(step + 1, next);
			}
			workgroup_meets<DIRECT>();
			if (DIRECT) {
				fill(step + STAGES, now);
			} else {
				load(step + 2);
			}
			__builtin_amdgcn_sched_barrier(0);
			if (kBusy) {
				read(next, 0, r[0], c[0]);
				mul(r[1], c[1]);
				spread();
			}
		}
	};
	if (busy) { /* of the whole wavefront; both loops meet the same barriers */
		loop(std::true_type{});
	} else {
		loop(std::false_type{});
	}
	if (DIRECT) {
		landed<0>(); /* what follows writes there */
	}
}

/*
 * The same for workgroups of four wavefronts, of which a compute unit has two: while one is at its beginning, its epilogue or a barrier, the other
 * multiplies.  Each has 80 KB of LDS: the rows' tiles of two steps, and the columns' of three halves of a step, asked for that long before they
 * are read.  For columns across the summed axis, whose half a step is half of the rows.
 * Tiles of 256 x 256, one to a compute unit, and these (32,768 rows of 32 experts; us): hidden_grad of 4096 to 2048 731 and 645, rows_grad of
 * 4096 to 4096 1032 and 1010, weight_grad of 4096 x 4096 into float32 1545 and 1415.  Columns along the axis stay with sum_steps: half a step of
 * them is half of a line (gated 4096 to 2048 1090 and 1145, product of 8192 rows 4096 x 4096 270 and 295), and units of 128 columns and a whole
 * step instead, for which the rows are read from LDS twice, gain nothing (1086 and 1094, 277 and 295).
 */
template <typename T, uint32_t ROW_FILLS, uint32_t COLUMN_FILLS, uint32_t ROWS_BYTES, uint32_t HALF_BYTES, uint32_t MF, uint32_t G, typename RowFrag,
	  typename ColumnFrag, typename FillRows, typename FillColumns, typename Also>
__device__ __forceinline__ void sum_halves(f32x4_t (&sums)[MF][2][G], bool busy, uint32_t steps, uint8_t *lds, const RowFrag &row_frag,
					   const ColumnFrag &column_frag, FillRows fill_rows, FillColumns fill_columns, Also also)
{
	static_assert(MF <= 4 && G <= 4, "groups of columns that a fragment has places for");
	u32x4_t r[2][MF], c[2][2 * G];
	auto read = [&](uint8_t *rows, uint8_t *columns, uint32_t half) __attribute__((always_inline)) {
#pragma unroll
		for (uint32_t m = 0; m < MF; m++) {
			r[half][m] = row_frag.get(rows, m * 16, half);
		}
#pragma unroll
		for (uint32_t j = 0; j < 2 * G; j++) {
			c[half][j] = column_frag.get(columns, j / G * kBlock + j % G * 16, 0);
		}
	};
	auto mul = [&](uint32_t half) __attribute__((always_inline)) {
#pragma unroll
		for (uint32_t j = 0; j < 2 * G; j++) {
#pragma unroll
			for (uint32_t m = 0; m < MF; m++) {
				sums[m][j / G][j % G] = multiply<T>(c[half][j], r[half][m], sums[m][j / G][j % G]);
			}
		}
		also(r[half]);
		spread_reads<MF * RowFrag::kReads + 2 * G * ColumnFrag::kReads, MF * G>();
	};
	if (steps == 0) {
		return;
	}
	uint8_t *rows = lds, *next_rows = lds + ROWS_BYTES;
	uint8_t *now = lds + 2 * ROWS_BYTES, *next = now + HALF_BYTES, *third = next + HALF_BYTES;
	fill_rows(0, rows);
	fill_columns(0, now);
	fill_columns(1, next);
	fill_rows(1, next_rows);
	fill_columns(2, third);
	landed<ROW_FILLS + 2 * COLUMN_FILLS>();
	workgroup_meets<true>();
	auto loop = [&](auto has_rows) __attribute__((always_inline)) {
		constexpr bool kBusy = decltype(has_rows)::value;
		auto turn = [&]() __attribute__((always_inline)) {
			uint8_t *const done = now;
			now = next;
			next = third;
			third = done;
		};
		if (kBusy) {
			read(rows, now, 0);
		}
		for (uint32_t step = 0; step < steps; step++) {
			landed<ROW_FILLS + COLUMN_FILLS>(); /* the columns' second half */
			workgroup_meets<true>();
			turn();
			fill_columns(2 * step + 3, third);
			__builtin_amdgcn_sched_barrier(0);
			if (kBusy) {
				read(rows, now, 1);
				mul(0);
			}
			landed<COLUMN_FILLS>(); /* the next step's rows and first half */
			workgroup_meets<true>();
			turn();
			fill_rows(step + 2, rows);
			fill_columns(2 * step + 4, third);
			uint8_t *const done = rows;
			rows = next_rows;
			next_rows = done;
			__builtin_amdgcn_sched_barrier(0);
			if (kBusy) {
				read(rows, now, 0);
				mul(1);
			}
		}
	};
	if (busy) {
		loop(std::true_type{});
	} else {
		loop(std::false_type{});
	}
	landed<0>();
}

/* ---- sums ----------------------------------------------------------------------------------------------------- */

/* The value, but not to be computed with outside of the loop: what would be there for every matrix that a loop might write takes the
 * registers of a tile's sums */
__device__ __forceinline__ uint32_t in_loop(uint32_t v)
{
	asm volatile("" : "+v"(v));
	return v;
}

/*
 * A tile's sums by rows: finish(row of the tile, lane % 16, columns of part 0, of part 1, what load(row) gave), eight columns of both parts in a lane, a
 * row in a quarter of a wavefront, so that what is read and written of it is one piece, and a block of 128 columns is sixteen
 * neighbouring lanes.  They are columns 8 (lane % 16) on of the part, or with SPLIT 4 (lane % 16) and 64 + 4 (lane % 16) on, with which four
 * bytes a column are whole lines.  The sums go through LDS, 64 rows of a tile of 256 at a time, so that one loop does for all of
 * them (unrolled over the registers the same epilogue was 200 KB of instructions); what is loaded is asked for one such turn ahead.
 * No barrier waits for what has been written.
 * whole: all of the tile's rows and columns are there; load and finish get it as a constant and have no conditions then (with them, every
 * eight values went through six branches: a tile of 256 x 256 with 1024 summed 40.4 us, without 37.4; 23 are the sums).
 * One row after the other: two at once took the registers of the sums.
 */
template <uint32_t WM, uint32_t WN, uint32_t MF, bool SPLIT, typename Load, typename Finish>
__device__ __forceinline__ void for_rows(const f32x4_t (&sums)[MF][2][8 / WN], uint8_t *lds, bool whole, Load load, Finish finish)
{
	static_assert(MF == 4, "four groups of rows");
	constexpr uint32_t G = 8 / WN, kGroups = WM == 4 ? 1 : 2; /* groups of 16 rows of a wavefront in a turn */
	constexpr uint32_t kRows = kGroups * 16, kLoops = 4 / kGroups, kTurns = kRows / WN / 4;
	const uint32_t lane = threadIdx.x & 63u, wave = uniform(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
	auto place = [&](uint32_t turn) { return (wave * kTurns + turn) * 4 + (lane >> 4); };
	auto row_of = [&](uint32_t loop, uint32_t at) { return at / kRows * 64 + loop * kRows + at % kRows; };
	using in_t = decltype(load(std::true_type{}, 0u, 0u));
	auto ask = [&](uint32_t loop, uint32_t turn) __attribute__((always_inline)) {
		const uint32_t r = row_of(loop, place(turn)), part_lane = in_loop(lane & 15u);
		return whole ? load(std::true_type{}, r, part_lane) : load(std::false_type{}, r, part_lane);
	};
	in_t in = ask(0, 0);
	auto put = [&](uint32_t m, const f32x4_t(&from)[2][G]) __attribute__((always_inline)) {
		const uint32_t r = wm * kRows + m * 16 + (lane & 15u);
#pragma unroll
		for (uint32_t p = 0; p < 2; p++) {
#pragma unroll
			for (uint32_t j = 0; j < G; j++) {
				const uint32_t chunk = p * 32 + (wn * G + j) * 4 + (lane >> 4);
				*reinterpret_cast<f32x4_t *>(lds + r * 1024 + ((chunk ^ (r & 15u)) << 4)) = from[p][j];
			}
		}
	};
#pragma unroll 1
	for (uint32_t loop = 0; loop < kLoops; loop++) {
		workgroup_meets<true>(); /* the tiles, or the rows before, have been read */
		if (kGroups == 1) {
			switch (loop) {
			case 0: put(0, sums[0]); break;
			case 1: put(0, sums[1]); break;
			case 2: put(0, sums[2]); break;
			default: put(0, sums[3]);
			}
		} else if (loop == 0) {
			put(0, sums[0]);
			put(1, sums[1]);
		} else {
			put(0, sums[2]);
			put(1, sums[3]);
		}
		workgroup_meets<true>();
#pragma unroll
		for (uint32_t i = 0; i < kTurns; i++) {
			const uint32_t at = place(i);
			const uint8_t *const from = lds + at * 1024;
			const uint32_t swizzle = at & 15u, chunk = SPLIT ? lane & 15u : (lane & 15u) * 2, other = SPLIT ? chunk + 16 : chunk + 1;
			auto get = [&](uint32_t c) { return *reinterpret_cast<const f32x4_t *>(from + ((c ^ swizzle) << 4)); };
			const f32x4_t a0 = get(chunk), a1 = get(other), b0 = get(chunk + 32), b1 = get(other + 32);
			const f32x8_t a = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7), b = __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7);
			const in_t now = in;
			if (i + 1 < kTurns) {
				in = ask(loop, i + 1);
			} else if (loop + 1 < kLoops) {
				in = ask(loop + 1, 0);
			}
			if (whole) {
				finish(std::true_type{}, row_of(loop, at), in_loop(lane & 15u), a, b, now);
			} else {
				finish(std::false_type{}, row_of(loop, at), in_loop(lane & 15u), a, b, now);
			}
			__builtin_amdgcn_sched_barrier(0);
		}
	}
}

/* A matrix of 16-bit, float32 or e4m3 values; none: p NULL */
struct matrix_t {
	uint8_t *p;
	uint64_t pitch;
	int type;
	float *scale; /* of e4m3: one to each block of columns */
	uint64_t scale_pitch;
};

/* `left` of V values at p, as words; zeros for the others */
template <typename U, uint32_t V, typename W> __device__ __forceinline__ void read_words(const uint8_t *p, uint32_t left, W &w)
{
	typedef U any_t __attribute__((ext_vector_type(V), aligned(sizeof(U))));
	static_assert(sizeof(any_t) <= sizeof(W), "room");
	if (left >= V) {
		const any_t all = *reinterpret_cast<const any_t *>(p);
		__builtin_memcpy(&w, &all, sizeof(all));
	} else {
		any_t some = {};
#pragma unroll
		for (uint32_t i = 0; i < V - 1; i++) {
			if (i < left) {
				some[i] = reinterpret_cast<const U *>(p)[i];
			}
		}
		__builtin_memcpy(&w, &some, sizeof(some));
	}
}

/* Eight values of a 16-bit or 8-bit type as they lie in memory, and the scale of those of 8 bits */
struct eight_t {
	u32x4_t words;
	float scale;
};
/* block: of the columns, for the scale */
__device__ __forceinline__ eight_t load_eight(const matrix_t &m, uint64_t row, uint64_t column, uint32_t left, uint32_t block)
{
	eight_t e = {};
	const uint8_t *const p = m.p + row * m.pitch;
	if (m.type == OFI_AMD_E4M3) {
		e.scale = row_at(m.scale, m.scale_pitch, row)[block];
		read_words<uint8_t, 8>(p + column, left, e.words);
	} else {
		read_words<uint16_t, 8>(p + column * 2, left, e.words);
	}
	return e;
}
template <typename T> __device__ __forceinline__ f32x8_t floats_of(u32x4_t w)
{
	return __builtin_convertvector(__builtin_bit_cast(raw_t<T, 8>, w), f32x8_t);
}
__device__ __forceinline__ f32x8_t values_of(const eight_t &e, int type)
{
	if (type == OFI_AMD_BFLOAT16) {
		return floats_of<bf16_t>(e.words);
	}
	if (type == OFI_AMD_FLOAT16) {
		return floats_of<f16_t>(e.words);
	}
	const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)e.words.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)e.words.x, true);
	const auto c = __builtin_amdgcn_cvt_pk_f32_fp8((int)e.words.y, false), d = __builtin_amdgcn_cvt_pk_f32_fp8((int)e.words.y, true);
	return f32x8_t{ a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1] } * e.scale;
}

__device__ __forceinline__ f32x8_t read_floats(const uint8_t *p, uint32_t left)
{
	f32x8_t v;
	read_words<float, 8>(p, left, v);
	return v;
}

/* Each value is rounded to the type once, to nearest even */
template <typename T, bool STREAM = false> __device__ __forceinline__ void write_as(uint8_t *p, uint32_t left, f32x8_t v)
{
	const auto r = __builtin_convertvector(v, raw_t<T, 8>);
	if (left >= 8) {
		auto *const q = reinterpret_cast<typename piece_t<T, 8>::anywhere *>(p);
		if (STREAM) {
			__builtin_nontemporal_store(r, q);
		} else {
			*q = r;
		}
	} else {
#pragma unroll
		for (uint32_t i = 0; i < 7; i++) {
			if (i < left) {
				reinterpret_cast<T *>(p)[i] = r[i];
			}
		}
	}
}

/* `left` of four values at p, which nothing reads again soon: zeros for the others */
__device__ __forceinline__ f32x4_t read_four(const float *p, uint32_t left)
{
	if (left >= 4) {
		return __builtin_nontemporal_load(reinterpret_cast<const piece_t<float, 4>::anywhere *>(p));
	}
	f32x4_t v;
	read_words<float, 4>(reinterpret_cast<const uint8_t *>(p), left, v);
	return v;
}
__device__ __forceinline__ void write_four(float *p, uint32_t left, f32x4_t v)
{
	if (left >= 4) {
		__builtin_nontemporal_store(v, reinterpret_cast<piece_t<float, 4>::anywhere *>(p));
	} else {
#pragma unroll
		for (uint32_t i = 0; i < 3; i++) {
			if (i < left) {
				p[i] = v[i];
			}
		}
	}
}

/* Eight columns of the row that is `row` behind `from`, if it is one of the rows there are, as far as columns are left; WHOLE: both are */
template <bool WHOLE, typename T, bool STREAM = false>
__device__ __forceinline__ void write_row_as(const matrix_t &m, uint64_t from, uint64_t column, uint32_t row, uint32_t rows, uint32_t left, f32x8_t v)
{
	if (WHOLE || (row < rows && left)) {
		write_as<T, STREAM>(m.p + from * m.pitch + column * sizeof(T) + row * m.pitch, WHOLE ? 8 : left, v);
	}
}

/* A block of 128 columns of a row, which sixteen lanes hold: values divided by their scale as the norms divide them (with a division's
 * rounding, then rounded to e4m3), and the scale.  All sixteen call. */
template <bool WHOLE>
__device__ __forceinline__ void write_block(const matrix_t &m, uint64_t from, uint64_t column, uint32_t block, uint32_t row, uint32_t rows, uint32_t left,
					    f32x8_t v)
{
	uint32_t most = 0;
#pragma unroll
	for (uint32_t i = 0; i < 8; i++) {
		const uint32_t bits = WHOLE || i < left ? abs_bits(v[i]) : 0u;
		most = bits > most ? bits : most;
	}
	const float scale = scale_of(max_bits_over<16>(most));
	const divisor_t by = divisor_of(scale);
	typedef uint32_t any8_t __attribute__((ext_vector_type(2), aligned(1)));
	any8_t w;
#pragma unroll
	for (int i = 0; i < 2; i++) {
		const int low = __builtin_amdgcn_cvt_pk_fp8_f32(quotient(v[4 * i], by), quotient(v[4 * i + 1], by), 0, false);
		w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(quotient(v[4 * i + 2], by), quotient(v[4 * i + 3], by), low, true);
	}
	if (WHOLE || (row < rows && left)) {
		if ((threadIdx.x & 15u) == 0) {
			row_at(m.scale, m.scale_pitch, from + row)[block] = scale;
		}
		uint8_t *const at = m.p + from * m.pitch + column + row * m.pitch;
		if (WHOLE || left >= 8) {
			*reinterpret_cast<any8_t *>(at) = w;
		} else {
#pragma unroll
			for (uint32_t i = 0; i < 7; i++) {
				if (i < left) {
					at[i] = (uint8_t)(w[i / 4] >> (8 * (i & 3)));
				}
			}
		}
	}
}

/* block: that of the columns */
template <bool WHOLE>
__device__ __forceinline__ void write_row(const matrix_t &m, uint64_t from, uint64_t column, uint32_t block, uint32_t row, uint32_t rows, uint32_t left,
					  f32x8_t v)
{
	if (m.type == OFI_AMD_E4M3) {
		write_block<WHOLE>(m, from, column, block, row, rows, left, v);
	} else if (m.type == OFI_AMD_BFLOAT16) {
		write_row_as<WHOLE, bf16_t>(m, from, column, row, rows, left, v);
	} else {
		write_row_as<WHOLE, f16_t>(m, from, column, row, rows, left, v);
	}
}

/* ---- activations ------------------------------------------------------------------------------------------------ */

/* 1 / (1 + e^-v): e^-v beyond float32's range leaves 0.  The reciprocal is the instruction's, off by one unit of 2^-24 or so */
__device__ __forceinline__ float logistic(float v) { return __builtin_amdgcn_rcpf(1.0f + __expf(-v)); }

/*
 * The normal distribution's share below v, and e^(-v^2/2).  Below 0 it is e^(-v^2/2) t P(t) with t = 1 / (1 + 0.45 |v| / sqrt 2): t P(t)
 * is half of e^(z^2) erfc(z), fitted over all z >= 0 (least squares in Chebyshev polynomials, weights drawn to the largest relative
 * errors), 3e-8 off at most.  In 32 bits 4e-7 of the share near 0; where it is tiny the bell's exponent, rounded twice, is off by up to 1.1 v^2
 * times 2^-24: 7e-7 of the share at v = -3, 2e-6 at -6, 4e-6 at -9, 7e-6 at -12 (bfloat16 rounds to 4e-3 of a value).
 * Rounded exactly (six more operations) the bell is 1.2e-7 off everywhere, and 8192 rows of 4096 with bias, gelu and residual 258 us for 253.
 * About 20 operations.
 */
__device__ __forceinline__ float normal_share(float v, float &bell)
{
	constexpr float kP[] = { 1.269426605e-01f, 1.269415725e-01f, 1.141360073e-01f, 8.762432375e-02f, 5.998388820e-02f,
				-1.120403144e-02f, 7.124375690e-02f, -1.503351952e-01f, 9.536814225e-02f, -2.070111786e-02f };
	const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(__builtin_fabsf(v), 0.45f * 0.70710678118654752f, 1.0f));
	float p = kP[9];
#pragma unroll
	for (int i = 8; i >= 0; i--) {
		p = __builtin_fmaf(p, t, kP[i]);
	}
	bell = __expf(-0.5f * v * v);
	const float below = p * t * bell;
	return v < 0.0f ? below : 1.0f - below;
}

template <int ACTIVATION> __device__ __forceinline__ float activated(float v)
{
	if constexpr (ACTIVATION == OFI_AMD_RELU) {
		return v < 0.0f ? 0.0f : v;
	} else if constexpr (ACTIVATION == OFI_AMD_SILU) {
		return v * logistic(v);
	} else if constexpr (ACTIVATION == OFI_AMD_GELU) {
		float bell;
		return v * normal_share(v, bell);
	} else {
		return v;
	}
}

/* The activation's value and its derivative.  0 has RELU's derivative 0. */
template <int ACTIVATION> __device__ __forceinline__ void activated_with_slope(float v, float &value, float &slope)
{
	if constexpr (ACTIVATION == OFI_AMD_RELU) {
		value = v < 0.0f ? 0.0f : v;
		slope = v > 0.0f ? 1.0f : v <= 0.0f ? 0.0f : v;
	} else if constexpr (ACTIVATION == OFI_AMD_SILU) {
		const float s = logistic(v);
		value = v * s;
		slope = __builtin_fmaf(value, 1.0f - s, s);
	} else if constexpr (ACTIVATION == OFI_AMD_GELU) {
		float bell;
		const float share = normal_share(v, bell);
		value = v * share;
		slope = __builtin_fmaf(v * 0.39894228040143268f, bell, share);
	} else {
		value = v;
		slope = 1.0f;
	}
}

/* f with the activation as a constant */
template <typename F> __device__ __forceinline__ void with_activation(int activation, F f)
{
	switch (activation) {
	case OFI_AMD_RELU: f(std::integral_constant<int, OFI_AMD_RELU>{}); break;
	case OFI_AMD_SILU: f(std::integral_constant<int, OFI_AMD_SILU>{}); break;
	case OFI_AMD_GELU: f(std::integral_constant<int, OFI_AMD_GELU>{}); break;
	default: f(std::integral_constant<int, OFI_AMD_NO_ACTIVATION>{});
	}
}

/* ---- on the host -------------------------------------------------------------------------------------------------- */

/* Bytes of an element of rows and weights, 0 for a type they do not have */
inline uint32_t product_type_size(int type)
{
	return type == OFI_AMD_BFLOAT16 || type == OFI_AMD_FLOAT16 ? 2u : type == OFI_AMD_E4M3 ? 1u : 0u;
}

inline int check_experts(const int32_t *d_offset, uint32_t n_experts, uint32_t max_rows, uint32_t a, uint32_t b)
{
	if (n_experts == 0 || a == 0 || b == 0 || (reinterpret_cast<uintptr_t>(d_offset) & 3u) || (!d_offset && n_experts != 1)) {
		return -EINVAL;
	}
	if (n_experts > kMostExperts || max_rows > 0x7fffffffu || a > kMostExpertWidth || b > kMostExpertWidth) {
		return -E2BIG;
	}
	return 0;
}

/* n_experts matrices of n rows */
inline bool stack_ok(const void *p, uint64_t pitch, uint64_t expert_pitch, uint32_t n_experts, uint64_t n, uint64_t bytes, uint32_t element)
{
	return rows_ok(p, pitch, n, bytes, element) && expert_pitch % element == 0 && expert_pitch < (1ull << 50) &&
	       (n_experts == 1 || expert_pitch >= (n - 1) * pitch + bytes);
}

inline bool scales_ok(const void *p, uint64_t pitch, uint64_t n, uint32_t blocks) { return rows_ok(p, pitch, n, 4ull * blocks, 4); }

constexpr uint32_t kMostPitch = 1u << 22;

/* Rows of `bytes` that whole chunks of 16 bytes make up, and that start on them, a tile of 256 rows within 31 bits */
inline bool in_chunks(const void *p, uint64_t pitch, uint64_t bytes)
{
	return ((reinterpret_cast<uintptr_t>(p) | pitch | bytes) & 15u) == 0 && pitch <= kMostPitch;
}

constexpr uint32_t kLanesOfLaunch = 1u << 31; /* within the 32 bits of a launch's size */

/* Calls launch(first tile, tiles) until all are launched, or one was not, which hipGetLastError then tells; `lanes` (a power of 2) are a
 * tile's, the tiles' number is a multiple of 8 */
template <typename F> inline void launch_tiles(uint64_t tiles, uint32_t lanes, F launch)
{
	const uint64_t most = kLanesOfLaunch / lanes;
	tiles = (tiles + 7) / 8 * 8;
	for (uint64_t at = 0; at < tiles; at += most) {
		if (!launch((uint32_t)at, (uint32_t)(tiles - at < most ? tiles - at : most))) {
			return;
		}
	}
}

/* Row tiles of BM that `max_rows` rows of experts can make */
inline uint64_t most_row_tiles(uint32_t max_rows, uint32_t n_experts, uint32_t bm)
{
	const uint64_t parts = n_experts < max_rows ? n_experts : max_rows; /* experts whose last tile may be part of one */
	return (max_rows - parts) / bm + parts;
}

/* Experts that have rows, at most, and the rows of each if all have the same */
inline void spread_of(uint32_t max_rows, uint32_t n_experts, uint32_t &experts, uint32_t &of_expert)
{
	experts = n_experts < max_rows ? n_experts : max_rows;
	of_expert = (max_rows + experts - 1) / experts;
}

/* Row tiles of 256, 128 or 64: the largest that the experts' rows fill and of which there are enough for the GPU.  256 with rows that
 * come through registers would not fit them. */
inline uint32_t row_tile_for(uint32_t max_rows, uint32_t n_experts, uint32_t n_tiles, bool most_is_256)
{
	uint32_t experts, of_expert;
	spread_of(max_rows, n_experts, experts, of_expert);
	auto fits = [&](uint32_t bm) {
		return of_expert > bm / 2 && (uint64_t)experts * ((of_expert + bm - 1) / bm) * n_tiles >= kComputeUnits;
	};
	return most_is_256 && fits(256) ? 256 : fits(128) ? 128 : 64;
}

/* Whether row tiles of 128 are filled and enough for two workgroups on each compute unit (sum_halves): 12,288 rows of 64 experts, 2048 summed to
 * 4096 columns 288 us, with one 302; 2048 rows of 16 are too few, and take 80 us in tiles of 64 */
inline bool pairs_fit(uint32_t max_rows, uint32_t n_experts, uint32_t n_tiles)
{
	uint32_t experts, of_expert;
	spread_of(max_rows, n_experts, experts, of_expert);
	return of_expert > 64 && (uint64_t)experts * ((of_expert + 127) / 128) * n_tiles >= 2 * kComputeUnits;
}

inline bool activation_ok(int a) { return a == OFI_AMD_NO_ACTIVATION || a == OFI_AMD_RELU || a == OFI_AMD_SILU || a == OFI_AMD_GELU; }

} // namespace ofi_amd

#endif
