/*
** Softmax cross entropy of the language model's head over the whole vocabulary, with its gradients
** (include/anni_adam.h, "the head's loss").
**
**   logits l[i][v] = sum_d x[i][d] w[d][v] + b[v]
**   nll[i] = log sum_v exp(l[i][v]) - l[i][target_i]
**   delta[i][v] = exp(l[i][v] - lse_i) - [v = target_i]
**   dx = scale delta w^T,  dw += scale x^T delta,  db += scale sum_i delta[i]
**
** scale is a factor of the float sums and no part of delta, which is rounded: nearly all of a loss' delta is -1 at
** the targets, a number of few bits, and a scale in it (a mean's 1 / rows) would be rounded alike in all of them, an
** error of up to 2^-8 that no sum averages out (96 tokens, db in bf16: 0.5 % off the formula's, 0.2 without).
**
** The first pass over the vocabulary keeps a maximum and a sum of exponentials per token and tile;
** scoring ends there, and nothing of the size of the logits is stored.  For gradients the second
** pass turns logits into delta (bf16, in the work area, a piece of the vocabulary of at most 512 MiB
** at a time), which the other two products read.  The logits come from the first pass where the work
** area has room for them, 8 bytes of traffic for each, and are computed again where it has not: a third
** more operations than the 6 rows d vocab that cannot be avoided (4096 tokens, 1536 x 100000: 1.39 +
** 0.38 ms against 1.20 + 1.38).  With float gradients delta is the sum of two bf16 numbers (16 bits
** of fraction, an error of 2^-17 against 2^-9), and the two products that read it run over both.
**
** The products are one template on bf16 operands with float sums: a workgroup of four or eight
** wavefronts owns a tile of the result and walks the contracted axis in steps of 64, which go from
** memory straight into LDS while the step before is multiplied, and feeds 32 x 32 x 16 matrix
** instructions from there.
** An operand lies in memory either with the contracted axis contiguous, or with its rows contiguous;
** the second kind is turned by the transposing LDS read, so nothing is transposed in memory.
**
** 4096 x 1536 x 100000 in bf16 runs at 900 TFLOP/s in the first pass (1.39 ms; 1050 without the logits it writes), 1100
** in dx and 1030 in dw, where the library's product of the same shape reaches 1090 (matrix pipes 69 % busy at 1.66 GHz; here 55 % at
** 2.05: the chip's power is what either runs into).
*/
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>
#include "adam_kernels.h"
#include "anni_adam.h"
#include "backend_state.h"
#include "head_plan.h"

namespace anni {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
/* sixteen bytes at any element: rows of an odd vocabulary are not aligned (the hardware does not mind) */
typedef u32x4 u32x4_any __attribute__((aligned(2)));

#define ANNI_LDS __attribute__((address_space(3)))

/*
** One operand of a product: element (r, k), 0 <= r < ROWS of the tile, k of a step.  BY_ROW: the
** rows are contiguous (element (r, k) at k ld + r), else the contracted axis (r ld + k).
**
** Its image in LDS is a list of 16-byte chunks in the order the lanes of a workgroup name them, so
** that a load can put them there itself, past the registers; a line's chunks are permuted by an
** exclusive or with its index (on the side of the memory address), so that the lanes of a fragment
** read spread over all banks.
**
** CHECK: the array ends inside tiles or its lines are not aligned to 16 bytes; such tiles go through
** registers.  Loads never leave the array, what lies beyond it reads as 0; no tile or step is
** launched whose first line lies beyond.
*/
struct Source {
	const uint16_t	*part[2];	/* second: the low halves, same shape */
	uint32_t	ld;
	int64_t		rows;		/* valid rows from row 0 */
	int64_t		depth;		/* valid length of the contracted axis */
	int		aligned;	/* every chunk is 16-byte aligned */
};

/*
** Sixteen bytes per lane from base + offset to 16 l behind `lds` (both uniform but the offset).  In
** assembly because behind the builtin the compiler waits for every such load before any read of LDS,
** and this one's whole point is to stay on its way; arrived() is the wait, before the barrier that
** hands the data over.  It writes no vector register, and loads of the compiler's own only ever wait for
** more than they must (they return in order).  m0 must have been written one instruction before its use;
** the clobber tells the compiler that a value of its own there is gone (its warning that the register is a
** reserved one says that it keeps none across statements anyway: the code is the same).
*/
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void memory_to_lds(const uint16_t *base, uint32_t offset, char *lds)
{
	const uint32_t at = (uint32_t)(uintptr_t)(ANNI_LDS char *)lds;

	asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
	    : : "s"(__builtin_amdgcn_readfirstlane(at)), "v"(offset), "s"(base) : "memory", "m0");
}
#pragma clang diagnostic pop

/* All but the LATER last loads have arrived. */
template <int LATER>
__device__ __forceinline__ void arrived(void)
{
	asm volatile("s_waitcnt vmcnt(%0)" : : "n"(LATER) : "memory");
}

/* One lane's place in an operand: kept across the steps, all else is uniform (registers are what is short). */
template <bool BY_ROW, bool CHECK, int ROWS, int THREADS>
struct Operand {
	static constexpr int kChunks = ROWS * kStep / 8 / THREADS;
	static constexpr int kBytes = ROWS * kStep * 2;
	static constexpr int kLine = BY_ROW ? ROWS / 8 : kStep / 8;	/* chunks to a line */
	static constexpr int kApart = THREADS / kLine;		/* lines between two chunks of a lane */
	uint32_t	offset;		/* elements from the tile's start to the lane's first chunk */
	int		line, col;	/* its line, and its place in it */
	u32x4		hold[CHECK ? kChunks : 1];
	int		short_by;	/* lines from the lane's first to the end: what lies beyond is 0 */
	bool		held;

	static __device__ __forceinline__ int turn(int line)
	{
		/*
		** LDS serves 256 bytes at a time: sixteen lines of one chunk, or by row 32 lanes with half a chunk
		** each, four lines of four chunks.  Short lines share those 256 bytes.
		*/
		if (!BY_ROW)
			return (line >> 1) & 7;
		return kLine == 8 ? (line & 2) << 1 : (line & 3) << 2;
	}

	__device__ __forceinline__ void init(const Source &src, int tid)
	{
		static_assert(kApart % (BY_ROW ? 4 : 16) == 0, "turn() is the same for all chunks of a lane");
		line = tid / kLine;
		col = ((tid % kLine) ^ turn(line)) * 8;
		offset = (uint32_t)line * src.ld + (uint32_t)col;
	}

	/* Do all of the tile's steps go through registers? */
	static __device__ __forceinline__ bool always_held(const Source &src, int64_t row0)
	{
		return CHECK && (src.rows - row0 < ROWS || !src.aligned);
	}

	/* Step `s` (of `steps` per part) on its way to `lds`, or into registers. */
	__device__ __forceinline__ void start(const Source &src, int64_t row0, int s, int steps, char *lds, int tid)
	{
		const int part = s >= steps ? 1 : 0;
		const int64_t k0 = (int64_t)(s - part * steps) * kStep;
		const uint16_t *base = src.part[part] + (BY_ROW ? k0 * src.ld + row0 : row0 * src.ld + k0);
		const int64_t rows_left = src.rows - row0;
		const int64_t depth_left = src.depth - k0;

		held = CHECK && (rows_left < ROWS || depth_left < kStep || !src.aligned);
		if (!CHECK || !held) {
			const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

#pragma unroll
			for (int i = 0; i < kChunks; i++)
				memory_to_lds(base + (int64_t)(i * kApart) * src.ld, offset * 2,
				    lds + (i * THREADS + wave * 64) * 16);
			return;
		}
		if constexpr (CHECK) {
			const int lines = (int)(BY_ROW ? (depth_left < kStep ? depth_left : kStep)
			    : (rows_left < ROWS ? rows_left : ROWS));
			const int cols = (int)(BY_ROW ? (rows_left < ROWS ? rows_left : ROWS)
			    : (depth_left < kStep ? depth_left : kStep));

			/* a lane's chunks share their place in the line: all of them whole, or none */
			if (col + 8 <= cols) {
#pragma unroll
				for (int i = 0; i < kChunks; i++) {
					const int at = line + i * kApart;

					hold[i] = *(const u32x4_any *)(base + (uint32_t)(at < lines ? at : lines - 1) * src.ld
					    + (uint32_t)col);
				}
			} else {
#pragma unroll
				for (int i = 0; i < kChunks; i++) {
					const int at = line + i * kApart;
					const uint16_t *q = base + (uint32_t)(at < lines ? at : lines - 1) * src.ld + (uint32_t)col;
					u32x4 w = {0u, 0u, 0u, 0u};

					/* from the last element down, each pushing the others up */
#pragma unroll 1
					for (int j = 7; j >= 0; j--) {
						const uint32_t e = col + j < cols ? q[j] : 0u;

						w.w = (w.w << 16) | (w.z >> 16);
						w.z = (w.z << 16) | (w.y >> 16);
						w.y = (w.y << 16) | (w.x >> 16);
						w.x = (w.x << 16) | e;
					}
					hold[i] = w;
				}
			}
			short_by = lines - line;
		}
	}

	/* What start() left in registers goes to `lds`. */
	__device__ __forceinline__ void finish(char *lds, int tid) const
	{
		if constexpr (CHECK) {
			if (held)
#pragma unroll
				for (int i = 0; i < kChunks; i++)
					*(u32x4 *)(lds + (tid + i * THREADS) * 16) = i * kApart < short_by ? hold[i]
					    : u32x4{0u, 0u, 0u, 0u};
		}
	}

	/*
	** Where a lane reads its fragments of BLOCKS blocks of 32 rows from row r0 on.  A fragment of a
	** 32 x 32 x 16 product: lane l holds row l % 32 of the block, places 16 sub + 8 (l / 32) .. + 7.
	** What the exclusive or touches needs an address of its own (by row: the block; else: the slice),
	** the rest is a constant distance.
	*/
	template <int BLOCKS>
	struct Reader {
		ANNI_LDS const char *at[BY_ROW ? BLOCKS : kStep / 16];

		__device__ __forceinline__ void init(const char *lds, int r0, int lane)
		{
			ANNI_LDS const char *base = (ANNI_LDS const char *)lds;

			if constexpr (BY_ROW) {
				/* each 16 lanes read four lines of 16 rows and get them turned: a lane one row of four lines */
				const int ln = (lane >> 5) * 8 + ((lane & 15) >> 2);

#pragma unroll
				for (int i = 0; i < BLOCKS; i++) {
					const int row = r0 + i * 32 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;

					at[i] = base + ln * kLine * 16 + ((row >> 3) ^ turn(ln)) * 16 + (row & 4) * 2;
				}
			} else {
				const int row = r0 + (lane & 31);

#pragma unroll
				for (int sub = 0; sub < kStep / 16; sub++)
					at[sub] = base + row * kLine * 16 + ((sub * 2 + (lane >> 5)) ^ turn(row)) * 16;
			}
		}

		__device__ __forceinline__ void move(int bytes)
		{
#pragma unroll
			for (int i = 0; i < (BY_ROW ? BLOCKS : kStep / 16); i++)
				at[i] += bytes;
		}

		__device__ __forceinline__ bf16x8 fragment(int block, int sub) const
		{
			if constexpr (BY_ROW) {
				ANNI_LDS const char *q = at[block] + sub * 16 * kLine * 16;
				union { i16x4 h[2]; bf16x8 f; } u;

				u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ANNI_LDS i16x4 *)q);
				u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ANNI_LDS i16x4 *)(q + 4 * kLine * 16));
				return u.f;
			} else {
				return *(ANNI_LDS const bf16x8 *)(at[sub] + block * 32 * kLine * 16);
			}
		}
	};
};

/*
** acc += A B^T over the steps [from, to): acc[i][j] is the 32 x 32 block (i, j) of the wavefront's part.
**
** LDS holds STAGES steps: one that is computed on, the others on their way.  The fragments of a
** 16-deep slice are read while the slice before is multiplied.  The one barrier of a step stands
** before its last slice's products, whose fragments are in registers by then: behind it the first
** fragments of the next step are read under those products, and the stage that everyone has read is
** filled again.  Large tiles are bound by the matrix pipes and take two stages; the small ones are
** bound by memory and need more on its way.
**
** Operands that go through registers (`held`) are one step ahead whatever STAGES, or, where that is
** only the last step of an axis that ends inside it, are put away as soon as they come.
**
** SUMS: on request also sum[j] = the sums of B's rows over the contracted axis (every register of a
** lane the same), by products with ones: two more matrix instructions to eight.
*/
template <class A, class B, int MB, int NB, int STAGES, bool SUMS>
struct Product {
	f32x16	acc[MB][NB];
	f32x16	sum[SUMS ? NB : 1];

	struct Slice {
		bf16x8	a[MB], b[NB];
	};

	typedef typename A::template Reader<MB> ReadA;
	typedef typename B::template Reader<NB> ReadB;

	__device__ __forceinline__ void clear(void)
	{
#pragma unroll
		for (int i = 0; i < MB; i++)
#pragma unroll
			for (int j = 0; j < NB; j++)
				acc[i][j] = f32x16{};
		if constexpr (SUMS)
#pragma unroll
			for (int j = 0; j < NB; j++)
				sum[j] = f32x16{};
	}

	static __device__ __forceinline__ void read(Slice &f, const ReadA &ra, const ReadB &rb, int sub)
	{
#pragma unroll
		for (int i = 0; i < MB; i++)
			f.a[i] = ra.fragment(i, sub);
#pragma unroll
		for (int j = 0; j < NB; j++)
			f.b[j] = rb.fragment(j, sub);
	}

	__device__ __forceinline__ void multiply(const Slice &f, bool sums)
	{
		if constexpr (SUMS)
			if (sums) {
				const u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};

#pragma unroll
				for (int j = 0; j < NB; j++)
					sum[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, ones), f.b[j],
					    sum[j], 0, 0, 0);
			}
#pragma unroll
		for (int i = 0; i < MB; i++)
#pragma unroll
			for (int j = 0; j < NB; j++)
				acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.a[i], f.b[j], acc[i][j], 0, 0, 0);
	}

	/* ra, rb: the first row of the wavefront's part in the tiles. */
	__device__ __forceinline__ void run(const Source &sa, const Source &sb, int64_t row_a, int64_t row_b, int from,
		int to, int steps, char *lds, int ra, int rb, int tid, bool sums)
	{
		constexpr int kStage = A::kBytes + B::kBytes;
		constexpr int kLater = (STAGES - 2) * (A::kChunks + B::kChunks);	/* loads of the steps after the next */
		const int lane = tid & 63;
		/* steps ahead: all stages, if nothing but an axis' last step goes through registers */
		const bool deep = STAGES > 2 && !A::always_held(sa, row_a) && !B::always_held(sb, row_b);
		const int ahead = deep ? STAGES - 1 : 1;
		A a;
		B b;
		ReadA reada;
		ReadB readb;
		Slice f0, f1;
		int here = 0;			/* where the stage that is computed on begins */

		static_assert(kStep == 64, "four slices");
		clear();
		if (from >= to)
			return;		/* an empty slice of the axis; the same in every lane of the workgroup */
		a.init(sa, tid);
		b.init(sb, tid);
		for (int k = 0; k < ahead && from + k < to; k++) {
			a.start(sa, row_a, from + k, steps, lds + k * kStage, tid);
			b.start(sb, row_b, from + k, steps, lds + k * kStage + A::kBytes, tid);
			a.finish(lds + k * kStage, tid);
			b.finish(lds + k * kStage + A::kBytes, tid);
		}
		arrived<0>();
		__syncthreads();
		reada.init(lds, ra, lane);
		readb.init(lds + A::kBytes, rb, lane);
		if (from + ahead < to)
			begin(a, b, sa, sb, row_a, row_b, from + ahead, steps, lds + ahead * kStage, deep, tid);
		read(f0, reada, readb, 0);
#pragma unroll 1
		for (int s = from; s < to; s++) {
			const int next = here + kStage < (ahead + 1) * kStage ? here + kStage : 0;

			read(f1, reada, readb, 1);
			multiply(f0, sums);
			__builtin_amdgcn_sched_barrier(0);
			read(f0, reada, readb, 2);
			multiply(f1, sums);
			__builtin_amdgcn_sched_barrier(0);
			read(f1, reada, readb, 3);
			multiply(f0, sums);
			__builtin_amdgcn_sched_barrier(0);
			if (s + 1 < to) {
				if (!deep) {
					a.finish(lds + next, tid);
					b.finish(lds + next + A::kBytes, tid);
				}
				if (deep && s + ahead < to)
					arrived<kLater>();
				else
					arrived<0>();
			}
			__syncthreads();
			/* ahead of the products: issuing those takes the wavefront as long as they run */
			if (s + 1 + ahead < to)
				begin(a, b, sa, sb, row_a, row_b, s + 1 + ahead, steps, lds + here, deep, tid);
			reada.move(next - here);
			readb.move(next - here);
			here = next;
			/* behind the last step this reads what lies in LDS, for nothing */
			read(f0, reada, readb, 0);
			multiply(f1, sums);
			__builtin_amdgcn_sched_barrier(0);
		}
		/* those reads are over before a caller's stores */
		__syncthreads();
	}

	static __device__ __forceinline__ void begin(A &a, B &b, const Source &sa, const Source &sb, int64_t row_a,
		int64_t row_b, int s, int steps, char *lds, bool deep, int tid)
	{
		a.start(sa, row_a, s, steps, lds, tid);
		b.start(sb, row_b, s, steps, lds + A::kBytes, tid);
		if (deep) {
			a.finish(lds, tid);
			b.finish(lds + A::kBytes, tid);
		}
	}
};

/* Row of register r of a 32 x 32 block in lane l; the column is l % 32. */
__device__ __forceinline__ int block_row(int r, int lane)
{
	return 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
}

/*
** Which tile a workgroup takes, and which of `slices` of its contracted axis.  Consecutive workgroups
** go to the eight dies in turn, so die x gets the x-th eighth of the list, and the list runs, slice
** by slice, over bands of eight tiles of the short axis: what a die works on at one time shares operands in its
** level-two cache.
*/
__device__ __forceinline__ bool tile_of(int64_t id, int64_t tiles_a, int64_t tiles_b, int slices, int64_t *ta,
	int64_t *tb, int *slice)
{
	const int64_t tiles = tiles_a * tiles_b;
	const int64_t n = tiles * slices;
	const int64_t per = (n + 7) / 8;
	int64_t at = (id & 7) * per + (id >> 3);
	const int64_t band = 8 * tiles_a;

	if ((id >> 3) >= per || at >= n)
		return false;
	*slice = (int)(at / tiles);
	at -= *slice * tiles;
	const int64_t g = at / band;
	const int64_t in = at - g * band;
	const int64_t wide = tiles_b - g * 8 < 8 ? tiles_b - g * 8 : 8;

	*ta = in / wide;
	*tb = g * 8 + in % wide;
	return true;
}

/* ---- clean copies of x, the targets, the bias, and w's lines --------------------------------------------- */

struct RowArgs {
	const uint16_t	*x;
	int64_t		ld_x;
	const int32_t	*target;
	int64_t		rows, rows_pad;
	int		d, d_pad, vocab;
	int64_t		vocab_pad;
	const float	*bias;		/* may be NULL */
	uint16_t	*xs;		/* [rows_pad][ld_xs] */
	int64_t		ld_xs;
	int32_t		*ts;
	float		*bs;
	const uint16_t	*w;
	uint16_t	*ws;		/* [d][ld_ws], or NULL */
	int64_t		ld_ws;
};

/* Eight elements from column c on of a line of n; zeros beyond. */
__device__ __forceinline__ u32x4 eight_of(const uint16_t *line, int c, int n)
{
	u32x4 w = {0u, 0u, 0u, 0u};

	if (c + 8 <= n) {
		w = *(const u32x4_any *)(line + c);
	} else if (c < n) {
		uint32_t e[8];

#pragma unroll
		for (int j = 0; j < 8; j++)
			e[j] = c + j < n ? line[c + j] : 0u;
		w = u32x4{e[0] | (e[1] << 16), e[2] | (e[3] << 16), e[4] | (e[5] << 16), e[6] | (e[7] << 16)};
	}
	return w;
}

/*
** xs[rows_pad][d_pad] = x, with zeros for rows without a target (whatever x holds there) and beyond
** rows and d; ts = target, -1 for rows without one; bs = bias, -inf beyond the vocabulary (which has
** probability 0 there, and so no delta).  The products then need no masks.  ws[d][vocab_pad] = w where
** its lines are to be aligned.
*/
__global__ __launch_bounds__(kThreads) void head_rows_kernel(RowArgs a)
{
	const int64_t per = a.d_pad / 8;
	const int64_t n = a.rows_pad * per;

	for (int64_t q = (int64_t)blockIdx.x * kThreads + threadIdx.x; q < n; q += (int64_t)gridDim.x * kThreads) {
		const int64_t r = q / per;
		const int c = (int)(q - r * per) * 8;
		const int32_t t = r < a.rows ? a.target[r] : -1;
		const bool live = t >= 0 && t < a.vocab;
		*(u32x4 *)(a.xs + r * a.ld_xs + c) = live ? eight_of(a.x + r * a.ld_x, c, a.d) : u32x4{0u, 0u, 0u, 0u};
		if (c == 0)
			a.ts[r] = live ? t : -1;
	}
	for (int64_t v = (int64_t)blockIdx.x * kThreads + threadIdx.x; v < a.vocab_pad;
	    v += (int64_t)gridDim.x * kThreads)
		a.bs[v] = v >= a.vocab ? -INFINITY : a.bias ? a.bias[v] : 0.0f;
	if (!a.ws)
		return;
	const int64_t per_w = a.vocab_pad / 8;

	for (int64_t q = (int64_t)blockIdx.x * kThreads + threadIdx.x; q < a.d * per_w; q += (int64_t)gridDim.x * kThreads) {
		const int64_t r = q / per_w;
		const int c = (int)(q - r * per_w) * 8;

		*(u32x4 *)(a.ws + r * a.ld_ws + c) = eight_of(a.w + r * a.vocab, c, a.vocab);
	}
}

/* ---- logits, by tile: their softmax's running statistics, or delta ----------------------------- */

struct LogitArgs {
	Source		w;		/* by row: w[d][vocab] */
	Source		x;		/* xs */
	const float	*bias;		/* bs */
	const int32_t	*target;	/* ts */
	int		steps;
	int64_t		tiles_v, tiles_t;
	int64_t		rows_pad;
	/* statistics */
	f32x2		*part;		/* [tiles_v][rows_pad]: maximum, sum of exp(l - maximum) */
	float		*target_logit;
	f32x4		*kept;		/* the logits themselves, see kept_block(); NULL: nobody wants them */
	int64_t		kept_v;		/* blocks along the vocabulary */
	/* delta */
	const float	*lse;
	int64_t		v0;		/* first vocabulary place of this piece */
	uint16_t	*delta;		/* [rows_pad][ld_delta], low halves behind the high ones */
	uint16_t	*delta_low;
	int64_t		ld_delta;
};

enum { kStats = 0, kDelta = 1, kDeltaPair = 2, kStatsKeep = 3 };

/*
** Logits that stay in memory lie as the accumulators do: blocks of 32 places by 32 tokens, four
** sixteen-byte words per lane, so that they go out and come back in whole kilobytes.
*/
__device__ __forceinline__ f32x4 *kept_block(f32x4 *kept, int64_t kept_v, int64_t token, int64_t place)
{
	return kept + ((token / 32) * kept_v + place / 32) * 256;
}

template <class S, int MODE>
__global__ __launch_bounds__(S::threads) void head_logits_kernel(LogitArgs a)
{
	constexpr int TT = S::tokens, TV = S::side;
	constexpr int WM = S::waves_side, WN = S::waves_tokens;
	typedef Operand<true, true, TV, S::threads> W;
	typedef Operand<false, false, TT, S::threads> X;
	constexpr int MB = TV / WM / 32, NB = TT / WN / 32;
	__shared__ __align__(16) char lds[S::stages * (W::kBytes + X::kBytes)];
	const int tid = threadIdx.x;
	const int lane = tid & 63;
	const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
	const int wm = wave / WN, wn = wave % WN;
	int64_t tv, tt;
	int whole;
	Product<W, X, MB, NB, S::stages, false> prod;
	auto &acc = prod.acc;

	if (!tile_of(blockIdx.x, a.tiles_v, a.tiles_t, 1, &tv, &tt, &whole))
		return;
	const int64_t v_tile = a.v0 + tv * TV;
	const int64_t t_tile = tt * TT;
	const int64_t v_base = v_tile + wm * (MB * 32);

	prod.run(a.w, a.x, v_tile, t_tile, 0, a.steps, a.steps, lds, wm * (MB * 32), wn * (NB * 32), tid, false);
#pragma unroll
	for (int i = 0; i < MB; i++)
#pragma unroll
		for (int q = 0; q < 4; q++) {
			const f32x4 b = *(const f32x4 *)(a.bias + v_base + i * 32 + block_row(4 * q, lane));

#pragma unroll
			for (int j = 0; j < NB; j++)
#pragma unroll
				for (int k = 0; k < 4; k++)
					acc[i][j][4 * q + k] += b[k];
			if ((q & 1) == 1)
				__builtin_amdgcn_sched_barrier(0);	/* all loads ahead of all sums take registers that there are not */
		}
	if constexpr (MODE == kStatsKeep) {
#pragma unroll
		for (int i = 0; i < MB; i++)
#pragma unroll
			for (int j = 0; j < NB; j++) {
				f32x4 *block = kept_block(a.kept, a.kept_v, t_tile + wn * (NB * 32) + j * 32, v_base + i * 32);

#pragma unroll
				for (int q = 0; q < 4; q++)
					__builtin_nontemporal_store(f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1],
					    acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]}, block + q * 64 + lane);
			}
	}
	if constexpr (MODE == kStats || MODE == kStatsKeep) {
		f32x2 *red = (f32x2 *)lds;	/* [WM][TT] */

#pragma unroll
		for (int j = 0; j < NB; j++) {
			const int t = wn * (NB * 32) + j * 32 + (lane & 31);
			/* the target's place among the lane's rows: a constant for each register */
			const int want = a.target[t_tile + t] - (int)v_base - block_row(0, lane);
			float top = -INFINITY, sum = 0.0f, hit = 0.0f;

#pragma unroll
			for (int i = 0; i < MB; i++)
#pragma unroll
				for (int r = 0; r < 16; r++) {
					top = fmaxf(top, acc[i][j][r]);
					if (want == i * 32 + block_row(r, 0))
						hit = acc[i][j][r];
				}
			top = fmaxf(top, __shfl_xor(top, 32, 64));
			/* nothing but -inf: every exponential is 0 against any finite maximum */
			const float ref = top == -INFINITY ? 0.0f : top;

#pragma unroll
			for (int i = 0; i < MB; i++)
#pragma unroll
				for (int r = 0; r < 16; r++)
					sum += __expf(acc[i][j][r] - ref);
			sum += __shfl_xor(sum, 32, 64);
			if (lane < 32)
				red[wm * TT + t] = f32x2{top, sum};
			if (want >= 0 && want < MB * 32 && (want & 4) == 0)
				a.target_logit[t_tile + t] = hit;
		}
		__syncthreads();
		for (int t = tid; t < TT; t += S::threads) {
			float top = -INFINITY, sum = 0.0f;

#pragma unroll
			for (int k = 0; k < WM; k++)
				top = fmaxf(top, red[k * TT + t].x);
			const float ref = top == -INFINITY ? 0.0f : top;

#pragma unroll
			for (int k = 0; k < WM; k++)
				sum += red[k * TT + t].y * __expf(red[k * TT + t].x - ref);
			a.part[tv * a.rows_pad + t_tile + t] = f32x2{top, sum};
		}
	} else {
#pragma unroll
		for (int j = 0; j < NB; j++) {
			const int64_t t = t_tile + wn * (NB * 32) + j * 32 + (lane & 31);
			const int want = a.target[t] - (int)v_base - block_row(0, lane);
			const bool live = a.target[t] >= 0;
			const float lse = a.lse[t];

#pragma unroll
			for (int i = 0; i < MB; i++)
#pragma unroll
				for (int r = 0; r < 16; r++) {
					float p = __expf(acc[i][j][r] - lse);

					if (want == i * 32 + block_row(r, 0))
						p -= 1.0f;
					acc[i][j][r] = live ? p : 0.0f;
				}
		}
		/*
		** A lane holds four places of one token at a time; the tile goes through LDS so that memory is
		** written in whole lines of 512 bytes (straight from the registers: 16 of every line at a time,
		** 0.35 ms slower for 4096 tokens of the 555M head).  Chunks are rotated by the token.
		*/
#pragma unroll
		for (int part = 0; part < (MODE == kDeltaPair ? 2 : 1); part++) {
			uint16_t *out = part ? a.delta_low : a.delta;

#pragma unroll
			for (int j = 0; j < NB; j++)
#pragma unroll
				for (int i = 0; i < MB; i++)
#pragma unroll
					for (int q = 0; q < 4; q++) {
						const int t = wn * (NB * 32) + j * 32 + (lane & 31);
						const int row = wm * (MB * 32) + i * 32 + block_row(4 * q, lane);
						u32x2 w;

						w.x = bf16_rne2(acc[i][j][4 * q], acc[i][j][4 * q + 1]);
						w.y = bf16_rne2(acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
						*(u32x2 *)(lds + t * (TV * 2) + ((row >> 3) ^ (t & (TV / 8 - 1))) * 16 + (row & 4) * 2) = w;
						if constexpr (MODE == kDeltaPair) {
							/* what the rounding left over, for the second part */
							acc[i][j][4 * q] -= __uint_as_float(w.x << 16);
							acc[i][j][4 * q + 1] -= __uint_as_float(w.x & 0xffff0000u);
							acc[i][j][4 * q + 2] -= __uint_as_float(w.y << 16);
							acc[i][j][4 * q + 3] -= __uint_as_float(w.y & 0xffff0000u);
						}
					}
			__syncthreads();
#pragma unroll
			for (int u = 0; u < TT * (TV / 8) / S::threads; u++) {
				const int c = u * S::threads + tid;
				const int t = c / (TV / 8);
				const int chunk = c % (TV / 8);

				*(u32x4 *)(out + (t_tile + t) * a.ld_delta + (v_tile - a.v0) + chunk * 8) =
				    *(const u32x4 *)(lds + t * (TV * 2) + (chunk ^ (t & (TV / 8 - 1))) * 16);
			}
			if (part == 0 && MODE == kDeltaPair)
				__syncthreads();
		}
	}
}

/* ---- the statistics of all tiles -> lse and nll ------------------------------------------------ */

constexpr int kFewTiles = 32;

/*
** Few tiles: a lane folds its token's alone, all on their way at once, by their common maximum.  The same
** function (so the same bits) here and in the pass over kept logits, which then needs no launch ahead of it.
*/
__device__ __forceinline__ f32x2 few_stats(const f32x2 *part, int64_t rows_pad, int tiles, int64_t t)
{
	f32x2 p[kFewTiles];
	float top = -INFINITY, sum = 0.0f;

#pragma unroll
	for (int k = 0; k < kFewTiles; k++)
		p[k] = k < tiles ? part[k * rows_pad + t] : f32x2{-INFINITY, 0.0f};
#pragma unroll
	for (int k = 0; k < kFewTiles; k++)
		top = fmaxf(top, p[k].x);
	const float ref = top == -INFINITY ? 0.0f : top;

#pragma unroll
	for (int k = 0; k < kFewTiles; k++)
		sum += p[k].y * __expf(p[k].x - ref);
	return f32x2{top, sum};
}

struct FinishArgs {
	const f32x2	*part;
	const float	*target_logit;
	const int32_t	*target;
	int64_t		tiles_v, rows, rows_pad;
	float		*lse;
	float		*nll;
};

/* The statistics (top, sum) and p of disjoint parts of the vocabulary -> of both. */
__device__ __forceinline__ void fold_stats(float &top, float &sum, f32x2 p)
{
	const float m = fmaxf(top, p.x);
	const float ref = m == -INFINITY ? 0.0f : m;

	sum = sum * __expf(top - ref) + p.y * __expf(p.x - ref);
	top = m;
}

/* lse of token t, and its nll. */
__device__ __forceinline__ float put_nll(const FinishArgs &a, int64_t t, f32x2 stats)
{
	const float log_sum = logf(stats.y);
	const float lse = stats.x + log_sum;

	if (a.lse)
		a.lse[t] = lse;
	if (t < a.rows)
		a.nll[t] = a.target[t] >= 0 ? (stats.x - a.target_logit[t]) + log_sum : 0.0f;
	return lse;
}

/*
** 16 tokens to a workgroup; its groups of 16 lanes, a wavefront of them for every four tiles up to
** sixteen wavefronts, share the tiles, eight at a time on their way (782 tiles, 96 tokens: 5.5 us;
** with 64 tokens to a workgroup and four on their way 11).  Folded in a fixed order.
*/
constexpr int kFinishWaves = 16;
constexpr int kFinishTokens = 16;

__global__ __launch_bounds__(kFinishWaves * 64) void head_finish_kernel(FinishArgs a)
{
	__shared__ f32x2 red[kFinishWaves * 64 / kFinishTokens][kFinishTokens];
	const int parts = blockDim.x / kFinishTokens;
	const int token = threadIdx.x % kFinishTokens;
	const int share = threadIdx.x / kFinishTokens;
	const int64_t t = (int64_t)blockIdx.x * kFinishTokens + token;
	float top = -INFINITY, sum = 0.0f;

	if (a.tiles_v <= kFewTiles) {
		if (share == 0)
			put_nll(a, t, few_stats(a.part, a.rows_pad, (int)a.tiles_v, t));
		return;
	}
	for (int64_t k0 = share; k0 < a.tiles_v; k0 += 8 * parts) {
		f32x2 p[8];
		float m = top;

#pragma unroll
		for (int u = 0; u < 8; u++) {
			const int64_t k = k0 + u * parts;

			p[u] = f32x2{-INFINITY, 0.0f};
			if (k < a.tiles_v)
				p[u] = a.part[k * a.rows_pad + t];
		}
#pragma unroll
		for (int u = 0; u < 8; u++)
			m = fmaxf(m, p[u].x);
		const float ref = m == -INFINITY ? 0.0f : m;

		sum *= __expf(top - ref);
#pragma unroll
		for (int u = 0; u < 8; u++)
			sum += p[u].y * __expf(p[u].x - ref);
		top = m;
	}
	red[share][token] = f32x2{top, sum};
	__syncthreads();
	/* the first wavefront: four lanes to a token, then those */
	if (threadIdx.x >= 64)
		return;
	for (int k = share + 4; k < parts; k += 4)
		fold_stats(top, sum, red[k][token]);
#pragma unroll
	for (int k = kFinishTokens; k < 64; k *= 2) {
		const f32x2 p = {__shfl_xor(top, k, 64), __shfl_xor(sum, k, 64)};

		fold_stats(top, sum, p);
	}
	if (share != 0)
		return;
	put_nll(a, t, f32x2{top, sum});
}

/* ---- delta from logits that were kept ------------------------------------------------------------ */

struct DeltaArgs {
	FinishArgs	finish;		/* few tiles: the tokens' statistics are folded here */
	int		few;
	f32x4		*kept;
	int64_t		kept_v;
	const int32_t	*target;
	const float	*lse;
	int		vocab;
	int64_t		v0;		/* of this piece */
	int64_t		groups_v;	/* of 128 places, in this piece */
	uint16_t	*delta;
	uint16_t	*delta_low;
	int64_t		ld_delta;
};

/*
** A stream: 4 bytes in and 2 (or 4) out for each.  32 tokens by 128 places to a workgroup, a block to
** a wavefront, turned in LDS into lines of 256 bytes.  4096 x 50000: 190 us, 6.4 TB/s; two parts,
** 4096 x 16384: 92 us, 5.8 TB/s.
*/
template <bool PAIR>
__global__ __launch_bounds__(kThreads) void head_delta_kernel(DeltaArgs a)
{
	__shared__ __align__(16) char lds[PAIR ? 2 : 1][32 * 256];
	const int tid = threadIdx.x;
	const int lane = tid & 63;
	const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
	const int64_t t0 = blockIdx.x / a.groups_v * 32;
	const int64_t c0 = blockIdx.x % a.groups_v * 128;	/* from the piece's start */
	const int64_t v_base = a.v0 + c0 + wave * 32;
	const int t = lane & 31;
	const int target = a.target[t0 + t];
	const int want = target - (int)v_base - block_row(0, lane);
	/* blocks that lie beyond the vocabulary as a whole may not have been written */
	const bool inside = v_base < a.vocab;
	const f32x4 *block = kept_block(a.kept, a.kept_v, t0, inside ? v_base : 0) + lane;
	f32x4 x[4];

	static_assert(kThreads == 256, "four blocks of 32 places");
#pragma unroll
	for (int q = 0; q < 4; q++)
		x[q] = __builtin_nontemporal_load(block + q * 64);
	float lse;

	if (a.few) {
		const f32x2 stats = few_stats(a.finish.part, a.finish.rows_pad, a.few, t0 + t);

		lse = stats.x + logf(stats.y);
		if (c0 == 0 && a.v0 == 0 && tid < 32)
			put_nll(a.finish, t0 + t, stats);
	} else {
		lse = a.lse[t0 + t];
	}
#pragma unroll
	for (int q = 0; q < 4; q++) {
		const int chunk = (wave * 4 + q) ^ (t & 15);
		u32x2 w;

#pragma unroll
		for (int k = 0; k < 4; k++) {
			float p = __expf(x[q][k] - lse);

			if (want == 8 * q + k)
				p -= 1.0f;
			x[q][k] = target >= 0 && inside ? p : 0.0f;
		}
		w.x = bf16_rne2(x[q].x, x[q].y);
		w.y = bf16_rne2(x[q].z, x[q].w);
		*(u32x2 *)(lds[0] + t * 256 + chunk * 16 + (lane >> 5) * 8) = w;
		if constexpr (PAIR) {
			const u32x2 low = {bf16_rne2(x[q].x - __uint_as_float(w.x << 16), x[q].y - __uint_as_float(w.x & 0xffff0000u)),
			    bf16_rne2(x[q].z - __uint_as_float(w.y << 16), x[q].w - __uint_as_float(w.y & 0xffff0000u))};

			*(u32x2 *)(lds[1] + t * 256 + chunk * 16 + (lane >> 5) * 8) = low;
		}
	}
	__syncthreads();
#pragma unroll
	for (int part = 0; part < (PAIR ? 2 : 1); part++)
#pragma unroll
		for (int u = 0; u < 2; u++) {
			const int line = u * 16 + (tid >> 4);
			const int chunk = tid & 15;

			*(u32x4 *)((part ? a.delta_low : a.delta) + (t0 + line) * a.ld_delta + c0 + chunk * 8) =
			    *(const u32x4 *)(lds[part] + line * 256 + (chunk ^ (line & 15)) * 16);
		}
}

/* ---- dx ---------------------------------------------------------------------------------------- */

struct DxArgs {
	Source		delta;
	Source		w;
	int		steps, parts, splits;
	int64_t		tiles_t, tiles_d;
	float		*slot;		/* [splits][rows_pad][d_slot] */
	int64_t		rows_pad;
	int		d_slot;
	int		add;		/* later pieces of the vocabulary add to the slots */
};

/*
** Each slice of the contracted axis (the vocabulary) has a slot of its own.  w's lines are the contiguous
** axis: 128 bytes of each per step.  4096 x 1536 x 50000 570 us, 1100 TFLOP/s; 96 x 1536 x 100000
** 104 us for w's 307 MB.
*/
template <class S>
__global__ __launch_bounds__(S::threads) void head_dx_kernel(DxArgs a)
{
	constexpr int TT = S::tokens, TD = S::side;
	constexpr int WM = S::waves_tokens, WN = S::waves_side;
	typedef Operand<false, false, TT, S::threads> D;
	typedef Operand<false, true, TD, S::threads> W;
	constexpr int MB = TT / WM / 32, NB = TD / WN / 32;
	__shared__ __align__(16) char lds[S::stages * (D::kBytes + W::kBytes)];
	const int tid = threadIdx.x;
	const int lane = tid & 63;
	const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
	const int wm = wave / WN, wn = wave % WN;
	const int total = a.steps * a.parts;
	int64_t tt, td;
	int slice;
	Product<D, W, MB, NB, S::stages, false> prod;
	auto &acc = prod.acc;

	if (!tile_of(blockIdx.x, a.tiles_t, a.tiles_d, a.splits, &tt, &td, &slice))
		return;
	const int from = (int)((int64_t)total * slice / a.splits);
	const int to = (int)((int64_t)total * (slice + 1) / a.splits);

	prod.run(a.delta, a.w, tt * TT, td * TD, from, to, a.steps, lds, wm * (MB * 32), wn * (NB * 32), tid, false);
	/* a block at a time: its old values are all on their way before the first store */
#pragma unroll
	for (int i = 0; i < MB; i++)
#pragma unroll
		for (int j = 0; j < NB; j++) {
			const int64_t t = tt * TT + wm * (MB * 32) + i * 32 + block_row(0, lane);
			const int64_t c = td * TD + wn * (NB * 32) + j * 32 + (lane & 31);
			float *p = a.slot + ((int64_t)slice * a.rows_pad + t) * a.d_slot + c;
			float old[16];

			if (a.add) {
#pragma unroll
				for (int r = 0; r < 16; r++)
					old[r] = p[(int64_t)block_row(r, 0) * a.d_slot];
#pragma unroll
				for (int r = 0; r < 16; r++)
					acc[i][j][r] += old[r];
			}
#pragma unroll
			for (int r = 0; r < 16; r++)
				p[(int64_t)block_row(r, 0) * a.d_slot] = acc[i][j][r];
		}
}

struct DxSumArgs {
	const float	*slot;
	int		splits;
	int64_t		rows, rows_pad;
	int		d, d_slot;
	const int32_t	*target;	/* ts */
	float		scale;
	void		*dx;
	int64_t		ld_dx;
};

/* ---- dw and db --------------------------------------------------------------------------------- */

struct DwArgs {
	Source		x;
	Source		delta;
	int		steps, parts;
	int64_t		tiles_d, tiles_v;
	int		d, vocab;
	int64_t		v0;
	void		*dw;		/* [d][vocab] or NULL */
	void		*db;		/* [vocab] or NULL */
	float		scale;
	int		splits;		/* slices of the tokens; more than one: into slots */
	float		*slot;		/* [splits][slot_rows + 1][ld_slot], the last line for db */
	int64_t		slot_rows, ld_slot;
};

/* base[i] += scale x, rounded once */
template <int GT>
__device__ __forceinline__ void add_to(void *base, int64_t i, float x, float scale)
{
	if constexpr (GT == kF32)
		((float *)base)[i] = __builtin_fmaf(scale, x, ((float *)base)[i]);
	else
		((uint16_t *)base)[i] = (uint16_t)bf16_rne(__builtin_fmaf(scale, x, bf16_widen(((uint16_t *)base)[i])));
}

/* The same for the first n of N neighbours: all loads ahead of the stores, which the compiler cannot tell apart. */
template <int GT, int N>
__device__ __forceinline__ void add_some(void *base, int64_t i, int64_t n, const float *x, float scale)
{
	float old[N];

#pragma unroll
	for (int e = 0; e < N; e++) {
		old[e] = 0.0f;
		if (e < n)
			old[e] = GT == kF32 ? ((float *)base)[i + e] : bf16_widen(((uint16_t *)base)[i + e]);
	}
#pragma unroll
	for (int e = 0; e < N; e++)
		if (e < n) {
			if constexpr (GT == kF32)
				((float *)base)[i + e] = __builtin_fmaf(scale, x[e], old[e]);
			else
				((uint16_t *)base)[i + e] = (uint16_t)bf16_rne(__builtin_fmaf(scale, x[e], old[e]));
		}
}

/* Sixteen bytes without their first `halves` 16-bit halves, the others in their place. */
__device__ __forceinline__ u32x4 moved_down(u32x4 w, int halves)
{
	if (halves & 4)
		w = u32x4{w.z, w.w, 0u, 0u};
	if (halves & 2)
		w = u32x4{w.y, w.z, w.w, 0u};
	if (halves & 1)
		w = u32x4{(w.x >> 16) | (w.y << 16), (w.y >> 16) | (w.z << 16), (w.z >> 16) | (w.w << 16), w.w >> 16};
	return w;
}

/*
** SIDE: of the tile both ways.  Small tiles, several workgroups to a compute unit, where the large ones would leave
** the chip idle; the rule (head_plan()) goes by the tiles and not by the tokens, so few tokens of a wide head
** take the large ones, one workgroup to a compute unit, and wait for dw between their few steps.
** 96 tokens, 1536 x 100000 bf16: 175 us for 614 MB of dw in and out, 3.5 TB/s; non-temporal accesses and
** old values read ahead of the products were no faster.  4096 tokens: 610 us for half the
** vocabulary, 1030 TFLOP/s.
*/
template <int SIDE, int GT, bool SLICED>
__global__ __launch_bounds__(SIDE == 256 ? 512 : 256, 2) void head_dw_kernel(DwArgs a)
{
	constexpr int kThreadsHere = SIDE == 256 ? 512 : 256;
	constexpr int WM = 2, WN = kThreadsHere / 64 / WM;
	typedef Operand<true, false, SIDE, kThreadsHere> X;
	typedef Operand<true, false, SIDE, kThreadsHere> D;
	constexpr int MB = SIDE / WM / 32, NB = SIDE / WN / 32;
	__shared__ __align__(16) char lds[2 * (X::kBytes + D::kBytes)];
	const int tid = threadIdx.x;
	const int lane = tid & 63;
	const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
	const int wm = wave / WN, wn = wave % WN;
	int64_t td, tv;
	int slice;
	Product<X, D, MB, NB, 2, true> prod;
	auto &acc = prod.acc;

	if (!tile_of(blockIdx.x, a.tiles_v, a.tiles_d, SLICED ? a.splits : 1, &tv, &td, &slice))
		return;
	/* the column sums: in the tiles of the first rows of x^T, by the wavefronts that hold the upper half */
	const bool sums = a.db != nullptr && td == 0 && wm == 0;

	const int total = a.steps * a.parts;
	const int from = SLICED ? (int)((int64_t)total * slice / a.splits) : 0;
	const int to = SLICED ? (int)((int64_t)total * (slice + 1) / a.splits) : total;

	prod.run(a.x, a.delta, td * SIDE, tv * SIDE, from, to, a.steps, lds, wm * (MB * 32), wn * (NB * 32), tid, sums);
	if constexpr (SLICED) {
		float *slot = a.slot + (int64_t)slice * (a.slot_rows + 1) * a.ld_slot;

#pragma unroll
		for (int j = 0; j < NB; j++) {
			const int64_t c = tv * SIDE + wn * (NB * 32) + j * 32 + (lane & 31);

			if (sums && lane < 32)
				slot[a.slot_rows * a.ld_slot + c] = prod.sum[j][0];
#pragma unroll
			for (int i = 0; i < MB; i++)
#pragma unroll
				for (int r = 0; r < 16; r++)
					slot[(td * SIDE + wm * (MB * 32) + i * 32 + block_row(r, lane)) * a.ld_slot + c] = acc[i][j][r];
		}
		return;
	}
	if (sums && lane < 32) {
#pragma unroll
		for (int j = 0; j < NB; j++) {
			const int64_t v = a.v0 + tv * SIDE + wn * (NB * 32) + j * 32 + lane;

			if (v < a.vocab)
				add_to<GT>(a.db, v, prod.sum[j][0], a.scale);
		}
	}
	if (!a.dw)
		return;
	/*
	** The tile through LDS, half its rows at a time, so that dw is read and written in whole lines (a
	** lane holds one column: two bytes of a line with bf16 gradients, and 96 tokens of the 555M head,
	** where this is most of the work, took 620 us).  A lane's chunks lie below each other; one that the
	** vocabulary ends in is read as the line's last sixteen bytes and moved down.
	*/
	constexpr int kWide = GT == kF32 ? 4 : 8;		/* elements in sixteen bytes */
	constexpr int kHalf = SIDE / 2;
	constexpr int kAcross = SIDE / kWide;			/* chunks to a line */
	constexpr int kApart = kThreadsHere / kAcross;		/* lines between two chunks of a lane */
	constexpr int kChunksOf = kHalf / kApart;		/* of a lane, per half */
	constexpr int kAhead = kChunksOf < 8 ? kChunksOf : 8;	/* of them on their way together */
	static_assert(kThreadsHere % kAcross == 0 && kChunksOf % kAhead == 0, "whole rounds");
	float *const tile = (float *)lds;			/* [kHalf][SIDE] */
	const int64_t v = a.v0 + tv * SIDE + tid % kAcross * kWide;
	const int64_t left = a.vocab - v;			/* elements from the lane's first on */
	const bool near = a.vocab >= kWide;			/* a line has sixteen bytes */
	const int beyond = left >= kWide ? 0 : left > 0 ? kWide - (int)left : kWide;
	char *const first = (char *)a.dw + (v - beyond) * (16 / kWide);

	auto line_of = [&](int h, int u) {
		const int row = tid / kAcross + u * kApart;

		return td * SIDE + (row / (kHalf / 2)) * kHalf + h * (kHalf / 2) + row % (kHalf / 2);
	};
	auto fetch = [&](int h, int u0, u32x4 (&old)[kAhead]) {
#pragma unroll
		for (int u = 0; u < kAhead; u++) {
			const int64_t k = line_of(h, u0 + u);

			if (k < a.d && beyond < kWide && near)
				old[u] = *(const u32x4_any *)(first + k * a.vocab * (16 / kWide));
		}
	};
	auto put = [&](int h, int u0, const u32x4 (&old)[kAhead]) {
#pragma unroll
		for (int u = 0; u < kAhead; u++) {
			const int64_t k = line_of(h, u0 + u);
			const float *x = tile + (tid / kAcross + (u0 + u) * kApart) * SIDE + tid % kAcross * kWide;
			u32x4 w = old[u];

			if (k >= a.d || beyond == kWide)
				continue;
			if (!near) {
				add_some<GT, kWide>(a.dw, k * a.vocab + v, left, x, a.scale);
				continue;
			}
			if (beyond)
				w = moved_down(w, beyond * (8 / kWide));
			if constexpr (GT == kF32) {
#pragma unroll
				for (int e = 0; e < 4; e++)
					w[e] = __float_as_uint(__builtin_fmaf(a.scale, x[e], __uint_as_float(w[e])));
			} else {
#pragma unroll
				for (int e = 0; e < 4; e++)
					w[e] = bf16_rne2(__builtin_fmaf(a.scale, x[2 * e], __uint_as_float(w[e] << 16)),
					    __builtin_fmaf(a.scale, x[2 * e + 1], __uint_as_float(w[e] & 0xffff0000u)));
			}
			if (beyond == 0) {
				*(u32x4_any *)(first + k * a.vocab * (16 / kWide)) = w;
				continue;
			}
#pragma unroll
			for (int e = 0; e < kWide; e++)
				if (e < left) {
					if constexpr (GT == kF32)
						((uint32_t *)a.dw)[k * a.vocab + v + e] = w[e];
					else
						((uint16_t *)a.dw)[k * a.vocab + v + e] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
				}
		}
	};
	u32x4 old[2][kAhead];

	/* where a half is one round, the second half's old values come with the first's */
	if constexpr (kChunksOf == kAhead) {
		fetch(0, 0, old[0]);
		fetch(1, 0, old[1]);
	}
#pragma unroll
	for (int h = 0; h < 2; h++) {
		if (h)
			__syncthreads();
#pragma unroll
		for (int i = 0; i < MB / 2; i++)
#pragma unroll
			for (int j = 0; j < NB; j++)
#pragma unroll
				for (int r = 0; r < 16; r++)
					tile[(wm * (kHalf / 2) + i * 32 + block_row(r, lane)) * SIDE + wn * (NB * 32) + j * 32
					    + (lane & 31)] = acc[h * (MB / 2) + i][j][r];
		__syncthreads();
		if constexpr (kChunksOf == kAhead) {
			put(h, 0, old[h]);
		} else {
#pragma unroll 1
			for (int u0 = 0; u0 < kChunksOf; u0 += kAhead) {
				fetch(h, u0, old[0]);
				put(h, u0, old[0]);
			}
		}
	}
}

struct DwSumArgs {
	const float	*slot;		/* [splits][slot_rows + 1][ld_slot] */
	int		splits;
	int64_t		slot_rows, ld_slot;
	int		d, vocab;
	int64_t		v0, count;	/* places of this piece */
	float		scale;
	void		*dw;
	void		*db;
};

/*
** dx = scale times the slots' sum in order, in the caller's type.  A row without a target has delta 0, but its
** product with a w that is not finite is NaN: it gets its 0 here (the target and the slots are loaded together; one
** behind the other 1 us more).
*/
template <int GT>
__device__ __forceinline__ void dx_sum(const DxSumArgs &a, int64_t block, int64_t blocks)
{
	const int64_t per = a.d_slot / 4;
	const int64_t n = a.rows * per;

	for (int64_t q = block * kThreads + threadIdx.x; q < n; q += blocks * kThreads) {
		const int64_t r = q / per;
		const int c = (int)(q - r * per) * 4;
		f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};

		if (c >= a.d)
			continue;
		const bool live = a.target[r] >= 0;

#pragma unroll 8
		for (int k = 0; k < a.splits; k++)
			s += *(const f32x4 *)(a.slot + ((int64_t)k * a.rows_pad + r) * a.d_slot + c);
		s = live ? s * a.scale : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
		for (int j = 0; j < 4; j++)
			if (c + j < a.d) {
				if constexpr (GT == kF32)
					((float *)a.dx)[r * a.ld_dx + c + j] = s[j];
				else
					((uint16_t *)a.dx)[r * a.ld_dx + c + j] = (uint16_t)bf16_rne(s[j]);
			}
	}
}

/* dw and db += scale times the slots' sums in order: a line of dw (or db, the last) to a row of `across` workgroups. */
template <int GT>
__device__ __forceinline__ void dw_sum(const DwSumArgs &a, int64_t block, int64_t blocks)
{
	const int64_t across = (a.count + kThreads - 1) / kThreads;
	const int64_t c = block % across * kThreads + threadIdx.x;

	if (c >= a.count)
		return;
	for (int64_t r = block / across; r <= a.d; r += blocks / across) {
		const bool last = r == a.d;
		const float *p = a.slot + (last ? a.slot_rows : r) * a.ld_slot + c;
		float s = 0.0f;

		if (last ? !a.db : !a.dw)
			continue;
#pragma unroll 8
		for (int k = 0; k < a.splits; k++)
			s += p[(int64_t)k * (a.slot_rows + 1) * a.ld_slot];
		add_to<GT>(last ? a.db : a.dw, last ? a.v0 + c : r * a.vocab + a.v0 + c, s, a.scale);
	}
}

/* Both in one launch: the first blocks_x workgroups are dx's, the others (a multiple of dw_sum's `across`) dw's. */
template <int GT>
__global__ __launch_bounds__(kThreads) void head_sums_kernel(DxSumArgs x, unsigned blocks_x, DwSumArgs w)
{
	if (blockIdx.x < blocks_x)
		dx_sum<GT>(x, blockIdx.x, blocks_x);
	else
		dw_sum<GT>(w, blockIdx.x - blocks_x, gridDim.x - blocks_x);
}

/* ---- launches ---------------------------------------------------------------------------------- */

static int rows_grid(int64_t items)
{
	const int64_t g = (items + kThreads - 1) / kThreads;

	return (int)(g > 8192 ? 8192 : g < 1 ? 1 : g);
}

template <class S, int MODE>
static void logits_go(hipStream_t st, const LogitArgs &a)
{
	hipLaunchKernelGGL((head_logits_kernel<S, MODE>), dim3((unsigned)up((size_t)(a.tiles_v * a.tiles_t), 8)),
	    dim3(S::threads), 0, st, a);
}

template <int MODE>
static void logits_launch(hipStream_t st, const HeadPlan &p, const LogitArgs &a)
{
	if constexpr (MODE == kStats || MODE == kStatsKeep)
		if (p.tile_t == 64) {
			logits_go<LogitsFew, MODE>(st, a);
			return;
		}
	/* (the small tiles' logits are few enough to be kept: delta is never formed from them anew) */
	if (p.tile_t == 128)
		logits_go<LogitsSome, MODE>(st, a);
	else
		logits_go<LogitsMany, MODE>(st, a);
}

/* The same from the logits that were kept, for `here` places (a multiple of kSide) of the piece. */
static void delta_launch(hipStream_t st, const HeadPlan &p, const LogitArgs &l, const FinishArgs &f, int few, int64_t here,
	int vocab)
{
	DeltaArgs a;

	memset(&a, 0, sizeof(a));
	a.finish = f;
	a.few = few;
	a.kept = l.kept;
	a.kept_v = l.kept_v;
	a.target = l.target;
	a.lse = l.lse;
	a.vocab = vocab;
	a.v0 = l.v0;
	a.groups_v = here / 128;
	a.delta = l.delta;
	a.delta_low = l.delta_low;
	a.ld_delta = l.ld_delta;
	const dim3 grid((unsigned)(p.rows_pad / 32 * a.groups_v));

	if (p.parts == 2)
		hipLaunchKernelGGL(head_delta_kernel<true>, grid, dim3(kThreads), 0, st, a);
	else
		hipLaunchKernelGGL(head_delta_kernel<false>, grid, dim3(kThreads), 0, st, a);
}

template <class S>
static void dx_go(hipStream_t st, const DxArgs &a)
{
	hipLaunchKernelGGL(head_dx_kernel<S>, dim3((unsigned)up((size_t)(a.tiles_t * a.tiles_d * a.splits), 8)),
	    dim3(S::threads), 0, st, a);
}

static void dx_launch(hipStream_t st, const HeadPlan &p, const DxArgs &a)
{
	if (p.dx == kDxFew)
		dx_go<DxFew>(st, a);
	else if (p.dx == kDxSome)
		dx_go<DxSome>(st, a);
	else
		dx_go<DxMany>(st, a);
}

template <int GT>
static void dw_launch(hipStream_t st, const HeadPlan &p, const DwArgs &a)
{
	const dim3 grid((unsigned)up((size_t)(a.tiles_d * a.tiles_v * a.splits), 8));

	if (a.splits > 1)
		hipLaunchKernelGGL((head_dw_kernel<128, GT, true>), grid, dim3(256), 0, st, a);
	else if (p.side_w == 128)
		hipLaunchKernelGGL((head_dw_kernel<128, GT, false>), grid, dim3(256), 0, st, a);
	else
		hipLaunchKernelGGL((head_dw_kernel<256, GT, false>), grid, dim3(512), 0, st, a);
}

/* x and w: may be NULL */
static void sums_launch(hipStream_t st, int grad_type, const DxSumArgs *x, const DwSumArgs *w)
{
	DxSumArgs ax;
	DwSumArgs aw;
	unsigned blocks_x = 0, blocks_w = 0;

	memset(&ax, 0, sizeof(ax));
	memset(&aw, 0, sizeof(aw));
	if (x) {
		ax = *x;
		blocks_x = (unsigned)rows_grid(x->rows * (x->d_slot / 4));
	}
	if (w) {
		aw = *w;
		blocks_w = (unsigned)(count(w->count, kThreads) * (w->d + 1 < 1024 ? w->d + 1 : 1024));
	}
	if (grad_type == ANNI_F32)
		hipLaunchKernelGGL(head_sums_kernel<kF32>, dim3(blocks_x + blocks_w), dim3(kThreads), 0, st, ax, blocks_x, aw);
	else
		hipLaunchKernelGGL(head_sums_kernel<kBF16>, dim3(blocks_x + blocks_w), dim3(kThreads), 0, st, ax, blocks_x, aw);
}

static int head_run(const anni_head_job &j, const HeadPlan &p, bool grad)
{
	const bool keep = grad && p.keeps && j.work_bytes >= p.bytes_keep;
	hipStream_t st = compute_stream();
	char *work = (char *)j.d_work;
	uint16_t *xs = (uint16_t *)(work + p.off_xs);
	int32_t *ts = (int32_t *)(work + p.off_ts);
	float *lse = (float *)(work + p.off_lse);
	const uint16_t *w = (const uint16_t *)j.d_w;
	RowArgs ra;
	LogitArgs la;
	FinishArgs fa;

	memset(&ra, 0, sizeof(ra));
	ra.x = (const uint16_t *)j.d_x;
	ra.ld_x = j.ld_x;
	ra.target = j.d_target;
	ra.rows = j.rows;
	ra.rows_pad = p.rows_pad;
	ra.d = j.d;
	ra.d_pad = p.d_pad;
	ra.vocab = j.vocab;
	ra.vocab_pad = p.vocab_pad;
	ra.bias = j.d_bias;
	ra.xs = xs;
	ra.ld_xs = p.ld_xs;
	ra.ts = ts;
	ra.bs = (float *)(work + p.off_bs);
	if (p.align) {
		ra.w = w;
		ra.ws = (uint16_t *)(work + p.off_ws);
		ra.ld_ws = p.ld_ws;
		w = ra.ws;
	}
	const int64_t chunks = p.rows_pad * (p.d_pad / 8), chunks_w = p.align ? j.d * (p.vocab_pad / 8) : 0;

	hipLaunchKernelGGL(head_rows_kernel, dim3(rows_grid(chunks > chunks_w ? chunks : chunks_w)), dim3(kThreads), 0, st, ra);

	memset(&la, 0, sizeof(la));
	la.w.part[0] = la.w.part[1] = w;
	la.w.ld = (uint32_t)(p.align ? p.ld_ws : j.vocab);
	la.w.rows = p.align ? p.vocab_pad : j.vocab;
	la.w.depth = j.d;
	la.w.aligned = p.align || (((uintptr_t)w & 15) == 0 && j.vocab % 8 == 0);
	la.x.part[0] = la.x.part[1] = xs;
	la.x.ld = (uint32_t)p.ld_xs;
	la.x.rows = p.rows_pad;
	la.x.depth = p.d_pad;
	la.bias = ra.bs;
	la.target = ts;
	la.steps = (j.d + kStep - 1) / kStep;
	la.tiles_v = p.tiles_v;
	la.tiles_t = p.rows_pad / p.tile_t;
	la.rows_pad = p.rows_pad;
	la.part = (f32x2 *)(work + p.off_part);
	la.target_logit = (float *)(work + p.off_hit);
	la.kept = (f32x4 *)(work + p.off_kept);
	la.kept_v = p.vocab_pad / 32;
	if (keep)
		logits_launch<kStatsKeep>(st, p, la);
	else
		logits_launch<kStats>(st, p, la);

	memset(&fa, 0, sizeof(fa));
	fa.part = la.part;
	fa.target_logit = la.target_logit;
	fa.target = ts;
	fa.tiles_v = p.tiles_v;
	fa.rows = j.rows;
	fa.rows_pad = p.rows_pad;
	fa.lse = lse;
	fa.nll = j.d_nll;
	/* nothing but the pass over the kept logits asks for them: it folds them itself */
	const int few = keep && p.tiles_v <= kFewTiles ? (int)p.tiles_v : 0;

	if (!few)
		hipLaunchKernelGGL(head_finish_kernel, dim3((unsigned)(p.rows_pad / kFinishTokens)),
		    dim3(p.tiles_v <= kFewTiles ? 64u : p.tiles_v < 4 * kFinishWaves ? (unsigned)up((size_t)p.tiles_v, 4) * 16
		    : kFinishWaves * 64), 0, st, fa);

	for (int64_t v0 = 0; grad && v0 < j.vocab; v0 += p.piece) {
		const int64_t left = j.vocab - v0;
		const int64_t here = left < p.piece ? (int64_t)up((size_t)left, kSide) : p.piece;
		uint16_t *delta = (uint16_t *)(work + p.off_delta);
		uint16_t *low = delta + p.rows_pad * p.ld_delta;
		DxArgs xa;
		DwArgs wa;
		DxSumArgs sx;
		DwSumArgs sw;

		la.v0 = v0;
		la.tiles_v = here / p.tile_v;
		la.lse = lse;
		la.delta = delta;
		la.delta_low = low;
		la.ld_delta = p.ld_delta;
		if (keep)
			delta_launch(st, p, la, fa, few, here, j.vocab);
		else if (p.parts == 2)
			logits_launch<kDeltaPair>(st, p, la);
		else
			logits_launch<kDelta>(st, p, la);

		memset(&wa, 0, sizeof(wa));
		wa.x = la.x;
		wa.x.rows = p.d_pad;
		wa.x.depth = p.rows_pad;
		wa.delta.part[0] = delta;
		wa.delta.part[1] = low;
		wa.delta.ld = (uint32_t)p.ld_delta;
		wa.delta.rows = here;
		wa.delta.depth = p.rows_pad;
		wa.steps = (int)(p.rows_pad / kStep);
		wa.parts = p.parts;
		wa.tiles_d = count(j.d, p.side_w);
		wa.tiles_v = here / p.side_w;
		wa.d = j.d;
		wa.vocab = j.vocab;
		wa.v0 = v0;
		wa.dw = j.d_dw;
		wa.db = j.d_db;
		wa.scale = (float)j.scale;
		wa.splits = p.splits_w;
		wa.slot = (float *)(work + p.off_slot_w);
		wa.slot_rows = p.slot_rows_w;
		wa.ld_slot = p.piece;
		if (!j.d_dw)
			wa.tiles_d = 1;			/* only the tiles that sum */
		if (j.d_dw || j.d_db) {
			if (j.grad_type == ANNI_F32)
				dw_launch<kF32>(st, p, wa);
			else
				dw_launch<kBF16>(st, p, wa);
		}
		if (j.d_dx) {
			memset(&xa, 0, sizeof(xa));
			xa.delta = wa.delta;
			xa.delta.rows = p.rows_pad;
			xa.delta.depth = here;
			xa.w.part[0] = xa.w.part[1] = w + v0;
			xa.w.ld = la.w.ld;
			xa.w.rows = j.d;
			xa.w.depth = p.align ? here : left;
			xa.w.aligned = la.w.aligned;	/* v0 is a multiple of kSide */
			xa.steps = (int)((left < here ? left : here) + kStep - 1) / kStep;
			xa.parts = p.parts;
			xa.splits = p.splits;
			xa.tiles_t = p.rows_pad / p.dx_t;
			xa.tiles_d = count(j.d, p.tile_d);	/* every tile has a valid row of w */
			xa.slot = (float *)(work + p.off_slot);
			xa.rows_pad = p.rows_pad;
			xa.d_slot = p.d_slot;
			xa.add = v0 > 0;
			dx_launch(st, p, xa);
		}
		/* the slices' sums: dw's behind every piece, dx's behind the last one */
		const bool sum_w = wa.splits > 1 && (j.d_dw || j.d_db);
		const bool sum_x = j.d_dx && left <= p.piece;

		if (sum_w) {
			memset(&sw, 0, sizeof(sw));
			sw.slot = wa.slot;
			sw.splits = wa.splits;
			sw.slot_rows = wa.slot_rows;
			sw.ld_slot = wa.ld_slot;
			sw.d = j.d;
			sw.vocab = j.vocab;
			sw.v0 = v0;
			sw.scale = wa.scale;
			sw.count = left < p.piece ? left : p.piece;
			sw.dw = j.d_dw;
			sw.db = j.d_db;
		}
		if (sum_x) {
			memset(&sx, 0, sizeof(sx));
			sx.slot = xa.slot;
			sx.splits = p.splits;
			sx.rows = j.rows;
			sx.rows_pad = p.rows_pad;
			sx.d = j.d;
			sx.d_slot = p.d_slot;
			sx.target = ts;
			sx.scale = wa.scale;
			sx.dx = j.d_dx;
			sx.ld_dx = j.ld_dx;
		}
		if (sum_w || sum_x)
			sums_launch(st, j.grad_type, sum_x ? &sx : nullptr, sum_w ? &sw : nullptr);
	}
	return hip_ok(hipGetLastError(), "head_loss") ? 0 : -1;
}

} /* namespace anni */

using namespace anni;

extern "C" {

size_t anni_head_loss_work_bytes(int64_t rows, int d, int vocab, int grad_type)
{
	HeadPlan p;

	return head_plan(rows, d, vocab, grad_type, &p) ? p.bytes : 0;
}

size_t anni_head_loss_work_bytes_keep(int64_t rows, int d, int vocab, int grad_type)
{
	HeadPlan p;

	return head_plan(rows, d, vocab, grad_type, &p) ? p.bytes_keep : 0;
}

int anni_head_loss(const anni_head_job *job)
{
	HeadPlan p;
	bool grad;

	if (!head_job_plan(job, &p, &grad) || !device_ready())
		return -1;
	return head_run(*job, p, grad);
}

} /* extern "C" */
