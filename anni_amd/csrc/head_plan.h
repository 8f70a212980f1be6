/*
** How a call of the head's loss is laid out, and which calls are refused: the shapes of the tiles,
** the rules that choose between them, the work area's parts, the checks of a job.  No device call in
** here, so it can be exercised on the host.
*/
#ifndef ANNI_HEAD_PLAN_H__
#define ANNI_HEAD_PLAN_H__

#include <stdint.h>
#include <string.h>
#include "anni_adam.h"

namespace anni {

constexpr int kStep = 64;		/* of the contracted axis per trip */
constexpr int kSide = 256;		/* of a result tile along the vocabulary or the model's width */

/* A tile of SIDE places (or columns of the model's width) and TOKENS tokens to a workgroup. */
template <int SIDE_, int TOKENS_, int WAVES_, int WAVES_SIDE_, int STAGES_> struct Shape {
	static constexpr int side = SIDE_;
	static constexpr int tokens = TOKENS_;
	static constexpr int waves = WAVES_;
	static constexpr int threads = WAVES_ * 64;
	static constexpr int waves_side = WAVES_SIDE_;		/* wavefronts along the side */
	static constexpr int waves_tokens = WAVES_ / WAVES_SIDE_;
	static constexpr int stages = STAGES_;
};

/*
** Tiles of vocabulary by tokens (the logits), of the model's width by tokens (dx).
** Many: two stages of the largest tile that fits, one workgroup to a compute unit.  Some: a quarter of
** it, two workgroups to a compute unit, where the large tiles would not fill the chip or w is read
** more than it is computed with (few rows).  Few: a quarter again, where even those are too few.
** head_plan() has the rule and what it goes by.
*/
typedef Shape<64, 64, 4, 2, 4> LogitsFew;
typedef Shape<128, 128, 8, 4, 2> LogitsSome;
typedef Shape<256, 256, 8, 2, 2> LogitsMany;
typedef Shape<128, 64, 4, 2, 3> DxFew;
typedef Shape<128, 128, 8, 4, 2> DxSome;
typedef Shape<256, 256, 8, 4, 2> DxMany;

/*
** The work area's matrices have lines of an odd number of 256 bytes.  Lines of a power of two put a
** tile's column of lines into one of the sixteen channels of the level-two cache.
*/
constexpr int kOdd = 128;
static_assert((kSide + kOdd) * 2 % 512 == 256, "lines of whole tiles, then 256 bytes");

enum { kDxFew, kDxSome, kDxMany };

struct HeadPlan {
	int	tile_t;		/* tokens per tile: 64 few, 128 some, 256 many */
	bool	small;		/* not many */
	int	tile_v;		/* the other side of the logits' tiles */
	int	dx;		/* kDxFew .. kDxMany */
	int	dx_t, tile_d;	/* its tiles */
	int	d_slot;		/* columns of a slot: whole tiles */
	int64_t	rows_pad;
	int	d_pad;
	int64_t	vocab_pad;
	int64_t	tiles_v;	/* of the logits, over the whole vocabulary */
	int64_t	piece;		/* vocabulary places per piece of delta, a multiple of kSide */
	int64_t	ld_xs, ld_delta;
	int	parts;		/* bf16 numbers per element of delta */
	int	splits;		/* slices of the vocabulary in dx */
	int	side_w;		/* of dw's tiles */
	int	splits_w;	/* slices of the tokens in dw */
	int64_t	slot_rows_w;
	bool	align;		/* w is copied to lines that are aligned */
	int64_t	ld_ws;
	size_t	off_ws, off_xs, off_ts, off_bs, off_part, off_hit, off_lse, off_delta, off_kept, off_slot, off_slot_w;
	bool	keeps;		/* the logits, if there is room */
	size_t	bytes;		/* the least work area */
	size_t	bytes_keep;	/* one that holds the logits between the passes */
};

static inline size_t up(size_t x, size_t a)
{
	return (x + a - 1) / a * a;
}

static inline int64_t count(int64_t n, int64_t tile)
{
	return (n + tile - 1) / tile;
}

static const int kUnits = 256;		/* compute units of an MI355X, a workgroup of a large tile each */
static const int64_t kHeadMaxRows = (int64_t)1 << 22;
static const int kHeadMaxD = 1 << 16;
static const int kHeadMaxVocab = 1 << 22;
static const int64_t kHeadMaxLogits = (int64_t)1 << 38;	/* 2^22 large tiles: what one launch may have */

/* grad_type: -1 = the loss alone. */
static inline bool head_plan(int64_t rows, int d, int vocab, int grad_type, HeadPlan *p)
{
	const size_t delta_most = (size_t)512 << 20;
	const size_t kept_least = (size_t)512 << 20;	/* logits that are kept in any case: no more than a piece of delta */
	size_t at = 0;
	int64_t large, middle;

	if (rows <= 0 || rows > kHeadMaxRows || d <= 0 || d > kHeadMaxD || vocab <= 0 || vocab > kHeadMaxVocab
	    || rows * vocab > kHeadMaxLogits
	    || (grad_type != -1 && grad_type != ANNI_F32 && grad_type != ANNI_BF16))
		return false;
	memset(p, 0, sizeof(*p));
	/*
	** A turn of large tiles, one to each compute unit, takes ten; the middle ones six for the first two
	** to each compute unit, and proportionally more beyond that.  Scoring, middle against large, in us:
	** 777 x 331 x 10007 28.8 / 38.7, 512 x 1024 x 16384 30 / 38, 1024 x 1024 x 16384 50 / 43,
	** 2048 x 1024 x 16384 86 / 76.  Small against middle: 512 x 512 x 4096 14.6 / 16.5,
	** 64 x 1536 x 50000 69 / 63.
	*/
	large = count(rows, 256) * count(vocab, 256);
	middle = count(rows, 128) * count(vocab, 128);
	if (count(large, kUnits) * 10 * 2 * kUnits <= (middle > 2 * kUnits ? middle : 2 * kUnits) * 6)
		p->tile_t = 256;
	else
		p->tile_t = middle < kUnits ? 64 : 128;
	p->small = p->tile_t != 256;
	p->tile_v = !p->small ? kSide : p->tile_t == 64 ? LogitsFew::side : LogitsSome::side;
	/*
	** dx: small tiles with the small ones of the logits, middle ones with the middle ones, and also where
	** the large ones would mostly cover what is not there: the middle ones take a third longer for the
	** same area (us, large against middle: 4096 x 331 x 16384 f32 167 / 174, 2314 x 64 x 69760 bf16 140 / 90).
	*/
	p->dx = p->tile_t == 64 ? kDxFew : p->small
	    || count(rows, 128) * count(d, 128) * 10 < count(rows, 256) * count(d, 256) * 28 ? kDxSome : kDxMany;
	p->dx_t = p->dx == kDxFew ? DxFew::tokens : p->dx == kDxMany ? DxMany::tokens : DxSome::tokens;
	p->tile_d = p->dx == kDxFew ? DxFew::side : p->dx == kDxMany ? DxMany::side : DxSome::side;
	p->rows_pad = (int64_t)up((size_t)rows, (size_t)p->tile_t);
	p->d_pad = (int)up((size_t)d, kSide);
	p->d_slot = (int)up((size_t)d, (size_t)p->tile_d);
	p->vocab_pad = (int64_t)up((size_t)vocab, kSide);
	p->tiles_v = count(vocab, p->tile_v);
	p->parts = grad_type == ANNI_F32 ? 2 : 1;
	p->ld_xs = p->d_pad + kOdd;
	/*
	** Lines that are not aligned go through registers, one step ahead.  That costs a step of the first turn
	** of tiles about 1.3 us and of a later one .45; a copy of w with aligned lines costs 3 us and .75
	** for each million of its elements.  Copied where it pays with a third to spare (scoring, us without / with:
	** 397 x 759 x 1455 32.6 / 20.4, 3000 x 1290 x 4882 96 / 62, 4096 x 712 x 50257 421 / 379, and against it 256 x
	** 712 x 50257 55 / 65, 500 x 128 x 1001 13 / 17).
	*/
	{
		const int64_t tiles = p->rows_pad / p->tile_t * p->tiles_v;
		const int64_t turns = count(tiles, p->small ? 2 * kUnits : kUnits);

		p->align = vocab % 8 != 0
		    && (double)count(d, kStep) * (1.3 + 0.45 * (double)(turns - 1)) > 1.3 * (3.0 + 0.75e-6 * d * vocab);
	}
	p->ld_ws = p->vocab_pad + kOdd;
	p->off_ws = at;
	if (p->align)
		at = up(at + (size_t)d * p->ld_ws * 2, 256);
	p->off_xs = at;
	at = up(at + (size_t)p->rows_pad * p->ld_xs * 2, 256);
	p->off_ts = at;
	at = up(at + (size_t)p->rows_pad * 4, 256);
	p->off_bs = at;
	at = up(at + (size_t)p->vocab_pad * 4, 256);
	p->off_part = at;
	at = up(at + (size_t)p->tiles_v * p->rows_pad * 8, 256);
	p->off_hit = at;
	at = up(at + (size_t)p->rows_pad * 4, 256);
	p->off_lse = at;
	at = up(at + (size_t)p->rows_pad * 4, 256);
	if (grad_type != -1) {
		const int64_t whole = p->vocab_pad;
		const int64_t fit = (int64_t)(delta_most / ((size_t)p->rows_pad * 2 * p->parts)) / kSide * kSide;
		const int64_t tiles = p->rows_pad / p->dx_t * count(d, p->tile_d);
		int64_t steps;

		const int64_t pieces = fit < kSide ? whole / kSide : (whole + fit - 1) / fit;

		/* pieces of about the same size: the last one would leave compute units idle */
		p->piece = (int64_t)up((size_t)((whole + pieces - 1) / pieces), kSide);
		p->ld_delta = p->piece + kOdd;
		steps = p->piece / kStep * p->parts;
		/*
		** Slices of the vocabulary in dx, each with a float slot for the whole of dx: the fewest that fill
		** nine tenths of the compute units' turns, of at least sixteen steps each, or of two while the slots
		** take no more than 8 MiB, which no one has to fetch from far (us, sixteen against two:
		** 254 x 64 x 256 9.7 / 4.8, 100 x 256 x 2001 18 / 7, 700 x 300 x 2000 17.5 / 11.3).
		*/
		const size_t near_slots = (size_t)8 << 20;
		const size_t slot = (size_t)p->rows_pad * (size_t)p->d_slot * 4;
		const int64_t units = p->dx == kDxMany ? kUnits : 2 * kUnits;	/* few tokens are bound by memory: more on its way */

		p->splits = 1;
		for (int k = 1; k <= 256 && (k * 16 <= steps || (k * 2 <= steps && (size_t)k * slot <= near_slots)); k++) {
			const int64_t groups = tiles * k;
			const int64_t turns = (groups + units - 1) / units;

			p->splits = k;
			if (groups * 10 >= turns * units * 9)
				break;
		}
		/*
		** dw: tiles of 128 by two to a compute unit take about seven tenths of the time of a turn of the
		** large ones (measured where either fills the chip), a quarter of the work each.
		*/
		{
			const int64_t large = count(d, 256) * count(p->piece, 256);
			const int64_t little = count(d, 128) * count(p->piece, 128);

			p->side_w = count(little, 2 * kUnits) * 7 < count(large, kUnits) * 10 ? 128 : 256;
			/*
			** Slices of the tokens while half the chip idles: of at least eight steps, or two while the slots
			** are near as well (us, dw with its sum: 254 x 64 x 256 10.8 / 9.0, 500 x 128 x 1000 14.6 / 10.1,
			** 900 x 100 x 1500 19.9 / 12).
			*/
			const size_t slot_w = (size_t)(count(d, 128) * 128 + 1) * (size_t)p->piece * 4;
			const int64_t steps_w = p->rows_pad / kStep * p->parts;

			p->splits_w = 1;
			while (little * p->splits_w * 2 <= kUnits && p->splits_w < 64 && (steps_w >= 16 * p->splits_w
			    || (steps_w >= 4 * p->splits_w && 2 * (size_t)p->splits_w * slot_w <= near_slots)))
				p->splits_w *= 2;
			if (p->splits_w > 1)
				p->side_w = 128;
			p->slot_rows_w = count(d, 128) * 128;
		}
		p->off_delta = at;
		at = up(at + (size_t)p->rows_pad * p->ld_delta * 2 * p->parts, 256);
		p->off_slot = at;
		at = up(at + (size_t)p->splits * p->rows_pad * p->d_slot * 4, 256);
		p->off_slot_w = at;
		if (p->splits_w > 1)
			at = up(at + (size_t)p->splits_w * (p->slot_rows_w + 1) * p->piece * 4, 256);
	}
	p->bytes = p->bytes_keep = at;
	if (grad_type != -1) {
		const size_t kept = (size_t)p->rows_pad * (size_t)p->vocab_pad * 4;

		/*
		** Keeping them writes and reads 8 bytes for each, computing them again takes 2 d operations.  us of
		** the two passes, kept / again: 2048 x 128 x 32768 155 / 132, 2048 x 256 x 32768 175 / 188,
		** 161 x 64 x 50304 34 / 28, 200 x 256 x 50304 33 / 38.  (The small tiles' are always kept: few.)
		*/
		if (d >= 192 || p->tile_t == 64) {
			p->off_kept = at;
			p->bytes_keep = at + kept;
			p->keeps = true;
			if (kept <= kept_least)
				p->bytes = p->bytes_keep;
		}
	}
	return true;
}

/*
** What anni_head_loss takes: a plan, and whether there are gradients to write.  Everything it refuses is
** refused here, before any device is looked for.  grad_type -1 is a question to the size functions; a job
** with gradients names a type of theirs (the plan of a loss alone has no part for them).
*/
static inline bool head_job_plan(const anni_head_job *job, HeadPlan *p, bool *grad)
{
	uintptr_t grad_mask;

	if (!job || !job->d_x || !job->d_w || !job->d_target || !job->d_nll || !job->d_work)
		return false;
	*grad = job->d_dx || job->d_dw || job->d_db;
	if (*grad && job->grad_type != ANNI_F32 && job->grad_type != ANNI_BF16)
		return false;
	if (!head_plan(job->rows, job->d, job->vocab, *grad ? job->grad_type : -1, p) || job->ld_x < job->d
	    || (job->d_dx && job->ld_dx < job->d) || job->work_bytes < p->bytes)
		return false;
	/* an element starts where its type may; the work area is ours to lay out */
	grad_mask = *grad && job->grad_type == ANNI_F32 ? 3 : 1;
	return (((uintptr_t)job->d_x | (uintptr_t)job->d_w) & 1) == 0
	    && (((uintptr_t)job->d_bias | (uintptr_t)job->d_target | (uintptr_t)job->d_nll) & 3) == 0
	    && (((uintptr_t)job->d_dx | (uintptr_t)job->d_dw | (uintptr_t)job->d_db) & grad_mask) == 0
	    && ((uintptr_t)job->d_work & 255) == 0;
}

} /* namespace anni */
#endif
