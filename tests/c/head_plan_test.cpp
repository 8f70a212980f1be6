// Host-only test of anni_amd/csrc/head_plan.h.  Without arguments: which jobs of the head's loss are
// refused and which are taken (the addresses are invented, nothing follows them), and what every plan
// has to hold for the launches made from it.  With "rows d vocab type" groups: the plans' shapes, a line each.
#include <cstdio>
#include <cstdlib>
#include <initializer_list>
#include "head_plan.h"

using namespace anni;

static int fails, refused, taken, plans;

#define CHECK(x) do { if (!(x)) { fails++; printf("line %d: %s\n", __LINE__, #x); } } while (0)

static const uintptr_t kAt = 4096;

static anni_head_job job_of(int grad_type)
{
	HeadPlan p;
	anni_head_job j;

	memset(&j, 0, sizeof(j));
	j.rows = 8;
	j.d = 16;
	j.vocab = 32;
	j.ld_x = 16;
	j.ld_dx = 16;
	j.d_x = j.d_w = j.d_work = (void *)kAt;
	j.d_target = (const int32_t *)kAt;
	j.d_nll = (float *)kAt;
	j.scale = 1.0;
	j.grad_type = grad_type;
	CHECK(head_plan(8, 16, 32, grad_type, &p));
	j.work_bytes = p.bytes;
	return j;
}

static void expect(bool want, const anni_head_job &j, int line)
{
	HeadPlan p;
	bool grad = false;
	const bool got = head_job_plan(&j, &p, &grad);

	(want ? taken : refused)++;
	if (got != want) {
		fails++;
		printf("line %d: %s\n", line, got ? "taken" : "refused");
	}
	/* what the launches of a job with gradients divide by and count with */
	if (got && grad && (p.piece <= 0 || p.side_w <= 0 || p.splits <= 0 || p.splits_w <= 0 || p.ld_delta <= 0)) {
		fails++;
		printf("line %d: taken with gradients and a plan that has none\n", line);
	}
}

#define TAKES(type, ...) do { anni_head_job j = job_of(type); __VA_ARGS__; expect(true, j, __LINE__); } while (0)
#define REFUSES(type, ...) do { anni_head_job j = job_of(type); __VA_ARGS__; expect(false, j, __LINE__); } while (0)

static void jobs(void)
{
	void *const at = (void *)kAt;

	/* the loss alone: the type is not looked at */
	TAKES(-1, );
	TAKES(-1, j.grad_type = ANNI_F32);
	TAKES(-1, j.grad_type = ANNI_FP8_E4M3);
	TAKES(-1, j.grad_type = 77; j.ld_dx = 0);
	for (int ty = ANNI_F32; ty <= ANNI_BF16; ty++) {
		TAKES(ty, );
		TAKES(ty, j.d_dx = at);
		TAKES(ty, j.d_dw = at);
		TAKES(ty, j.d_db = at);
		TAKES(ty, j.d_dx = j.d_dw = j.d_db = at; j.d_bias = (const float *)kAt; j.ld_x = j.ld_dx = 83);
		TAKES(ty, j.d_dw = at; j.work_bytes += 1000; j.ld_dx = 0);
		/* a type that no gradient has, with the loss alone's work area and with all of it */
		for (int bad : { -1, -2, ANNI_FP8_E4M3, ANNI_Q8, 4, INT32_MIN, INT32_MAX }) {
			REFUSES(ty, j.d_dw = at; j.grad_type = bad);
			REFUSES(ty, j.d_dx = at; j.grad_type = bad);
			REFUSES(ty, j.d_db = at; j.grad_type = bad; j.work_bytes = (size_t)1 << 40);
			REFUSES(-1, j.d_dx = j.d_dw = j.d_db = at; j.grad_type = bad);
		}
		REFUSES(ty, j.d_dw = at; j.work_bytes -= 1);
		REFUSES(-1, j.d_dw = at; j.grad_type = ty);	/* the loss alone's work area */
		REFUSES(ty, j.d_dx = at; j.ld_dx = 15);
		REFUSES(ty, j.d_dx = (void *)(kAt + 1));
		REFUSES(ty, j.d_dw = (void *)(kAt + 1));
		REFUSES(ty, j.d_db = (void *)(kAt + 1));
		if (ty == ANNI_F32) {
			REFUSES(ty, j.d_dx = (void *)(kAt + 2));
			REFUSES(ty, j.d_dw = (void *)(kAt + 2));
			REFUSES(ty, j.d_db = (void *)(kAt + 2));
		} else {
			TAKES(ty, j.d_dx = j.d_dw = j.d_db = (void *)(kAt + 2));
		}
	}
	REFUSES(0, j.d_x = nullptr);
	REFUSES(0, j.d_w = nullptr);
	REFUSES(0, j.d_target = nullptr);
	REFUSES(0, j.d_nll = nullptr);
	REFUSES(0, j.d_work = nullptr);
	for (int64_t rows : { (int64_t)0, (int64_t)-3, kHeadMaxRows + 1, INT64_MIN, INT64_MAX })
		REFUSES(0, j.rows = rows; j.work_bytes = SIZE_MAX);
	for (int d : { 0, -1, kHeadMaxD + 1, INT32_MIN, INT32_MAX })
		REFUSES(0, j.d = d; j.ld_x = INT64_MAX; j.work_bytes = SIZE_MAX);
	for (int vocab : { 0, -1, kHeadMaxVocab + 1, INT32_MIN, INT32_MAX })
		REFUSES(0, j.vocab = vocab; j.work_bytes = SIZE_MAX);
	REFUSES(0, j.rows = ((int64_t)1 << 20) + 1; j.vocab = 1 << 18; j.work_bytes = SIZE_MAX);
	REFUSES(0, j.ld_x = 15);
	REFUSES(0, j.ld_x = -16);
	REFUSES(0, j.d_x = (void *)(kAt + 1));
	REFUSES(0, j.d_w = (void *)(kAt + 1));
	REFUSES(0, j.d_target = (const int32_t *)(kAt + 2));
	REFUSES(0, j.d_nll = (float *)(kAt + 1));
	REFUSES(0, j.d_bias = (const float *)(kAt + 2));
	REFUSES(0, j.d_work = (void *)(kAt + 128));
	REFUSES(-1, j.work_bytes -= 1);
	REFUSES(0, j.work_bytes = 0);
	{
		HeadPlan p;
		bool grad;

		CHECK(!head_job_plan(nullptr, &p, &grad));
	}
}

/* What head_run() and the kernels take for granted of a plan. */
static void plan_holds(int64_t rows, int d, int vocab, int ty)
{
	HeadPlan p;

	plans++;
	CHECK(head_plan(rows, d, vocab, ty, &p));
	CHECK(p.rows_pad >= rows && p.rows_pad % p.tile_t == 0 && p.rows_pad % p.dx_t == 0 && p.rows_pad % kStep == 0);
	CHECK(p.d_pad >= d && p.d_pad % kSide == 0 && p.vocab_pad >= vocab && p.vocab_pad % kSide == 0);
	CHECK(p.tiles_v * p.tile_v <= p.vocab_pad && (p.tiles_v - 1) * p.tile_v < vocab);
	CHECK(p.off_ws <= p.off_xs && p.off_xs < p.off_ts && p.off_ts < p.off_bs && p.off_bs < p.off_part
	    && p.off_part < p.off_hit && p.off_hit < p.off_lse && p.off_lse < p.bytes && p.bytes <= p.bytes_keep);
	CHECK((p.off_xs | p.off_ts | p.off_bs | p.off_part | p.off_hit | p.off_lse | p.off_delta | p.off_kept | p.off_slot
	    | p.off_slot_w) % 256 == 0);
	if (ty == -1) {
		CHECK(p.bytes == p.bytes_keep && !p.keeps);
		return;
	}
	CHECK(p.parts == (ty == ANNI_F32 ? 2 : 1));
	CHECK(p.piece > 0 && p.piece % kSide == 0 && p.piece <= p.vocab_pad && p.ld_delta >= p.piece);
	CHECK(p.side_w == 128 || p.side_w == 256);
	CHECK(p.splits >= 1 && p.splits <= p.piece / kStep * p.parts);
	CHECK(p.splits_w >= 1 && p.splits_w <= p.rows_pad / kStep * p.parts && (p.splits_w == 1 || p.side_w == 128));
	CHECK(p.d_slot >= d && p.d_slot % p.tile_d == 0 && p.slot_rows_w >= d);
	CHECK(p.off_delta < p.off_slot && p.off_slot < p.off_slot_w && p.off_slot_w <= p.bytes);
	CHECK(p.off_slot - p.off_delta >= (size_t)p.rows_pad * p.ld_delta * 2 * p.parts);
	CHECK(p.off_slot_w - p.off_slot >= (size_t)p.splits * p.rows_pad * p.d_slot * 4);
	/* the small tiles have no pass that forms delta from logits computed again */
	CHECK(p.tile_t != 64 || (p.keeps && p.bytes == p.bytes_keep));
	if (p.keeps)
		CHECK(p.bytes_keep - p.off_kept >= (size_t)p.rows_pad * p.vocab_pad * 4);
}

int main(int argc, char **argv)
{
	static const int64_t rows[] = { 1, 2, 63, 64, 65, 96, 127, 129, 254, 517, 777, 1024, 2048, 4096, 8192, 65537, 1 << 22 };
	static const int ds[] = { 1, 7, 64, 128, 191, 192, 331, 712, 1024, 1536, 4096, 1 << 16 };
	static const int vocabs[] = { 1, 7, 130, 255, 256, 257, 1000, 10007, 16384, 50257, 65536, 100000, 1 << 22 };

	for (int i = 1; i + 3 < argc; i += 4) {
		HeadPlan p;

		if (!head_plan(atoll(argv[i]), atoi(argv[i + 1]), atoi(argv[i + 2]), atoi(argv[i + 3]), &p))
			return 1;
		printf("logits %d dx %d dw %d slices_dx %d slices_dw %d pieces %d copied %d keeps %d always %d\n", p.tile_t, p.dx,
		    p.side_w, p.splits > 1, p.splits_w > 1, p.piece ? (int)count(p.vocab_pad, p.piece) : 0, p.align, p.keeps,
		    p.keeps && p.bytes == p.bytes_keep);
	}
	if (argc > 1)
		return 0;
	jobs();
	for (int64_t r : rows)
		for (int d : ds)
			for (int v : vocabs)
				if (r * v <= kHeadMaxLogits)
					for (int ty = -1; ty <= ANNI_BF16; ty++)
						plan_holds(r, d, v, ty);
	if (fails)
		printf("%d failed\n", fails);
	else
		printf("ok refused %d taken %d plans %d\n", refused, taken, plans);
	return fails != 0;
}
