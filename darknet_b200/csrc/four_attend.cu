// xnor_b200_kv4_attend: how a call is cut into tiles of columns and splits of its positions, and its checks (the kernels: four_attend.cuh).
#include <climits>
#include <cmath>

#include "four_attend.cuh"

namespace xnor
{

int validate_kv4(const xnor_b200_kv4_cache * c, const xnor_b200_kv4_rows * r);

static AttendPlan plan_attend(const xnor_b200_kv4_cache & c, const xnor_b200_kv4_rows & r, int heads, int window)
{
	AttendPlan a;
	const long long columns = (long long)r.tokens * (heads / c.kv_heads);
	// tiles of columns: every tile goes over the cache and makes operands of its codes (which is some two thirds of a tile of eight)
	a.nt = 1;
	if (c.dim <= 128)
	{
		for (int nt = 2; nt <= 3; ++nt)
		{
			const long long cost = (columns + nt * 8 - 1) / (nt * 8) * (2 + nt), least = (columns + a.nt * 8 - 1) / (a.nt * 8) * (2 + a.nt);
			if (cost < least) { a.nt = nt; }
		}
	}
	const long long tiles = (columns + a.nt * 8 - 1) / (a.nt * 8), base = tiles * c.kv_heads * r.batch;
	a.tiles = (int)(tiles < INT_MAX ? tiles : INT_MAX);
	long long most = (long long)r.max_pages * c.page;                          // positions that a tile may see
	if (window > 0 && most > (long long)window + r.tokens) { most = (long long)window + r.tokens; }
	const long long steps = (most + 15) / 16, sms = sm_count();
	// A CTA costs about 2 us of an SM's time before and after its steps, and hides latency for the others; its sums have to be joined: up to two
	// on an SM as long as each of their warps has a pair of steps, more where the steps are many.  One sequence, us at 2 / 3 / 4 CTAs on an
	// SM: 8 heads of 128 channels by 64, 16384 positions 18.8 / 18.9 / 16.4, 65536 44 / 34.7 / 29.3, 131072 78 / 59 / 48.4, 262144 145 / 104 / 82;
	// 8 heads of 64 by 32, 16384 15.5 / 15.5 / 15.0, 65536 33 / 30.5 / 26, 131072 56 / 49 / 40.5; 2 heads of 64 by 16 (four times the splits a
	// head to join), 32768 14.5 / 14.5 / 16.1, 65536 16.7 / 16.7 / 20.9, 131072 20.9 / 22.5 / 23.8, 262144 29.7 / 30.0 / 29.2.
	const int on_sm = attend_on_sm(c.dim / 32, a.nt);
	long long splits = 1;
	for (int k = 1; k <= on_sm; ++k)
	{
		const long long s = k * sms / base, least = k <= 2 ? 2 * FA_WARPS : k == 3 ? 32 : 60;
		if (s > splits && (k <= 2 || s * least <= steps)) { splits = s; }
		if (k <= 2 && splits * least > steps) { splits = steps / least > 1 ? steps / least : 1; }
	}
	if (splits > FJ_SPLITS) { splits = FJ_SPLITS; }
	a.cluster = splits <= 8;
	a.splits = (int)splits;
	return a;
}

static int check_attend(const xnor_b200_kv4_cache * cache, const xnor_b200_kv4_rows * rows, int heads, int window)
{
	const int rc = validate_kv4(cache, rows);
	if (rc != XNOR_B200_OK) { return rc; }
	if (heads <= 0 || heads % cache->kv_heads != 0 || window < 0) { return XNOR_B200_ERR_INVALID; }
	if ((long long)cache->pages * cache->kv_heads * (cache->page / 16) > 0x7fffffffLL) { return XNOR_B200_ERR_TOO_LARGE; }
	const AttendPlan a = plan_attend(*cache, *rows, heads, window);
	if ((long long)a.tiles * cache->kv_heads > 65535 || (long long)rows->tokens * (heads / cache->kv_heads) > INT_MAX) { return XNOR_B200_ERR_TOO_LARGE; }
	return XNOR_B200_OK;
}

}  // namespace xnor

using namespace xnor;

extern "C" size_t xnor_b200_kv4_attend_scratch_bytes(const xnor_b200_kv4_cache * cache, const xnor_b200_kv4_rows * rows, int heads, int window)
{
	if (check_attend(cache, rows, heads, window) != XNOR_B200_OK) { return 0; }
	const AttendPlan a = plan_attend(*cache, *rows, heads, window);
	return a.cluster ? 0 : (size_t)rows->batch * cache->kv_heads * a.tiles * a.splits * a.nt * 8 * (cache->dim + 4) * sizeof(float);
}

extern "C" int xnor_b200_kv4_attend(const xnor_b200_kv4_cache * cache, const xnor_b200_kv4_rows * rows, const xnor_b200_kv4_tensor * q, int heads,
		float scale, int window, const xnor_b200_kv4_tensor * output, float * lse, void * scratch, size_t scratch_bytes, void * stream)
{
	const int rc = check_attend(cache, rows, heads, window);
	if (rc != XNOR_B200_OK) { return rc; }
	if (q == nullptr || output == nullptr || q->data == nullptr || output->data == nullptr) { return XNOR_B200_ERR_NULL; }
	if (!four_dtype_ok(q->dtype) || q->dtype != output->dtype || !std::isfinite(scale)) { return XNOR_B200_ERR_INVALID; }
	const size_t size = four_size(q->dtype);
	if (((uintptr_t)q->data & (size - 1)) != 0 || ((uintptr_t)output->data & (size - 1)) != 0 || ((uintptr_t)lse & 3) != 0) { return XNOR_B200_ERR_ALIGNMENT; }
	const AttendPlan plan = plan_attend(*cache, *rows, heads, window);
	AttendParams p = {};
	if (!plan.cluster)
	{
		if (scratch == nullptr) { return XNOR_B200_ERR_NULL; }
		if (scratch_bytes < xnor_b200_kv4_attend_scratch_bytes(cache, rows, heads, window)) { return XNOR_B200_ERR_SCRATCH; }
		if (((uintptr_t)scratch & 15) != 0) { return XNOR_B200_ERR_ALIGNMENT; }
		p.partial = (float *)scratch;
	}
	p.c = *cache;
	p.r = *rows;
	p.q = *q;
	p.out = *output;
	p.lse = lse;
	p.scale_log2 = scale * 1.4426950408889634f;
	p.heads = heads;
	p.share = heads / cache->kv_heads;
	p.window = window;
	const long long room = (long long)rows->max_pages * cache->page;
	p.room = room < INT_MAX ? (int)room : INT_MAX;
	p.splits = plan.splits;
	p.tiles = plan.tiles;
	const auto fits = [size](const xnor_b200_kv4_tensor & t, long long bytes)
	{
		return (uintptr_t)t.data % bytes == 0 && t.stride_sequence * (long long)size % bytes == 0 && t.stride_token * (long long)size % bytes == 0
				&& t.stride_head * (long long)size % bytes == 0;
	};
	p.wide_q = fits(*q, 16);
	p.wide_out = fits(*output, (long long)size * 4);
	const cudaStream_t s = (cudaStream_t)stream;
	switch (q->dtype)
	{
		case XNOR_B200_F32: return launch_attend_f32(p, plan, s);
		case XNOR_B200_F16: return launch_attend_f16(p, plan, s);
		default: return launch_attend_bf16(p, plan, s);
	}
}
