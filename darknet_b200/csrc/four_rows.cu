// Rows of values to four bits and back: the weights of a matrix (load time), and the tokens of a paged cache of keys and values.
//
//   low = min rounded down to fp16, scale = (max - low) / 15 rounded up to fp16, code = round((v - low) / scale), half to even
//
// Both roundings are outwards, so nothing is clipped and every value comes back within half a scale.  Rounding the difference and the
// quotient up in fp32 on the way gives the same scale as one rounding of the exact quotient: each step's result is the smallest fp32 value
// not below, and an fp16 value (times 15) is one of those.  NaN counts as 0, and what fp16 cannot hold as its largest value.
//
// A thread owns eight neighbours, one word of codes; the 4, 8 or 16 threads of a group find its minimum and maximum by shuffles.
#include "four_common.cuh"

namespace xnor
{

constexpr int FR_THREADS = 128;

// Eight neighbours of a group, `there` of them real, to a word of codes; every lane of the group returns (scale, low).
__device__ __forceinline__ uint32_t quantize8(float (&v)[8], int there, int group_lanes, __half2 & pair)
{
	float low = INFINITY, top = -INFINITY;
	#pragma unroll
	for (int i = 0; i < 8; ++i)
	{
		v[i] = v[i] != v[i] ? 0.0f : fminf(fmaxf(v[i], -65504.0f), 65504.0f);
		if (i < there) { low = fminf(low, v[i]); top = fmaxf(top, v[i]); }
	}
	for (int m = 1; m < group_lanes; m <<= 1)
	{
		low = fminf(low, __shfl_xor_sync(0xffffffffu, low, m));
		top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
	}
	const __half l = __float2half_rd(low);
	const float base = __half2float(l);
	const __half s = __float2half_ru(__fdiv_ru(__fsub_ru(top, base), 15.0f));
	const float step = __half2float(s);
	pair = __halves2half2(s, l);
	uint32_t word = 0;
	#pragma unroll
	for (int i = 0; i < 8; ++i)
	{
		const float q = step > 0.0f && i < there ? rintf(__fdiv_rn(v[i] - base, step)) : 0.0f;
		word |= (uint32_t)fminf(fmaxf(q, 0.0f), 15.0f) << (4 * i);
	}
	return word;
}

// One block a row; k need not fill the last group, nor the last 16 bytes of codes (0 there).
template <class T>
__global__ void __launch_bounds__(FR_THREADS)
four_weights_kernel(const T * __restrict__ weights, long long ld, int k, int group, uint32_t * __restrict__ codes, __half2 * __restrict__ scales, int wide)
{
	const int words = (int)(four_row_bytes(k) / 4), groups = (k + group - 1) / group, lanes = group / 8;
	const T * row = weights + (long long)blockIdx.x * ld;
	for (int w0 = 0; w0 < groups * lanes; w0 += FR_THREADS)
	{
		const int w = w0 + threadIdx.x, there = min(8, k - 8 * w);
		float v[8];
		eight_f32(load8(row + 8 * (long long)w, there, wide != 0), v);
		__half2 pair;
		const uint32_t word = quantize8(v, there, lanes, pair);
		if (w < words) { codes[(size_t)blockIdx.x * words + w] = word; }
		if (w % lanes == 0 && w < groups * lanes) { scales[(size_t)blockIdx.x * groups + w / lanes] = pair; }
	}
}

// The page and the place of row i of sequence b; page < 0: there is none.
__device__ __forceinline__ void find_row(const xnor_b200_kv4_cache & c, const xnor_b200_kv4_rows & r, int b, int i, long long & page, int & place)
{
	const int count = r.counts != nullptr ? __ldg(r.counts + b) : r.tokens;
	const long long at = (long long)__ldg(r.lengths + b) - count + i;
	page = -1;
	place = 0;
	if (i >= count || at < 0 || at >= (long long)r.max_pages * c.page) { return; }
	const int p = __ldg(r.table + (long long)b * r.max_pages + at / c.page);
	if (p >= 0 && p < c.pages) { page = p; place = (int)(at % c.page); }
}

struct RowsParams
{
	xnor_b200_kv4_cache c;
	xnor_b200_kv4_rows r;
	xnor_b200_kv4_tensor t[2];       // keys, values
	int wide[2];                     // rows of it start on 16 bytes
};

// One block a row of tokens and half (keys or values).
template <class T>
__global__ void __launch_bounds__(FR_THREADS)
kv4_append_kernel(const RowsParams p)
{
	const int half = blockIdx.y, b = blockIdx.x / p.r.tokens, i = blockIdx.x - b * p.r.tokens;
	long long page;
	int place;
	find_row(p.c, p.r, b, i, page, place);
	if (page < 0) { return; }
	const xnor_b200_kv4_tensor & t = p.t[half];
	const int words = p.c.dim / 8, lanes = p.c.group / 8, groups = p.c.dim / p.c.group, total = words * p.c.kv_heads;
	const T * src = (const T *)t.data + b * t.stride_sequence + i * t.stride_token;
	uint32_t * codes = (uint32_t *)(half ? p.c.v_codes : p.c.k_codes);
	__half2 * scales = (__half2 *)(half ? p.c.v_scales : p.c.k_scales);
	for (int w0 = 0; w0 < total; w0 += FR_THREADS)
	{
		const int w = w0 + threadIdx.x, head = w / words, word = w - head * words;
		float v[8];
		eight_f32(load8(src + head * t.stride_head + 8 * word, w < total ? 8 : 0, p.wide[half] != 0), v);
		__half2 pair;
		const uint32_t c = quantize8(v, 8, lanes, pair);
		if (w >= total) { continue; }
		const long long row = (page * p.c.kv_heads + head) * p.c.page + place;
		codes[row * words + word] = c;
		if (word % lanes == 0) { scales[row * groups + word / lanes] = pair; }
	}
}

template <class T>
__global__ void __launch_bounds__(FR_THREADS)
kv4_read_kernel(const RowsParams p)
{
	const int half = blockIdx.y, b = blockIdx.x / p.r.tokens, i = blockIdx.x - b * p.r.tokens;
	long long page;
	int place;
	find_row(p.c, p.r, b, i, page, place);
	const xnor_b200_kv4_tensor & t = p.t[half];
	const int words = p.c.dim / 8, lanes = p.c.group / 8, groups = p.c.dim / p.c.group, total = words * p.c.kv_heads;
	T * dst = (T *)t.data + b * t.stride_sequence + i * t.stride_token;
	const uint32_t * codes = (const uint32_t *)(half ? p.c.v_codes : p.c.k_codes);
	const __half2 * scales = (const __half2 *)(half ? p.c.v_scales : p.c.k_scales);
	for (int w = threadIdx.x; w < total; w += FR_THREADS)
	{
		const int head = w / words, word = w - head * words;
		float v[8] = {};
		if (page >= 0)
		{
			const long long row = (page * p.c.kv_heads + head) * p.c.page + place;
			const uint32_t c = codes[row * words + word];
			const float2 sl = __half22float2(scales[row * groups + word / lanes]);
			#pragma unroll
			for (int e = 0; e < 8; ++e) { v[e] = __fmaf_rn(sl.x, (float)((c >> (4 * e)) & 15), sl.y); }
		}
		store8(dst + head * t.stride_head + 8 * word, p.wide[half] != 0, v);
	}
}

static bool aligned(const void * p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

int validate_kv4(const xnor_b200_kv4_cache * c, const xnor_b200_kv4_rows * r)
{
	if (c == nullptr || r == nullptr) { return XNOR_B200_ERR_NULL; }
	if (c->pages <= 0 || c->kv_heads <= 0 || c->page <= 0 || c->page % 16 != 0 || c->dim <= 0 || c->dim % 32 != 0 || !four_group_ok(c->group)
			|| c->dim % c->group != 0 || r->batch <= 0 || r->tokens <= 0 || r->max_pages <= 0) { return XNOR_B200_ERR_INVALID; }
	if (c->dim > XNOR_B200_KV4_MAX_DIM || c->kv_heads > 65535 || c->page > (1 << 20) || (long long)r->batch * r->tokens > 0x7fffffffLL) { return XNOR_B200_ERR_TOO_LARGE; }
	if (c->k_codes == nullptr || c->k_scales == nullptr || c->v_codes == nullptr || c->v_scales == nullptr || r->table == nullptr || r->lengths == nullptr)
	{
		return XNOR_B200_ERR_NULL;
	}
	if (!aligned(c->k_codes, 16) || !aligned(c->v_codes, 16) || !aligned(c->k_scales, 16) || !aligned(c->v_scales, 16) || !aligned(r->table, 4)
			|| !aligned(r->lengths, 4) || !aligned(r->counts, 4)) { return XNOR_B200_ERR_ALIGNMENT; }
	return XNOR_B200_OK;
}

static int fill_rows(RowsParams & p, const xnor_b200_kv4_cache * c, const xnor_b200_kv4_rows * r, const xnor_b200_kv4_tensor * k, const xnor_b200_kv4_tensor * v)
{
	const int rc = validate_kv4(c, r);
	if (rc != XNOR_B200_OK) { return rc; }
	if (k == nullptr || v == nullptr || k->data == nullptr || v->data == nullptr) { return XNOR_B200_ERR_NULL; }
	if (!four_dtype_ok(k->dtype) || k->dtype != v->dtype) { return XNOR_B200_ERR_INVALID; }
	p.c = *c;
	p.r = *r;
	const xnor_b200_kv4_tensor * both[2] = {k, v};
	for (int i = 0; i < 2; ++i)
	{
		const xnor_b200_kv4_tensor & t = *both[i];
		const long long size = (long long)four_size(t.dtype);
		if (!aligned(t.data, (size_t)size)) { return XNOR_B200_ERR_ALIGNMENT; }
		p.t[i] = t;
		p.wide[i] = aligned(t.data, 16) && t.stride_sequence * size % 16 == 0 && t.stride_token * size % 16 == 0 && t.stride_head * size % 16 == 0;
	}
	return XNOR_B200_OK;
}

}  // namespace xnor

using namespace xnor;

extern "C" size_t xnor_b200_w4_code_bytes(const xnor_b200_w4_desc * d)
{
	return d == nullptr || d->n <= 0 || d->k <= 0 || !four_group_ok(d->group) ? 0 : (size_t)d->n * four_row_bytes(d->k);
}

extern "C" size_t xnor_b200_w4_scale_bytes(const xnor_b200_w4_desc * d)
{
	return d == nullptr || d->n <= 0 || d->k <= 0 || !four_group_ok(d->group) ? 0 : (size_t)d->n * ((size_t)(d->k - 1) / d->group + 1) * 4;
}

extern "C" int xnor_b200_w4_quantize(const xnor_b200_w4_desc * d, const void * weights, int dtype, long long ld, uint8_t * codes, void * scales, void * stream)
{
	if (d == nullptr || weights == nullptr || codes == nullptr || scales == nullptr) { return XNOR_B200_ERR_NULL; }
	if (d->n <= 0 || d->k <= 0 || !four_group_ok(d->group) || !four_dtype_ok(dtype) || ld < 0) { return XNOR_B200_ERR_INVALID; }
	if (d->k > XNOR_B200_W4_MAX_K) { return XNOR_B200_ERR_TOO_LARGE; }
	const size_t size = four_size(dtype);
	if (!aligned(weights, size) || !aligned(codes, 16) || !aligned(scales, 4)) { return XNOR_B200_ERR_ALIGNMENT; }
	const int wide = aligned(weights, 16) && ld * (long long)size % 16 == 0;
	const cudaStream_t s = (cudaStream_t)stream;
	if (dtype == XNOR_B200_F32)
	{
		four_weights_kernel<<<d->n, FR_THREADS, 0, s>>>((const float *)weights, ld, d->k, d->group, (uint32_t *)codes, (__half2 *)scales, wide);
	}
	else if (dtype == XNOR_B200_F16)
	{
		four_weights_kernel<<<d->n, FR_THREADS, 0, s>>>((const __half *)weights, ld, d->k, d->group, (uint32_t *)codes, (__half2 *)scales, wide);
	}
	else
	{
		four_weights_kernel<<<d->n, FR_THREADS, 0, s>>>((const __nv_bfloat16 *)weights, ld, d->k, d->group, (uint32_t *)codes, (__half2 *)scales, wide);
	}
	return check_launch();
}

extern "C" int xnor_b200_kv4_append(const xnor_b200_kv4_cache * cache, const xnor_b200_kv4_rows * rows, const xnor_b200_kv4_tensor * k,
		const xnor_b200_kv4_tensor * v, void * stream)
{
	RowsParams p;
	const int rc = fill_rows(p, cache, rows, k, v);
	if (rc != XNOR_B200_OK) { return rc; }
	const dim3 grid((unsigned)(rows->batch * rows->tokens), 2);
	const cudaStream_t s = (cudaStream_t)stream;
	if (k->dtype == XNOR_B200_F32) { kv4_append_kernel<float><<<grid, FR_THREADS, 0, s>>>(p); }
	else if (k->dtype == XNOR_B200_F16) { kv4_append_kernel<__half><<<grid, FR_THREADS, 0, s>>>(p); }
	else { kv4_append_kernel<__nv_bfloat16><<<grid, FR_THREADS, 0, s>>>(p); }
	return check_launch();
}

extern "C" int xnor_b200_kv4_read(const xnor_b200_kv4_cache * cache, const xnor_b200_kv4_rows * rows, const xnor_b200_kv4_tensor * k,
		const xnor_b200_kv4_tensor * v, void * stream)
{
	RowsParams p;
	const int rc = fill_rows(p, cache, rows, k, v);
	if (rc != XNOR_B200_OK) { return rc; }
	const dim3 grid((unsigned)(rows->batch * rows->tokens), 2);
	const cudaStream_t s = (cudaStream_t)stream;
	if (k->dtype == XNOR_B200_F32) { kv4_read_kernel<float><<<grid, FR_THREADS, 0, s>>>(p); }
	else if (k->dtype == XNOR_B200_F16) { kv4_read_kernel<__half><<<grid, FR_THREADS, 0, s>>>(p); }
	else { kv4_read_kernel<__nv_bfloat16><<<grid, FR_THREADS, 0, s>>>(p); }
	return check_launch();
}
