// Rows of values to four bits and back: the weights of a matrix (load time), and the tokens of a paged cache of keys and values.
//
//   low = min rounded down to fp16, scale = (max - low) / 15 rounded up to fp16, code = round((v - low) / scale), half to even
//
// Both roundings are outwards, so nothing is clipped and every value comes back within half a scale.  Rounding the difference and the
// quotient up in fp32 on the way gives the same scale as one rounding of the exact quotient: each step's result is the smallest fp32 value
// not below, and an fp16 value (times 15) is one of those.  NaN counts as 0, and what fp16 cannot hold as its largest value.
//
// A thread owns 16 neighbours, two words of codes; the 2, 4 or 8 threads of a group find its minimum and maximum by shuffles.  Bound by
// what a thread has to do rather than by memory, so: the minimum and the maximum of 16-bit values are taken in pairs; the scale is one
// product and a check; the quotient is a product with 1/scale, whose nearest integer is the bits of its sum with 1.5 * 2^23, and the
// remainder tells whether it is close to a half and which way it has to go; what fp16 cannot hold and NaN show in the minimum and the
// maximum.  4 x 2048 tokens (three quarters of them new) of 8 heads of 128 fp16 channels, keys and values: 13.6 us, 2.5 TB/s; 29 with
// divisions and 8 neighbours a thread.  The other way 9.4 us, 3.6 TB/s.  A matrix of 16384 x 16384 fp32 values: 199 us, 6.2 TB/s; 4096 x 4096
// of fp16, from the L2, 18.6 us.
#include "four_common.cuh"

namespace xnor
{

constexpr int FR_THREADS = 128;

__device__ __forceinline__ float reciprocal(float v)
{
	float r;
	asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
	return r;
}

// Least and largest of eight neighbours, NaN where there is one.
__device__ __forceinline__ void least_and_largest(const Eight<float> & e, float & low, float & top)
{
	const float * v = reinterpret_cast<const float *>(e.raw);
	low = top = v[0];
	#pragma unroll
	for (int i = 1; i < 8; ++i)
	{
		low = min_nan(low, v[i]);
		top = max_nan(top, v[i]);
	}
}
__device__ __forceinline__ void least_and_largest(const Eight<__half> & e, float & low, float & top)
{
	const __half2 * v = reinterpret_cast<const __half2 *>(e.raw);
	const float2 l = __half22float2(__hmin2_nan(__hmin2_nan(v[0], v[1]), __hmin2_nan(v[2], v[3])));
	const float2 t = __half22float2(__hmax2_nan(__hmax2_nan(v[0], v[1]), __hmax2_nan(v[2], v[3])));
	low = min_nan(l.x, l.y);
	top = max_nan(t.x, t.y);
}
__device__ __forceinline__ void least_and_largest(const Eight<__nv_bfloat16> & e, float & low, float & top)
{
	const __nv_bfloat162 * v = reinterpret_cast<const __nv_bfloat162 *>(e.raw);
	const float2 l = __bfloat1622float2(__hmin2_nan(__hmin2_nan(v[0], v[1]), __hmin2_nan(v[2], v[3])));
	const float2 t = __bfloat1622float2(__hmax2_nan(__hmax2_nan(v[0], v[1]), __hmax2_nan(v[2], v[3])));
	low = min_nan(l.x, l.y);
	top = max_nan(t.x, t.y);
}

// 16 neighbours of a group, `there` of them real, to two words of codes; every lane of the group returns (scale, low).
template <class T>
__device__ __forceinline__ uint2 quantize16(const Eight<T> & e0, const Eight<T> & e1, int there, int group_lanes, __half2 & pair)
{
	float v[16], low, top, more_low, more_top;
	eight_f32(e0, reinterpret_cast<float (&)[8]>(v[0]));
	eight_f32(e1, reinterpret_cast<float (&)[8]>(v[8]));
	least_and_largest(e0, low, top);
	least_and_largest(e1, more_low, more_top);
	low = min_nan(low, more_low);
	top = max_nan(top, more_top);
	if (there < 16 || !(low >= -65504.0f && top <= 65504.0f))
	{
		low = INFINITY;
		top = -INFINITY;
		#pragma unroll
		for (int i = 0; i < 16; ++i)
		{
			v[i] = v[i] != v[i] ? 0.0f : fminf(fmaxf(v[i], -65504.0f), 65504.0f);
			low = i < there ? fminf(low, v[i]) : low;
			top = i < there ? fmaxf(top, v[i]) : top;
		}
	}
	for (int m = 1; m < group_lanes; m <<= 1)
	{
		low = fminf(low, __shfl_xor_sync(0xffffffffu, low, m));
		top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
	}
	const __half l = __float2half_rd(low);
	const float base = __half2float(l), range = __fsub_ru(top, base);
	// the smallest fp16 value whose 15-fold is not below the range (a product of 15 bits, exact): next to the rounded quotient
	uint32_t bits = __half_as_ushort(__float2half_rn(range * (1.0f / 15.0f)));
	if (15.0f * __half2float(__ushort_as_half((unsigned short)bits)) < range) { ++bits; }
	else if (bits > 0 && 15.0f * __half2float(__ushort_as_half((unsigned short)(bits - 1))) >= range) { --bits; }
	const __half s = __ushort_as_half((unsigned short)bits);
	const float step = __half2float(s), by = step > 0.0f ? reciprocal(step) : 0.0f;
	pair = __halves2half2(s, l);
	// the bits of 1.5 * 2^23 + code are 0x4b400000 + code: times 16^i they add up to the word and a constant
	//
	// Next to a half the quotient (off by less than 2^-21 of what is below 16, with the difference's rounding) may have gone the wrong way.
	// The remainder says so: the difference less what it lost in rounding, exactly; where it is a half the even code is the nearest.  A scale
	// of 0 has no remainder.
	uint32_t word[2] = {0u - 0x4b400000u * 0x11111111u, 0u - 0x4b400000u * 0x11111111u};
	const float near = step * (0.5f - 0x1p-16f);
	#pragma unroll
	for (int i = 0; i < 16; ++i)
	{
		const float d = v[i] - base, t = fmaf(d, by, 12582912.0f), rest = fmaf(-(t - 12582912.0f), step, d);
		uint32_t bits_of = __float_as_uint(t);
		if (fabsf(rest) > near)
		{
			const float back = d - v[i], lost = (v[i] - (d - back)) - (base + back);                  // v - low = d + lost
			const float over = (rest - 0.5f * step) + lost, under = (rest + 0.5f * step) + lost;
			const bool odd = bits_of & 1;
			bits_of += over > 0.0f || (over == 0.0f && odd) ? 1 : under < 0.0f || (under == 0.0f && odd) ? -1 : 0;
			asm volatile("");                                     // (a branch that is hardly ever taken)
		}
		word[i / 8] += bits_of * (1u << (4 * (i % 8)));
	}
	if (there < 16)                                           // what is not there is 0
	{
		word[0] &= there >= 8 ? 0xffffffffu : (1u << (4 * max(there, 0))) - 1;
		word[1] &= there <= 8 ? 0 : (1u << (4 * (there - 8))) - 1;
	}
	return make_uint2(word[0], word[1]);
}

// One block a row; k need not fill the last group, nor the last 16 bytes of codes (0 there).
template <class T>
__global__ void __launch_bounds__(FR_THREADS)
four_weights_kernel(const T * __restrict__ weights, long long ld, int k, int group, uint32_t * __restrict__ codes, __half2 * __restrict__ scales, int wide)
{
	const int twos = (int)(four_row_bytes(k) / 8), groups = (k + group - 1) / group, lanes = group / 16;
	const T * row = weights + (long long)blockIdx.x * ld;
	for (int w0 = 0; w0 < groups * lanes; w0 += FR_THREADS)
	{
		const int w = w0 + threadIdx.x, there = max(0, min(16, k - 16 * w));
		const Eight<T> e0 = load8(row + 16 * (long long)w, there, wide != 0), e1 = load8(row + 16 * (long long)w + 8, there - 8, wide != 0);
		__half2 pair;
		const uint2 two = quantize16(e0, e1, there, lanes, pair);
		if (w < twos) { ((uint2 *)codes)[(size_t)blockIdx.x * twos + w] = two; }
		if (w % lanes == 0 && w < groups * lanes) { scales[(size_t)blockIdx.x * groups + w / lanes] = pair; }
	}
}

// The page and the place of row i of sequence b; page < 0: there is none.
__device__ __forceinline__ void find_row(const xnor_b200_kv4_cache & c, const xnor_b200_kv4_rows & r, int b, int i, int & page, int & place)
{
	const int count = r.counts != nullptr ? r.counts[b] : r.tokens;
	const long long at = (long long)r.lengths[b] - count + i;
	page = -1;
	place = 0;
	if (i >= count || at < 0 || at > 0x7fffffffLL) { return; }               // (a length is below 2^31)
	const uint32_t of = (uint32_t)at / (uint32_t)c.page;
	if (of >= (uint32_t)r.max_pages) { return; }
	const int p = r.table[(size_t)b * r.max_pages + of];
	if (p >= 0 && p < c.pages) { page = p; place = (int)((uint32_t)at - of * (uint32_t)c.page); }
}

struct RowsParams
{
	xnor_b200_kv4_cache c;
	xnor_b200_kv4_rows r;
	xnor_b200_kv4_tensor t[2];       // keys, values
	int wide[2];                     // rows of it start on 16 bytes
	int words;                       // of a row of tokens, all heads
	int warps;                       // that share a row
	uint32_t by_words;               // ceil(2^32 / words of a head): the high half of a product with it divides what is below 2^27
};

// What a thread does: the words of one row from `first` on.  Every thread of a warp goes through the same number of turns (the groups'
// shuffles need all of them).
struct RowsTask
{
	int i, first, step;
};

__device__ __forceinline__ RowsTask task_of(const RowsParams & p)
{
	RowsTask k;
	k.step = 32 * p.warps;
	k.first = p.warps == 1 ? (int)threadIdx.x % 32 : (int)threadIdx.x;
	k.i = p.warps == 1 ? (int)(blockIdx.x * (FR_THREADS / 32) + threadIdx.x / 32) : (int)blockIdx.x;
	return k;
}

// A block takes one row, or each of its warps one: of keys or of values.
template <class T>
__global__ void __launch_bounds__(FR_THREADS)
kv4_append_kernel(const RowsParams p)
{
	pdl_wait();
	pdl_trigger();
	const int half = blockIdx.z, b = blockIdx.y;
	const RowsTask k = task_of(p);
	if (k.i >= p.r.tokens) { return; }
	int page, place;
	find_row(p.c, p.r, b, k.i, page, place);
	if (page < 0) { return; }
	const xnor_b200_kv4_tensor & t = p.t[half];
	const int twos = p.c.dim / 16, lanes = p.c.group / 16, groups = p.c.dim / p.c.group, shift = p.c.group == 32 ? 1 : p.c.group == 64 ? 2 : 3;
	const T * src = (const T *)t.data + b * t.stride_sequence + k.i * t.stride_token;
	const size_t row0 = (size_t)page * p.c.kv_heads * p.c.page + place;
	uint2 * codes = (uint2 *)(half ? p.c.v_codes : p.c.k_codes);
	__half2 * scales = (__half2 *)(half ? p.c.v_scales : p.c.k_scales);
	const int all = p.words / 2;
	#pragma unroll 1
	for (int w0 = 0; w0 < all; w0 += k.step)
	{
		const int w = w0 + k.first, head = (int)__umulhi((uint32_t)w * 2, p.by_words), two = w - head * twos;
		const T * from = src + head * t.stride_head + 16 * two;
		const Eight<T> e0 = load8(from, w < all ? 8 : 0, p.wide[half] != 0), e1 = load8(from + 8, w < all ? 8 : 0, p.wide[half] != 0);
		__half2 pair;
		const uint2 c = quantize16(e0, e1, 16, lanes, pair);
		if (w >= all) { continue; }
		const size_t row = row0 + (size_t)head * p.c.page;
		codes[row * twos + two] = c;
		if ((two & (lanes - 1)) == 0) { scales[row * groups + (two >> shift)] = pair; }
	}
}

// Codes as pairs of fp16 numbers, the low four bits of each half (even) or the next four (odd).
__device__ __forceinline__ float2 even_values(uint32_t w)
{
	return __half22float2(__hadd2(as_half2(masked<0x000F000Fu, true>(w)), as_half2(0xE400E400u)));
}
__device__ __forceinline__ float2 odd_values(uint32_t w)
{
	return __half22float2(__hfma2(as_half2(masked<0x00F000F0u, true>(w)), as_half2(0x2C002C00u), as_half2(0xD400D400u)));
}

template <class T>
__global__ void __launch_bounds__(FR_THREADS)
kv4_read_kernel(const RowsParams p)
{
	pdl_wait();
	pdl_trigger();
	const int half = blockIdx.z, b = blockIdx.y;
	const RowsTask k = task_of(p);
	if (k.i >= p.r.tokens) { return; }
	int page, place;
	find_row(p.c, p.r, b, k.i, page, place);
	const xnor_b200_kv4_tensor & t = p.t[half];
	const int words = p.c.dim / 8, groups = p.c.dim / p.c.group, shift = p.c.group == 32 ? 2 : p.c.group == 64 ? 3 : 4;
	T * dst = (T *)t.data + b * t.stride_sequence + k.i * t.stride_token;
	const size_t row0 = (size_t)max(page, 0) * p.c.kv_heads * p.c.page + place;
	const uint32_t * codes = (const uint32_t *)(half ? p.c.v_codes : p.c.k_codes);
	const uint32_t * scales = (const uint32_t *)(half ? p.c.v_scales : p.c.k_scales);
	// four words at a time, all loaded before the first is stored (the compiler does not move a load in front of a store)
	constexpr int AHEAD = 4;
	#pragma unroll 1
	for (int w0 = k.first; w0 < p.words; w0 += AHEAD * k.step)
	{
		uint32_t c[AHEAD] = {}, pair[AHEAD] = {};
		#pragma unroll
		for (int j = 0; j < AHEAD; ++j)
		{
			const int w = w0 + j * k.step, head = (int)__umulhi((uint32_t)w, p.by_words), word = w - head * words;
			if (page < 0 || w >= p.words) { continue; }
			const size_t row = row0 + (size_t)head * p.c.page;
			c[j] = codes[row * words + word];
			pair[j] = scales[row * groups + (word >> shift)];
		}
		#pragma unroll
		for (int j = 0; j < AHEAD; ++j)
		{
			const int w = w0 + j * k.step, head = (int)__umulhi((uint32_t)w, p.by_words), word = w - head * words;
			if (w >= p.words) { break; }
			float v[8];
			const uint32_t up = upper(c[j]);
			const float2 sl = halves(pair[j]);
			const float2 pairs[4] = {even_values(c[j]), odd_values(c[j]), even_values(up), odd_values(up)};     // 0 and 4, 1 and 5, 2 and 6, 3 and 7
			#pragma unroll
			for (int e = 0; e < 4; ++e)
			{
				v[e] = __fmaf_rn(sl.x, pairs[e].x, sl.y);
				v[e + 4] = __fmaf_rn(sl.x, pairs[e].y, sl.y);
			}
			store8(dst + head * t.stride_head + 8 * word, p.wide[half] != 0, v);
		}
	}
}

static bool aligned(const void * p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

int validate_kv4(const xnor_b200_kv4_cache * c, const xnor_b200_kv4_rows * r)
{
	if (c == nullptr || r == nullptr) { return XNOR_B200_ERR_NULL; }
	if (c->pages <= 0 || c->kv_heads <= 0 || c->page <= 0 || c->page % 16 != 0 || c->dim <= 0 || c->dim % 32 != 0 || !four_group_ok(c->group)
			|| c->dim % c->group != 0 || r->batch <= 0 || r->tokens <= 0 || r->max_pages <= 0) { return XNOR_B200_ERR_INVALID; }
	if (c->dim > XNOR_B200_KV4_MAX_DIM || c->kv_heads > 65535 || c->page > (1 << 20) || r->batch > 65535) { return XNOR_B200_ERR_TOO_LARGE; }
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
	p.words = c->kv_heads * (c->dim / 8);
	// a warp a row where there are rows enough to fill a block with them; fewer are the sooner done the more threads they have
	p.warps = r->tokens >= FR_THREADS / 32 ? 1 : FR_THREADS / 32;
	p.by_words = (uint32_t)((0xffffffffu / (uint32_t)(c->dim / 8)) + 1);
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
	const dim3 grid((unsigned)(p.warps == 1 ? (rows->tokens - 1) / (FR_THREADS / 32) + 1 : rows->tokens), (unsigned)rows->batch, 2);
	const cudaStream_t s = (cudaStream_t)stream;
	if (k->dtype == XNOR_B200_F32) { return launch_four(kv4_append_kernel<float>, grid, FR_THREADS, 0, 1, s, p); }
	if (k->dtype == XNOR_B200_F16) { return launch_four(kv4_append_kernel<__half>, grid, FR_THREADS, 0, 1, s, p); }
	return launch_four(kv4_append_kernel<__nv_bfloat16>, grid, FR_THREADS, 0, 1, s, p);
}

extern "C" int xnor_b200_kv4_read(const xnor_b200_kv4_cache * cache, const xnor_b200_kv4_rows * rows, const xnor_b200_kv4_tensor * k,
		const xnor_b200_kv4_tensor * v, void * stream)
{
	RowsParams p;
	const int rc = fill_rows(p, cache, rows, k, v);
	if (rc != XNOR_B200_OK) { return rc; }
	const dim3 grid((unsigned)(p.warps == 1 ? (rows->tokens - 1) / (FR_THREADS / 32) + 1 : rows->tokens), (unsigned)rows->batch, 2);
	const cudaStream_t s = (cudaStream_t)stream;
	if (k->dtype == XNOR_B200_F32) { return launch_four(kv4_read_kernel<float>, grid, FR_THREADS, 0, 1, s, p); }
	if (k->dtype == XNOR_B200_F16) { return launch_four(kv4_read_kernel<__half>, grid, FR_THREADS, 0, 1, s, p); }
	return launch_four(kv4_read_kernel<__nv_bfloat16>, grid, FR_THREADS, 0, 1, s, p);
}
