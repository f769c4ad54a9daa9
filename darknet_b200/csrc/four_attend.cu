// Attention of a few tokens of each sequence over its cached keys and values, which lie in pages of four-bit rows.
//
//   out = sum_j softmax_j(scale * q . k_j) v_j over the positions j that the token sees, its own and those before it (the last `window`)
//
// Bound by the cache's way from memory: every row is read once, for all heads of queries that share it.  A query (head, token) is a
// column; a warp takes 16 positions at a time, its columns eight by eight, and both products run on the tensor cores with the codes as
// they lie (four_common.cuh):
//   scores  [16 positions x 8 columns] = codes of k . q         then  scale_k * that + low_k * sum(q), group by group
//   out     [16 channels x 8 columns] += codes of v . (p * scale_v), and sum(p * low_v) beside it in fp32
// q and p * scale_v are fp16 next to powers of two of their own (q: of the column; scale_v: of the largest so far), fp32 and fp16 calls
// split p * scale_v into two parts, fp32 calls q too.  The running maximum moves only when a score passes it by more than 2^8, so most
// steps neither exchange it nor rescale.
//
// A CTA has four warps that share a run of positions, step by step, each with a ring of its own; then their sums meet in shared memory.
// Long sequences are split over CTAs: up to eight of them are a cluster and meet in its shared memory, more leave their sums in the
// scratch buffer and a second kernel joins them.  Everything is summed in a fixed order.
#include <cooperative_groups.h>

#include <climits>
#include <cmath>

#include "four_common.cuh"

namespace xnor
{

namespace cg = cooperative_groups;

int validate_kv4(const xnor_b200_kv4_cache * c, const xnor_b200_kv4_rows * r);

constexpr int FA_WARPS = 4, FA_THREADS = 32 * FA_WARPS;
constexpr int FA_STAGES = 4;
constexpr float FA_SLACK = 8.0f;                          // how far (log2) a score may pass the running maximum

struct AttendParams
{
	xnor_b200_kv4_cache c;
	xnor_b200_kv4_rows r;
	xnor_b200_kv4_tensor q, out;
	float * lse;
	float * partial;              // [sequence][head of keys][tile][split][column]: dim sums, maximum, total; NULL: the CTAs of a cluster meet
	float scale_log2;             // scale * log2(e)
	int heads, share;             // heads of queries, and how many of them a head of keys serves
	int window, splits, tiles;    // tiles of columns
	int wide_q;
};

// What a tile of columns sees of its sequence.  Tokens of rows i0 .. i1.
struct Span
{
	int count;
	long long at;                 // position of row 0
	long long end;                // positions that there are
	long long first, last;        // first 16-position step and the one behind the last, of all columns
};

__device__ __forceinline__ Span span_of(const AttendParams & p, int b, int i0, int i1)
{
	Span s;
	s.count = p.r.counts != nullptr ? __ldg(p.r.counts + b) : p.r.tokens;
	const int length = __ldg(p.r.lengths + b);
	s.at = (long long)length - s.count;
	s.end = min((long long)length, (long long)p.r.max_pages * p.c.page);
	i1 = min(i1, s.count - 1);
	const long long to = i1 < i0 ? 0 : min(s.end, s.at + i1 + 1);
	const long long from = p.window > 0 ? max(0LL, s.at + i0 + 1 - p.window) : 0;
	s.first = from / 16;
	s.last = to > from ? (to + 15) / 16 : s.first;
	return s;
}

// Steps of one split: the same for the kernel and for the one that joins.
__device__ __forceinline__ long long steps_of_split(const Span & s, int splits)
{
	const long long n = s.last - s.first;
	return max((n + splits - 1) / splits, (long long)FA_WARPS);
}

__device__ __forceinline__ float exp2_fast(float v)
{
	float r;
	asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
	return r;
}

// What the sums at maximum m count for next to those at maximum `top`
__device__ __forceinline__ float weight_of(float m, float top) { return m == -INFINITY ? 0.0f : exp2_fast(m - top); }

__device__ __forceinline__ uint32_t transposed(uint32_t v)
{
	uint32_t r;
	asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
	return r;
}

template <class T> struct Parts { static constexpr int Q = 1, P = 1; };
template <> struct Parts<__half> { static constexpr int Q = 1, P = 2; };
template <> struct Parts<float> { static constexpr int Q = 2, P = 2; };

__host__ __device__ __forceinline__ int attend_pitch(int nb) { return (nb | 1) * 16; }           // of a row of codes: an odd number of 16 bytes
__host__ __device__ __forceinline__ int attend_stage(int nb, int groups) { return 32 * attend_pitch(nb) + 2 * 16 * groups * 4; }
__host__ __device__ __forceinline__ int attend_q_pitch(int nb) { return (nb | 1) * 64; }

// NB: most blocks of 32 channels.  GB: blocks of a group.  NT: tiles of eight columns.
template <class T, int NB, int GB, int NT>
__global__ void __launch_bounds__(FA_THREADS)
four_attend_kernel(const AttendParams p)
{
	constexpr int QP = Parts<T>::Q, PP = Parts<T>::P, COLS = NT * 8, GROUPS = NB / GB;
	using How = Codes<T>;
	constexpr bool CENTRED = How::CENTRED;
	extern __shared__ __align__(128) unsigned char smem[];
	const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
	const int dim = p.c.dim, nb = dim / 32, groups = dim / (32 * GB);
	const int pitch = attend_pitch(nb), stage_bytes = attend_stage(nb, groups), q_pitch = attend_q_pitch(nb);
	unsigned char * ring = smem + warp * FA_STAGES * stage_bytes;
	unsigned char * s_q = smem + FA_WARPS * FA_STAGES * stage_bytes;                  // [part][column][q_pitch]
	float * s_qf = (float *)(s_q + QP * COLS * q_pitch);                              // [column]
	float * s_qsum = s_qf + COLS;                                                     // [group][column]
	long long * s_from = (long long *)(s_qsum + GROUPS * COLS);                       // [column]: positions that it sees
	long long * s_to = s_from + COLS;
	float * s_m = (float *)(s_to + COLS);                                             // [warp][column]
	float * s_l = s_m + FA_WARPS * COLS;

	const int b = blockIdx.z, head = blockIdx.y / p.tiles, tile = blockIdx.y % p.tiles, split = blockIdx.x;
	const int col0 = tile * COLS, cols = min(COLS, p.r.tokens * p.share - col0);
	const Span span = span_of(p, b, col0 / p.share, (col0 + cols - 1) / p.share);
	const long long per = steps_of_split(span, p.splits);
	const long long begin = span.first + split * per, end = min(span.last, begin + per);

	// ---- the ring: a step's keys and values, 16 positions of one page
	const int page_steps = p.c.page / 16;
	long long next = begin + warp;                            // the step that the next request is for
	long long next_page = next / page_steps;
	int next_sub = (int)(next - next_page * page_steps), next_id = -1;
	auto look_up = [&]() { next_id = next < end ? __ldg(p.r.table + (long long)b * p.r.max_pages + next_page) : -1; };
	uint32_t live = 0;                                        // a bit a stage: its page is one of the cache's
	auto request = [&](int stage)
	{
		const bool there = next_id >= 0 && next_id < p.c.pages;
		live = (live & ~(1u << stage)) | ((there ? 1u : 0u) << stage);
		if (there)
		{
			const uint32_t at = four_smem(ring) + stage * stage_bytes;
			const size_t row = ((size_t)next_id * p.c.kv_heads + head) * p.c.page + next_sub * 16;
			const uint8_t * kc = p.c.k_codes + row * (dim / 2), * vc = p.c.v_codes + row * (dim / 2);
			#pragma unroll
			for (int j = 0; j < NB / 2; ++j)
			{
				const int i = j * 32 + lane;
				if (i < 16 * nb)
				{
					const uint32_t to = at + i / nb * pitch + i % nb * 16;
					copy16(to, kc + i * 16, true);
					copy16(to + 16 * pitch, vc + i * 16, true);
				}
			}
			if (lane < 8 * groups)
			{
				const int i = lane % (4 * groups);
				const char * src = (const char *)(lane < 4 * groups ? p.c.k_scales : p.c.v_scales) + row * groups * 4;
				copy16(at + 32 * pitch + lane * 16, src + i * 16, true);
			}
			if (GROUPS > 4 && lane + 32 < 8 * groups)
			{
				const int i = (lane + 32) % (4 * groups);
				const char * src = (const char *)(lane + 32 < 4 * groups ? p.c.k_scales : p.c.v_scales) + row * groups * 4;
				copy16(at + 32 * pitch + (lane + 32) * 16, src + i * 16, true);
			}
		}
		copies_close();
		next += FA_WARPS;
		next_sub += FA_WARPS;
		while (next_sub >= page_steps) { next_sub -= page_steps; ++next_page; }
		look_up();
	};
	look_up();
	#pragma unroll
	for (int i = 0; i < FA_STAGES - 1; ++i) { request(i); }

	// ---- the queries: a warp takes a column, a lane eight channels
	for (int c = warp; c < COLS; c += FA_WARPS)
	{
		const int i = (col0 + c) / p.share, h = head * p.share + (col0 + c) % p.share;
		const bool there = c < cols && i < span.count;
		float v[8] = {};
		if (there && lane < dim / 8)
		{
			load8((const T *)p.q.data + b * p.q.stride_sequence + i * p.q.stride_token + h * p.q.stride_head + lane * 8, 8, p.wide_q != 0, v);
		}
		uint32_t largest = 0;
		float part = 0.0f;
		#pragma unroll
		for (int e = 0; e < 8; ++e)
		{
			largest = max(largest, __float_as_uint(fabsf(v[e])));
			part += v[e];
		}
		largest = __reduce_max_sync(0xffffffffu, largest);
		#pragma unroll
		for (int m = 1; m < GB * 4; m <<= 1) { part += __shfl_xor_sync(0xffffffffu, part, m); }
		if (lane < dim / 8 && lane % (GB * 4) == 0) { s_qsum[lane / (GB * 4) * COLS + c] = part * p.scale_log2; }
		float factor, inverse;
		fit_f16(largest, factor, inverse);
		if (lane == 0)
		{
			s_qf[c] = inverse * (How::UNIT * p.scale_log2);
			const long long at = span.at + i;
			s_to[c] = there ? min(span.end, at + 1) : 0;
			s_from[c] = there && p.window > 0 ? max(0LL, at + 1 - p.window) : 0;
		}
		if (lane < dim / 8)
		{
			float high[8], rest[8];
			#pragma unroll
			for (int e = 0; e < 8; ++e) { split_f16(factor == 0.0f ? 0.0f : v[e] * factor * (e & 1 ? How::ODD : 1.0f), high[e], rest[e]); }
			unsigned char * at = s_q + c * q_pitch + lane * 16;
			*reinterpret_cast<uint4 *>(at) = make_uint4(pair_f16(high[0], high[4]), pair_f16(high[2], high[6]), pair_f16(high[1], high[5]), pair_f16(high[3], high[7]));
			if (QP == 2)
			{
				*reinterpret_cast<uint4 *>(at + COLS * q_pitch) = make_uint4(pair_f16(rest[0], rest[4]), pair_f16(rest[2], rest[6]), pair_f16(rest[1], rest[5]), pair_f16(rest[3], rest[7]));
			}
		}
	}
	__syncthreads();
	// Positions that every column sees: no step inside them asks again
	long long all_from = 0, all_to = LLONG_MAX;
	for (int c = 0; c < cols; ++c)
	{
		if ((col0 + c) / p.share >= span.count) { continue; }
		all_from = max(all_from, s_from[c]);
		all_to = min(all_to, s_to[c]);
	}

	float o[NB][2][NT][4] = {};                               // [block][even, odd channels][tile][channel g: columns 2t, 2t+1; channel g + 8]
	float lows[GROUPS][NT][2] = {};                           // sum(p * low_v) of this lane's positions
	float top[NT][2], total[NT][2] = {};                      // running maximum (log2), sum(p) of this lane's positions
	#pragma unroll
	for (int nt = 0; nt < NT; ++nt) { top[nt][0] = top[nt][1] = -INFINITY; }
	uint32_t unit_top = 0;                                    // scales of values up to these fp16 bits fit
	float unit = 1.0f;                                        // what p * scale_v is multiplied by: a power of two

	int stage = 0;
	for (long long step = begin + warp; step < end; step += FA_WARPS)
	{
		request((stage + FA_STAGES - 1) % FA_STAGES);
		copies_wait<FA_STAGES - 1>();
		__syncwarp();
		const unsigned char * at = ring + stage * stage_bytes;
		const bool there = live >> stage & 1;
		stage = (stage + 1) % FA_STAGES;
		if (!there) { continue; }
		const uint32_t * k_pairs = (const uint32_t *)(at + 32 * pitch), * v_pairs = k_pairs + 16 * groups;

		// ---- scores
		float s[NT][4] = {}, low_part[NT][4] = {};
		#pragma unroll
		for (int gr = 0; gr < GROUPS; ++gr)
		{
			if (gr >= groups) { continue; }
			float acc[NT][4] = {};
			#pragma unroll
			for (int j = 0; j < GB; ++j)
			{
				const int blk = gr * GB + j;
				const uint32_t w0 = *(const uint32_t *)(at + g * pitch + blk * 16 + t * 4);
				const uint32_t w1 = *(const uint32_t *)(at + (g + 8) * pitch + blk * 16 + t * 4);
				const uint32_t even[4] = {even_codes<CENTRED>(w0), even_codes<CENTRED>(w1), even_codes<CENTRED>(w0 >> 8), even_codes<CENTRED>(w1 >> 8)};
				const uint32_t odd[4] = {odd_codes<CENTRED>(w0), odd_codes<CENTRED>(w1), odd_codes<CENTRED>(w0 >> 8), odd_codes<CENTRED>(w1 >> 8)};
				#pragma unroll
				for (int nt = 0; nt < NT; ++nt)
				{
					#pragma unroll
					for (int part = 0; part < QP; ++part)
					{
						const uint4 qs = *(const uint4 *)(s_q + (part * COLS + nt * 8 + g) * q_pitch + blk * 64 + t * 16);
						mma_16816(acc[nt], even, qs.x, qs.y);
						mma_16816(acc[nt], odd, qs.z, qs.w);
					}
				}
			}
			float2 sl0 = halves(k_pairs[g * groups + gr]), sl1 = halves(k_pairs[(g + 8) * groups + gr]);
			sl0.y += How::SHIFT * sl0.x;
			sl1.y += How::SHIFT * sl1.x;
			#pragma unroll
			for (int nt = 0; nt < NT; ++nt)
			{
				const float2 qsum = *(const float2 *)(s_qsum + gr * COLS + nt * 8 + t * 2);
				s[nt][0] += sl0.x * acc[nt][0];
				s[nt][1] += sl0.x * acc[nt][1];
				s[nt][2] += sl1.x * acc[nt][2];
				s[nt][3] += sl1.x * acc[nt][3];
				low_part[nt][0] += sl0.y * qsum.x;
				low_part[nt][1] += sl0.y * qsum.y;
				low_part[nt][2] += sl1.y * qsum.x;
				low_part[nt][3] += sl1.y * qsum.y;
			}
		}
		#pragma unroll
		for (int nt = 0; nt < NT; ++nt)
		{
			const float2 qf = *(const float2 *)(s_qf + nt * 8 + t * 2);
			s[nt][0] = s[nt][0] * qf.x + low_part[nt][0];
			s[nt][1] = s[nt][1] * qf.y + low_part[nt][1];
			s[nt][2] = s[nt][2] * qf.x + low_part[nt][2];
			s[nt][3] = s[nt][3] * qf.y + low_part[nt][3];
		}

		// ---- what is not seen: neither its score nor its scales count, whatever they are
		float2 sv[GROUPS][2];
		#pragma unroll
		for (int gr = 0; gr < GROUPS; ++gr)
		{
			sv[gr][0] = gr < groups ? halves(v_pairs[g * groups + gr]) : make_float2(0.0f, 0.0f);
			sv[gr][1] = gr < groups ? halves(v_pairs[(g + 8) * groups + gr]) : make_float2(0.0f, 0.0f);
			sv[gr][0].y += How::SHIFT * sv[gr][0].x;
			sv[gr][1].y += How::SHIFT * sv[gr][1].x;
		}
		const long long pos = step * 16;
		if (pos < all_from || pos + 16 > all_to)
		{
			#pragma unroll
			for (int r = 0; r < 2; ++r)
			{
				bool any = false;
				#pragma unroll
				for (int nt = 0; nt < NT; ++nt)
				{
					#pragma unroll
					for (int e = 0; e < 2; ++e)
					{
						const int c = nt * 8 + t * 2 + e;
						const bool seen = pos + g + 8 * r >= s_from[c] && pos + g + 8 * r < s_to[c];
						s[nt][2 * r + e] = seen ? s[nt][2 * r + e] : -INFINITY;
						any |= seen;
					}
				}
				#pragma unroll
				for (int gr = 0; gr < GROUPS; ++gr)
				{
					if (!any) { sv[gr][r] = make_float2(0.0f, 0.0f); }
				}
			}
		}

		// ---- the maximum, and the unit of the values' scales, where they have to move
		bool move = false;
		#pragma unroll
		for (int nt = 0; nt < NT; ++nt)
		{
			#pragma unroll
			for (int e = 0; e < 4; ++e) { move |= !(s[nt][e] <= top[nt][e & 1] + FA_SLACK); }         // (a NaN moves it, too)
		}
		// (a scale that is not finite makes sums that are not, in any unit: it does not take the others' bits away)
		uint32_t largest = 0;
		#pragma unroll
		for (int gr = 0; gr < GROUPS; ++gr)
		{
			const uint32_t a = __float_as_uint(fabsf(sv[gr][0].x)), c = __float_as_uint(fabsf(sv[gr][1].x));
			largest = max(largest, max(a < 0x7f800000u ? a : 0, c < 0x7f800000u ? c : 0));
		}
		move |= largest > unit_top;
		if (__any_sync(0xffffffffu, move))
		{
			largest = __reduce_max_sync(0xffffffffu, largest);
			float rescale = 1.0f;
			if (largest > unit_top)
			{
				const uint32_t e = largest >> 23;
				const float now = __uint_as_float((260 - e) << 23);       // 2^(6 - (e - 127)): the largest scale comes to [2^6, 2^7)
				rescale = unit_top == 0 ? 1.0f : now / unit;
				unit = now;
				unit_top = e << 23 | 0x7fffffu;
			}
			#pragma unroll
			for (int nt = 0; nt < NT; ++nt)
			{
				#pragma unroll
				for (int e = 0; e < 2; ++e)
				{
					// a NaN counts as an infinity: that makes the column's sums NaN
					s[nt][e] = s[nt][e] != s[nt][e] ? INFINITY : s[nt][e];
					s[nt][2 + e] = s[nt][2 + e] != s[nt][2 + e] ? INFINITY : s[nt][2 + e];
					float m = fmaxf(s[nt][e], s[nt][2 + e]);
					m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
					m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
					m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
					if (m <= top[nt][e] + FA_SLACK) { m = top[nt][e]; }       // others moved theirs: a column's sums depend on its own scores alone
					const float keep = m == top[nt][e] ? 1.0f : weight_of(top[nt][e], m);
					top[nt][e] = m;
					total[nt][e] *= keep;
					#pragma unroll
					for (int gr = 0; gr < GROUPS; ++gr) { lows[gr][nt][e] *= keep; }
					#pragma unroll
					for (int blk = 0; blk < NB; ++blk)
					{
						#pragma unroll
						for (int odd = 0; odd < 2; ++odd)
						{
							o[blk][odd][nt][e] *= keep * rescale;
							o[blk][odd][nt][2 + e] *= keep * rescale;
						}
					}
				}
			}
		}

		// ---- weights: 0 for what is not seen
		float w[NT][4];
		#pragma unroll
		for (int nt = 0; nt < NT; ++nt)
		{
			#pragma unroll
			for (int e = 0; e < 4; ++e)
			{
				w[nt][e] = s[nt][e] == -INFINITY ? 0.0f : exp2_fast(s[nt][e] - top[nt][e & 1]);
				total[nt][e & 1] += w[nt][e];
			}
		}

		// ---- values
		const uint32_t pick = g < 4 ? 0x5410u : 0x7632u;      // the half of a word that holds this lane's channels
		#pragma unroll
		for (int gr = 0; gr < GROUPS; ++gr)
		{
			if (gr >= groups) { continue; }
			uint32_t pv[NT][PP][2];
			#pragma unroll
			for (int nt = 0; nt < NT; ++nt)
			{
				#pragma unroll
				for (int r = 0; r < 2; ++r)
				{
					const float scale = sv[gr][r].x * unit, wx = w[nt][2 * r], wy = w[nt][2 * r + 1];
					lows[gr][nt][0] += wx == 0.0f ? 0.0f : wx * sv[gr][r].y;
					lows[gr][nt][1] += wy == 0.0f ? 0.0f : wy * sv[gr][r].y;
					const float x = wx == 0.0f ? 0.0f : wx * scale, y = wy == 0.0f ? 0.0f : wy * scale;
					const uint32_t high = pair_f16(x, y);
					pv[nt][0][r] = transposed(high);
					if (PP == 2)
					{
						const float2 back = halves(high);
						pv[nt][PP - 1][r] = transposed(pair_f16(x - back.x, y - back.y));
					}
				}
			}
			#pragma unroll
			for (int j = 0; j < GB; ++j)
			{
				const int blk = gr * GB + j;
				const unsigned char * vw = at + 16 * pitch + 2 * t * pitch + blk * 16 + (g & 3) * 4;
				const uint32_t x = __byte_perm(*(const uint32_t *)vw, *(const uint32_t *)(vw + pitch), pick);
				const uint32_t y = __byte_perm(*(const uint32_t *)(vw + 8 * pitch), *(const uint32_t *)(vw + 9 * pitch), pick);
				const uint32_t even[4] = {even_codes<CENTRED>(x), even_codes<CENTRED>(x >> 8), even_codes<CENTRED>(y), even_codes<CENTRED>(y >> 8)};
				const uint32_t odd[4] = {odd_codes<CENTRED>(x), odd_codes<CENTRED>(x >> 8), odd_codes<CENTRED>(y), odd_codes<CENTRED>(y >> 8)};
				#pragma unroll
				for (int nt = 0; nt < NT; ++nt)
				{
					#pragma unroll
					for (int part = 0; part < PP; ++part)
					{
						mma_16816(o[blk][0][nt], even, pv[nt][part][0], pv[nt][part][1]);
						mma_16816(o[blk][1][nt], odd, pv[nt][part][0], pv[nt][part][1]);
					}
				}
			}
		}
		__syncwarp();
	}

	// ---- the warps' sums meet
	copies_wait<0>();
	__syncwarp();
	const int u_pitch = dim + 4;
	float * u = (float *)ring;                                // [column][channel]
	#pragma unroll
	for (int nt = 0; nt < NT; ++nt)
	{
		#pragma unroll
		for (int e = 0; e < 2; ++e)
		{
			float l = total[nt][e];
			#pragma unroll
			for (int m = 4; m < 32; m <<= 1) { l += __shfl_xor_sync(0xffffffffu, l, m); }
			const int c = nt * 8 + t * 2 + e;
			if (g == 0)
			{
				s_m[warp * COLS + c] = top[nt][e];
				s_l[warp * COLS + c] = l;
			}
			#pragma unroll
			for (int gr = 0; gr < GROUPS; ++gr)
			{
				float low = lows[gr][nt][e];
				#pragma unroll
				for (int m = 4; m < 32; m <<= 1) { low += __shfl_xor_sync(0xffffffffu, low, m); }
				if (gr >= groups) { continue; }
				#pragma unroll
				for (int j = 0; j < GB; ++j)
				{
					const int blk = gr * GB + j;
					float * to = u + c * u_pitch + blk * 32 + (g & 3) * 8 + (g >> 2) * 4;
					const float even = How::UNIT / unit, odd = even * How::ODD;
					to[0] = o[blk][0][nt][e] * even + low;
					to[2] = o[blk][0][nt][2 + e] * even + low;
					to[1] = o[blk][1][nt][e] * odd + low;
					to[3] = o[blk][1][nt][2 + e] * odd + low;
				}
			}
		}
	}
	__syncthreads();
	float * first_u = (float *)smem;
	const int warp_floats = FA_STAGES * stage_bytes / 4;
	for (int i = threadIdx.x; i < cols * dim; i += FA_THREADS)
	{
		const int c = i / dim, d = i - c * dim;
		float m = s_m[c];
		#pragma unroll
		for (int w = 1; w < FA_WARPS; ++w) { m = fmaxf(m, s_m[w * COLS + c]); }
		float v = 0.0f;
		#pragma unroll
		for (int w = 0; w < FA_WARPS; ++w)
		{
			const float by = weight_of(s_m[w * COLS + c], m);
			v += by == 0.0f ? 0.0f : by * first_u[w * warp_floats + c * u_pitch + d];
		}
		first_u[c * u_pitch + d] = v;
	}
	__syncthreads();
	if (threadIdx.x < COLS)
	{
		const int c = threadIdx.x;
		float m = s_m[c], l = 0.0f;
		for (int w = 1; w < FA_WARPS; ++w) { m = fmaxf(m, s_m[w * COLS + c]); }
		for (int w = 0; w < FA_WARPS; ++w) { l += s_l[w * COLS + c] * weight_of(s_m[w * COLS + c], m); }
		s_m[c] = m;
		s_l[c] = l;
	}

	// ---- the splits' sums meet
	if (p.partial != nullptr)
	{
		__syncthreads();
		if (begin >= end) { return; }
		float * to = p.partial + (((size_t)(b * p.c.kv_heads + head) * p.tiles + tile) * p.splits + split) * COLS * (dim + 2);
		for (int i = threadIdx.x; i < cols * dim; i += FA_THREADS) { to[i] = first_u[i / dim * u_pitch + i % dim]; }
		if (threadIdx.x < cols)
		{
			to[COLS * dim + threadIdx.x] = s_m[threadIdx.x];
			to[COLS * (dim + 1) + threadIdx.x] = s_l[threadIdx.x];
		}
		return;
	}
	const cg::cluster_group cluster = cg::this_cluster();
	const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
	cluster.sync();
	for (int i = rank * FA_THREADS + threadIdx.x; i < cols * dim; i += ranks * FA_THREADS)
	{
		const int c = i / dim, d = i - c * dim, row = (col0 + c) / p.share, h = head * p.share + (col0 + c) % p.share;
		float m = -INFINITY, l = 0.0f, v = 0.0f;
		for (int r = 0; r < ranks; ++r) { m = fmaxf(m, cluster.map_shared_rank(s_m, r)[c]); }
		for (int r = 0; r < ranks; ++r)
		{
			const float by = weight_of(cluster.map_shared_rank(s_m, r)[c], m);
			l += by == 0.0f ? 0.0f : by * cluster.map_shared_rank(s_l, r)[c];
			v += by == 0.0f ? 0.0f : by * cluster.map_shared_rank(first_u, r)[c * u_pitch + d];
		}
		const bool none = row >= span.count || m == -INFINITY;
		((T *)p.out.data)[b * p.out.stride_sequence + row * p.out.stride_token + h * p.out.stride_head + d] = from_f32<T>(none ? 0.0f : v / l);
		if (p.lse != nullptr && d == 0)
		{
			p.lse[((size_t)b * p.r.tokens + row) * p.heads + h] = none ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
		}
	}
	cluster.sync();                                           // nobody leaves while its sums are read
}

// One block a column: joins what the splits left.
template <class T>
__global__ void __launch_bounds__(FA_THREADS)
four_attend_join_kernel(const AttendParams p, int cols_of_tile)
{
	const int b = blockIdx.z, head = blockIdx.y, col = blockIdx.x, tile = col / cols_of_tile, c = col - tile * cols_of_tile;
	const int row = col / p.share, h = head * p.share + col % p.share, dim = p.c.dim;
	const int col0 = tile * cols_of_tile, cols = min(cols_of_tile, p.r.tokens * p.share - col0);
	const Span span = span_of(p, b, col0 / p.share, (col0 + cols - 1) / p.share);
	const long long per = steps_of_split(span, p.splits);
	const int used = (int)((span.last - span.first + per - 1) / per);
	const float * from = p.partial + ((size_t)(b * p.c.kv_heads + head) * p.tiles + tile) * p.splits * cols_of_tile * (dim + 2);
	const size_t pitch = (size_t)cols_of_tile * (dim + 2);
	float m = -INFINITY, l = 0.0f;
	for (int s = 0; s < used; ++s) { m = fmaxf(m, from[s * pitch + cols_of_tile * dim + c]); }
	for (int s = 0; s < used; ++s)
	{
		const float by = weight_of(from[s * pitch + cols_of_tile * dim + c], m);
		l += by == 0.0f ? 0.0f : by * from[s * pitch + cols_of_tile * (dim + 1) + c];
	}
	const bool none = row >= span.count || m == -INFINITY;
	for (int d = threadIdx.x; d < dim; d += FA_THREADS)
	{
		float v = 0.0f;
		for (int s = 0; s < used; ++s)
		{
			const float by = weight_of(from[s * pitch + cols_of_tile * dim + c], m);
			v += by == 0.0f ? 0.0f : by * from[s * pitch + c * dim + d];
		}
		((T *)p.out.data)[b * p.out.stride_sequence + row * p.out.stride_token + h * p.out.stride_head + d] = from_f32<T>(none ? 0.0f : v / l);
	}
	if (p.lse != nullptr && threadIdx.x == 0)
	{
		p.lse[((size_t)b * p.r.tokens + row) * p.heads + h] = none ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
	}
}

// Tiles of columns and splits of a call.
struct AttendPlan
{
	int nt, tiles, splits;
	bool cluster;
};

static AttendPlan plan_attend(const xnor_b200_kv4_cache & c, const xnor_b200_kv4_rows & r, int heads, int window)
{
	AttendPlan a;
	const long long columns = (long long)r.tokens * (heads / c.kv_heads);
	a.nt = columns > 8 && c.dim <= 128 ? 2 : 1;
	const long long tiles = (columns + a.nt * 8 - 1) / (a.nt * 8), base = tiles * c.kv_heads * r.batch;
	a.tiles = (int)(tiles < INT_MAX ? tiles : INT_MAX);
	long long most = (long long)r.max_pages * c.page;                          // positions that a tile may see
	if (window > 0 && most > (long long)window + r.tokens) { most = (long long)window + r.tokens; }
	const long long steps = (most + 15) / 16, want = 4LL * sm_count();
	long long splits = (want + base - 1) / base, room = steps / (2 * FA_WARPS);
	if (splits > room) { splits = room; }
	if (splits < 1) { splits = 1; }
	a.cluster = splits <= 8;
	if (a.cluster)
	{
		a.splits = 1;
		while (a.splits < splits) { a.splits *= 2; }
	}
	else { a.splits = (int)splits; }
	return a;
}

template <class T, int NB, int GB, int NT>
static int launch_attend(const AttendParams & p, const AttendPlan & plan, cudaStream_t stream)
{
	const int nb = p.c.dim / 32, groups = p.c.dim / p.c.group;
	const size_t smem = (size_t)FA_WARPS * FA_STAGES * attend_stage(nb, groups) + (size_t)Parts<T>::Q * NT * 8 * attend_q_pitch(nb)
			+ (size_t)NT * 8 * (4 + (NB / GB) * 4 + 16 + FA_WARPS * 8);
	const auto kernel = four_attend_kernel<T, NB, GB, NT>;
	const int rc = ensure_dynamic_smem((const void *)kernel, smem);
	if (rc != XNOR_B200_OK) { return rc; }
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = dim3((unsigned)plan.splits, (unsigned)(p.c.kv_heads * plan.tiles), (unsigned)p.r.batch);
	cfg.blockDim = dim3(FA_THREADS, 1, 1);
	cfg.dynamicSmemBytes = smem;
	cfg.stream = stream;
	cudaLaunchAttribute attr[1];
	attr[0].id = cudaLaunchAttributeClusterDimension;
	attr[0].val.clusterDim.x = plan.cluster ? (unsigned)plan.splits : 1;
	attr[0].val.clusterDim.y = 1;
	attr[0].val.clusterDim.z = 1;
	cfg.attrs = attr;
	cfg.numAttrs = 1;
	const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
	if (e != cudaSuccess) { return cuda_fail(e); }
	if (!plan.cluster)
	{
		four_attend_join_kernel<T><<<dim3((unsigned)(p.r.tokens * p.share), (unsigned)p.c.kv_heads, (unsigned)p.r.batch), FA_THREADS, 0, stream>>>(p, NT * 8);
	}
	return check_launch();
}

template <class T, int NB, int GB>
static int launch_attend_columns(const AttendParams & p, const AttendPlan & plan, cudaStream_t stream)
{
	if constexpr (NB <= 4)
	{
		if (plan.nt == 2) { return launch_attend<T, NB, GB, 2>(p, plan, stream); }
	}
	return launch_attend<T, NB, GB, 1>(p, plan, stream);
}

template <class T>
static int launch_attend_shape(const AttendParams & p, const AttendPlan & plan, cudaStream_t stream)
{
	const int d = p.c.dim, g = p.c.group;
	if (d <= 64) { return g == 32 ? launch_attend_columns<T, 2, 1>(p, plan, stream) : launch_attend_columns<T, 2, 2>(p, plan, stream); }
	if (d <= 128)
	{
		return g == 32 ? launch_attend_columns<T, 4, 1>(p, plan, stream) : g == 64 ? launch_attend_columns<T, 4, 2>(p, plan, stream)
				: launch_attend_columns<T, 4, 4>(p, plan, stream);
	}
	return g == 32 ? launch_attend_columns<T, 8, 1>(p, plan, stream) : g == 64 ? launch_attend_columns<T, 8, 2>(p, plan, stream)
			: launch_attend_columns<T, 8, 4>(p, plan, stream);
}

static int check_attend(const xnor_b200_kv4_cache * cache, const xnor_b200_kv4_rows * rows, int heads, int window)
{
	const int rc = validate_kv4(cache, rows);
	if (rc != XNOR_B200_OK) { return rc; }
	if (heads <= 0 || heads % cache->kv_heads != 0 || window < 0) { return XNOR_B200_ERR_INVALID; }
	const AttendPlan a = plan_attend(*cache, *rows, heads, window);
	if (rows->batch > 65535 || (long long)a.tiles * cache->kv_heads > 65535 || (long long)rows->tokens * (heads / cache->kv_heads) > INT_MAX) { return XNOR_B200_ERR_TOO_LARGE; }
	return XNOR_B200_OK;
}

}  // namespace xnor

using namespace xnor;

extern "C" size_t xnor_b200_kv4_attend_scratch_bytes(const xnor_b200_kv4_cache * cache, const xnor_b200_kv4_rows * rows, int heads, int window)
{
	if (check_attend(cache, rows, heads, window) != XNOR_B200_OK) { return 0; }
	const AttendPlan a = plan_attend(*cache, *rows, heads, window);
	return a.cluster ? 0 : (size_t)rows->batch * cache->kv_heads * a.tiles * a.splits * a.nt * 8 * (cache->dim + 2) * sizeof(float);
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
	p.splits = plan.splits;
	p.tiles = plan.tiles;
	p.wide_q = ((uintptr_t)q->data & 15) == 0 && q->stride_sequence * (long long)size % 16 == 0 && q->stride_token * (long long)size % 16 == 0
			&& q->stride_head * (long long)size % 16 == 0;
	const cudaStream_t s = (cudaStream_t)stream;
	switch (q->dtype)
	{
		case XNOR_B200_F32: return launch_attend_shape<float>(p, plan, s);
		case XNOR_B200_F16: return launch_attend_shape<__half>(p, plan, s);
		default: return launch_attend_shape<__nv_bfloat16>(p, plan, s);
	}
}
