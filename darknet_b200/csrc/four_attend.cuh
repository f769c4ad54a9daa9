// Attention of a few tokens of each sequence over its cached keys and values, which lie in pages of four-bit rows.
//
//   out = sum_j softmax_j(scale * q . k_j) v_j over the positions j that the token sees, its own and those before it (the last `window`)
//
// Every row of the cache is read once for all heads of queries that share it.  A query (head, token) is a column; a warp takes two steps of 16
// positions at a time, its columns eight by eight, and both products run on the tensor cores with the codes as they lie (four_common.cuh):
//   scores  [16 positions x 8 columns] = codes of k . q         then  scale_k * that + low_k * sum(q), group by group
//   out     [16 channels x 8 columns] += (codes of v - 8) . (p * scale_v), and sum(p * (low_v + 8 * scale_v)) beside it in fp32
// (around the middle code, so that the two hardly cancel).
// q and p * scale_v are fp16 next to powers of two of their own (q: of the column; p * scale_v: of the largest of the column and the group so
// far); p * scale_v is two parts, fp32 calls' q too.  The running maximum moves only when a score passes it by more than 2^8 (a published
// refinement of the running softmax), so most steps neither exchange it nor rescale.
//
// A CTA has four warps that share a run of positions, two steps by two, each with a ring of its own; then their sums meet in shared memory.
// Long sequences are split over CTAs: up to eight of them are a cluster and meet in its shared memory, more leave their sums in the
// scratch buffer and a second kernel joins them.  Everything is summed in a fixed order.
//
// What bounds it: issue slots, where a tile of columns is enough.  32 positions of 128 channels in one group take some 705 instructions of a
// warp for the 4.4 KB they come in, 176 of them the masks and shifts of the codes (on a pipe of half the rate), 32 the additions of their sums;
// one sequence of 131072 tokens, 8 heads of keys and 64 of queries, is read at 4.3 TB/s once it runs, 2.9 TB/s from launch to end (48 us; the
// copy rate is 6.5 TB/s).  Before and after its steps a CTA costs 900 instructions a warp: calls of few positions are that and a chain of four
// loads (lengths, table, codes, sums): 7.6 us.  Three tiles of columns take all registers there are, eight warps on an SM: those wait for
// one another's results (a third of the issue slots in use).  Tried and slower: five CTAs on an SM (96 registers: 50 against 45 us, of an
// earlier build), three stages (52).
#pragma once

#include <cooperative_groups.h>

#include <climits>

#include "four_common.cuh"

namespace xnor
{

namespace cg = cooperative_groups;

constexpr int FA_WARPS = 4, FA_THREADS = 32 * FA_WARPS;
constexpr int FA_STAGES = 2;
constexpr float FA_SLACK = 8.0f;                          // how far (log2) a score may pass the running maximum
constexpr int FA_MOST_UNIT = 127 + 64, FA_MOST_P = 15;     // of p * scale_v: the largest unit's exponent, and log2 of the largest product in it

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
	int room;                     // positions that a row of the table has pages for
	int wide_q, wide_out;         // rows start on 16 bytes; four channels of a row on their size
};

// What a tile of columns sees of its sequence.  Tokens of rows i0 .. i1.
struct Span
{
	int count;
	int at;                       // position of row 0
	int end;                      // positions that there are
	int first, last;              // first step of 16 positions and the one behind the last, of all columns
};

// The token that a column asks for (one token: no division; this and its like are a good part of a short call).
__device__ __forceinline__ int row_of(const AttendParams & p, int col) { return p.r.tokens == 1 ? 0 : col / p.share; }

// The first position that a token at `at` sees.
__device__ __forceinline__ int seen_from(int window, int at) { return window > 0 && at >= window ? at - window + 1 : 0; }

__device__ __forceinline__ Span span_of(const AttendParams & p, int b, int i0, int i1)
{
	Span s;
	const int count = p.r.counts != nullptr ? max(p.r.counts[b], 0) : p.r.tokens;
	s.count = min(count, p.r.tokens);
	const int length = max(p.r.lengths[b], 0);
	s.at = length - count;
	s.end = min(length, p.room);
	i1 = min(i1, s.count - 1);
	const int to = i1 < i0 ? 0 : min(s.end, s.at + i1 + 1), from = i1 < i0 ? 0 : seen_from(p.window, s.at + i0);
	s.first = from / 16;
	s.last = to > from ? (to - 1) / 16 + 1 : s.first;
	return s;
}

// Steps of one split, whole pairs for each warp: the same for the kernel and for the one that joins.
__device__ __forceinline__ int steps_of_split(const Span & s, int splits)
{
	const int n = s.last - s.first, each = splits == 1 ? n : (int)((uint32_t)(n + splits - 1) / (uint32_t)splits);
	return max((each + 1) / 2 * 2, 2 * FA_WARPS);
}

__device__ __forceinline__ float exp2_fast(float v)
{
	float r;
	asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
	return r;
}

// What the sums at maximum m count for next to those at maximum `top`
__device__ __forceinline__ float weight_of(float m, float top) { return m == -INFINITY ? 0.0f : exp2_fast(m - top); }

__device__ __forceinline__ void add_weighted(float4 & v, float by, const float4 & u)
{
	v.x += by * u.x;
	v.y += by * u.y;
	v.z += by * u.z;
	v.w += by * u.w;
}

// Four channels of a row, from its sums at maximum m and their total l.
template <class T>
__device__ __forceinline__ void write_out(const AttendParams & p, int b, int row, int head, int d, bool none, float m, float l, const float4 & v)
{
	none |= m == -INFINITY;
	T * to = (T *)p.out.data + b * p.out.stride_sequence + row * p.out.stride_token + head * p.out.stride_head + d;
	const float by = 1.0f / l;
	struct alignas(4 * sizeof(T)) Four { T v[4]; } four;
	four.v[0] = from_f32<T>(none ? 0.0f : v.x * by);
	four.v[1] = from_f32<T>(none ? 0.0f : v.y * by);
	four.v[2] = from_f32<T>(none ? 0.0f : v.z * by);
	four.v[3] = from_f32<T>(none ? 0.0f : v.w * by);
	if (p.wide_out) { *reinterpret_cast<Four *>(to) = four; }
	else
	{
		#pragma unroll
		for (int i = 0; i < 4; ++i) { to[i] = four.v[i]; }
	}
	if (p.lse != nullptr && d == 0)
	{
		p.lse[((size_t)b * p.r.tokens + row) * p.heads + head] = none ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
	}
}

__device__ __forceinline__ uint32_t transposed(uint32_t v)
{
	uint32_t r;
	asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
	return r;
}

// fp16 parts of queries and of weights times scales.  Weights of 11 bits show, in bf16 calls too: of 64 sequences' results one in ten was not
// the bf16 value next to the exact one, with two parts one in 1600 is not (a tenth of the time: 39.5 us for 35.9).
template <class T> struct Parts { static constexpr int Q = 1, P = 2; };
template <> struct Parts<float> { static constexpr int Q = 2, P = 2; };

// A stage holds 32 positions: rows of keys' codes, rows of values' codes, scales.  A lane reads GB words of a row of a group; the pitches
// put rows that are read at a time into different banks.
// CTAs that an SM holds: 128 registers a thread for most shapes, shared memory for the widest.
__host__ __device__ constexpr int attend_on_sm(int nb, int nt) { return nt >= 2 ? (nb <= 2 && nt == 2 ? 3 : 2) : nb <= 5 ? 4 : nb <= 7 ? 3 : 2; }

template <int NB, int GB, int NT, int QP>
struct AttendShape
{
	static constexpr int GROUPS = NB / GB, COLS = NT * 8;
	static constexpr int K_PITCH = (GROUPS | 1) * 16 * GB, V_PITCH = (NB | 1) * 16, Q_PITCH = (NB | 1) * 64;
	static constexpr int V_AT = 32 * K_PITCH, PAIRS_AT = V_AT + 32 * V_PITCH, STAGE = PAIRS_AT + 2 * 32 * GROUPS * 4;
	static constexpr int U_PITCH = NB * 32 + 4, WARP = FA_STAGES * STAGE > COLS * U_PITCH * 4 ? FA_STAGES * STAGE : COLS * U_PITCH * 4;
	static constexpr size_t SMEM = (size_t)FA_WARPS * WARP + QP * COLS * Q_PITCH + COLS * (4 + GROUPS * 4 + 8 + FA_WARPS * 8 + (GROUPS == 1 ? FA_WARPS * 4 + 8 : FA_WARPS * GROUPS * 4));
};

template <int W>
__device__ __forceinline__ void load_words(uint32_t (&w)[W], const void * p)
{
	if (W == 4)
	{
		const uint4 v = *(const uint4 *)p;
		w[0] = v.x; w[W / 4] = v.y; w[W / 2] = v.z; w[W - 1] = v.w;
	}
	else if (W == 2)
	{
		const uint2 v = *(const uint2 *)p;
		w[0] = v.x; w[W - 1] = v.y;
	}
	else { w[0] = *(const uint32_t *)p; }
}

// The (scale, low) pairs of a position, of all its groups.
template <int GROUPS>
__device__ __forceinline__ void load_pairs(uint32_t (&w)[GROUPS], const uint32_t * p)
{
	if constexpr (GROUPS == 1 || GROUPS == 2 || GROUPS == 4) { load_words<GROUPS>(w, p); }
	else if constexpr (GROUPS == 8)
	{
		load_words<4>(reinterpret_cast<uint32_t (&)[4]>(w[0]), p);
		load_words<4>(reinterpret_cast<uint32_t (&)[4]>(w[4]), p + 4);
	}
	else
	{
		#pragma unroll
		for (int i = 0; i < GROUPS; ++i) { w[i] = p[i]; }
	}
}

// Weights of 16 positions times the scales of a group, in the columns' units: operands of the product with the codes; `most`: the largest of
// them.  WILD: a weight of 0 counts as nothing, whatever the scale (a branch that is hardly ever taken costs less than selecting every time).
template <bool WILD, int NT, int PP>
__device__ __forceinline__ void weigh(uint32_t (&pv)[NT][PP][2], const float (&w)[NT][4], uint32_t pair0, uint32_t pair1, const float2 (&unit)[NT], __half2 & most)
{
	#pragma unroll
	for (int r = 0; r < 2; ++r)
	{
		const float scale = halves(r == 0 ? pair0 : pair1).x;
		#pragma unroll
		for (int nt = 0; nt < NT; ++nt)
		{
			const float wx = w[nt][2 * r], wy = w[nt][2 * r + 1];
			const float x = WILD && wx == 0.0f ? 0.0f : wx * unit[nt].x * scale, y = WILD && wy == 0.0f ? 0.0f : wy * unit[nt].y * scale;
			const uint32_t high = pair_f16(x, y);
			most = __hmax2(most, __habs2(as_half2(high)));
			pv[nt][0][r] = transposed(high);
			if (PP == 2)
			{
				const float2 back = halves(high);
				pv[nt][PP - 1][r] = transposed(pair_f16(x - back.x, y - back.y));
			}
		}
	}
}

// The largest |weight * scale| of 32 positions, of this lane's two columns, to 8 bits.  What is not finite makes sums that are not, in any unit:
// it does not take the others' bits away.
template <int GROUPS>
__device__ __forceinline__ float2 most_of(const float (&w)[2][4], const uint32_t (&pairs)[2][2][GROUPS], int group)
{
	float most[2] = {0.0f, 0.0f};
	#pragma unroll
	for (int i = 0; i < 8; ++i)
	{
		const float v = fabsf(w[i / 4][i % 4] * halves(pairs[i / 4][i / 2 % 2][group]).x);
		most[i & 1] = v < INFINITY ? fmaxf(most[i & 1], v) : most[i & 1];
	}
	__nv_bfloat162 both = __floats2bfloat162_rn(most[0], most[1]);
	#pragma unroll
	for (int m = 4; m < 32; m <<= 1) { both = __hmax2(both, __shfl_xor_sync(0xffffffffu, both, m)); }
	return __bfloat1622float2(both);
}

// Powers of two are handled by their exponents' bits (127: 1).
__device__ __forceinline__ int exponent_of(float v) { return (int)(__float_as_uint(v) >> 23); }
__device__ __forceinline__ float power_of(int exponent) { return exponent > 0 ? __uint_as_float((uint32_t)exponent << 23) : 0.0f; }

// The exponent of the unit that brings `most` to [2^6, 2^7), where that of `unit` would bring it to FA_MOST_P or more.
__device__ __forceinline__ int unit_for(float most, int unit)
{
	const int e = exponent_of(most);
	return e + unit >= 2 * 127 + FA_MOST_P ? 2 * 127 + 6 - e : unit;
}

// The sums of weight * (value of code 8) of 16 positions.
template <bool WILD, int NT>
__device__ __forceinline__ void weigh_lows(float (&lows)[NT][2], const float (&w)[NT][4], uint32_t pair0, uint32_t pair1)
{
	#pragma unroll
	for (int r = 0; r < 2; ++r)
	{
		const float2 sl = halves(r == 0 ? pair0 : pair1);
		const float middle = sl.y + 8.0f * sl.x;
		#pragma unroll
		for (int nt = 0; nt < NT; ++nt)
		{
			const float wx = w[nt][2 * r], wy = w[nt][2 * r + 1];
			lows[nt][0] = WILD && wx == 0.0f ? lows[nt][0] : lows[nt][0] + wx * middle;
			lows[nt][1] = WILD && wy == 0.0f ? lows[nt][1] : lows[nt][1] + wy * middle;
		}
	}
}

// NB: blocks of 32 channels.  GB: blocks of a group.  NT: tiles of eight columns.
template <class T, int NB, int GB, int NT>
__global__ void __launch_bounds__(FA_THREADS, attend_on_sm(NB, NT))
four_attend_kernel(const AttendParams p)
{
	constexpr int QP = Parts<T>::Q, PP = Parts<T>::P;
	using S = AttendShape<NB, GB, NT, QP>;
	using How = Codes<T>;
	constexpr int COLS = S::COLS, GROUPS = S::GROUPS, DIM = NB * 32;
	constexpr bool CENTRED = How::CENTRED;
	extern __shared__ __align__(128) unsigned char smem[];
	const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
	unsigned char * ring = smem + warp * S::WARP;
	unsigned char * s_q = smem + FA_WARPS * S::WARP;                                  // [part][column]
	float * s_qf = (float *)(s_q + QP * COLS * S::Q_PITCH);                           // [column]
	float * s_qsum = s_qf + COLS;                                                     // [group][column]
	int * s_from = (int *)(s_qsum + GROUPS * COLS);                                   // [column]: positions that it sees
	int * s_to = s_from + COLS;
	float * s_m = (float *)(s_to + COLS);                                             // [warp][column]
	float * s_l = s_m + FA_WARPS * COLS, * s_by = s_l + FA_WARPS * COLS;
	float * s_top = s_by + FA_WARPS * COLS, * s_all = s_top + COLS;                   // [column]
	float * s_unit = s_by + warp * GROUPS * COLS;             // [group][column], of each warp; in the room of the last three, which come when all are through

	pdl_wait();

	const int b = blockIdx.z, head = p.tiles == 1 ? blockIdx.y : blockIdx.y / p.tiles, tile = p.tiles == 1 ? 0 : blockIdx.y % p.tiles, split = blockIdx.x;
	const int col0 = tile * COLS, cols = min(COLS, p.r.tokens * p.share - col0);
	const Span span = span_of(p, b, row_of(p, col0), row_of(p, col0 + cols - 1));
	const int per = steps_of_split(span, p.splits);
	const int begin = min(span.last, span.first + split * per), end = min(span.last, begin + per);

	// ---- the ring.  A step is 16 positions of one page; a warp takes two at a time.
	const int page_steps = p.c.page / 16;
	const uint32_t ring_at = four_smem(ring);
	int next = begin + 2 * warp;                              // the step that the next request is for
	int next_page = next / page_steps, next_sub = next - next_page * page_steps;
	const int32_t * table = p.r.table + (size_t)b * p.r.max_pages;
	int next_id[2];
	auto look_up = [&]()
	{
		next_id[0] = next < end ? table[next_page] : -1;
		next_id[1] = next + 1 < end ? table[next_page + (next_sub + 1 >= page_steps)] : -1;
	};
	// what a lane copies of a step: COPIES times 16 bytes of keys' and of values' codes, and of the scales (keys' first, then values')
	constexpr int COPIES = (NB + 1) / 2, STEP_CODES = 8 * DIM, STEP_SCALES = 64 * GROUPS;       // bytes of a step in memory
	const uint8_t * const k_from = p.c.k_codes + lane * 16, * const v_from = p.c.v_codes + lane * 16;
	const char * pairs_from[GROUPS > 4 ? 2 : 1];
	uint32_t pairs_to[GROUPS > 4 ? 2 : 1], k_to[32 % NB == 0 ? 1 : COPIES], v_to[32 % NB == 0 ? 1 : COPIES];
	#pragma unroll
	for (int j = 0; j < (32 % NB == 0 ? 1 : COPIES); ++j)
	{
		const int i = j * 32 + lane;
		k_to[j] = ring_at + i / NB * S::K_PITCH + i % NB * 16;
		v_to[j] = ring_at + S::V_AT + i / NB * S::V_PITCH + i % NB * 16;
	}
	#pragma unroll
	for (int j = 0; j < (GROUPS > 4 ? 2 : 1); ++j)
	{
		const int i = j * 32 + lane, own = i - 4 * GROUPS;
		pairs_from[j] = own < 0 ? (const char *)p.c.k_scales + i * 16 : (const char *)p.c.v_scales + own * 16;
		pairs_to[j] = ring_at + S::PAIRS_AT + (own < 0 ? i : own + 8 * GROUPS) * 16;
	}
	uint32_t live = 0;                                        // a bit a step of a stage: its page is one of the cache's
	auto request = [&](int stage)
	{
		live &= ~(3u << (stage * 2));
		#pragma unroll
		for (int h = 0; h < 2; ++h)
		{
			if ((uint32_t)next_id[h] >= (uint32_t)p.c.pages) { continue; }
			live |= 1u << (stage * 2 + h);
			const int sub = h == 0 ? next_sub : next_sub + 1 >= page_steps ? 0 : next_sub + 1;
			const uint32_t step = ((uint32_t)next_id[h] * p.c.kv_heads + head) * page_steps + sub;      // (fits: a step has 128 bytes and more)
			const uint8_t * k = k_from + (size_t)step * STEP_CODES, * v = v_from + (size_t)step * STEP_CODES;
			const uint32_t at = stage * S::STAGE;
			#pragma unroll
			for (int j = 0; j < COPIES; ++j)
			{
				if ((j + 1) * 32 <= 16 * NB || j * 32 + lane < 16 * NB)
				{
					const uint32_t kt = 32 % NB == 0 ? k_to[0] + j * (32 / NB) * S::K_PITCH : k_to[32 % NB == 0 ? 0 : j];
					const uint32_t vt = 32 % NB == 0 ? v_to[0] + j * (32 / NB) * S::V_PITCH : v_to[32 % NB == 0 ? 0 : j];
					copy16(kt + at + h * 16 * S::K_PITCH, k + j * 512, true);
					copy16(vt + at + h * 16 * S::V_PITCH, v + j * 512, true);
				}
			}
			#pragma unroll
			for (int j = 0; j < (GROUPS > 4 ? 2 : 1); ++j)
			{
				if (j * 32 + lane < 8 * GROUPS) { copy16(pairs_to[j] + at + h * STEP_SCALES, pairs_from[j] + (size_t)step * STEP_SCALES, true); }
			}
		}
		copies_close();
		next += 2 * FA_WARPS;
		next_sub += 2 * FA_WARPS;
		while (next_sub >= page_steps) { next_sub -= page_steps; ++next_page; }
		look_up();
	};
	look_up();
	#pragma unroll
	for (int i = 0; i < FA_STAGES - 1; ++i) { request(i); }

	// ---- the queries: a lane takes eight channels, half a warp a column (a whole one where there are more than 128 channels)
	constexpr int SIDE = NB <= 4 ? 16 : 32;
	const int side = lane % SIDE;
	#pragma unroll
	for (int c0 = 0; c0 < COLS; c0 += FA_THREADS / SIDE)
	{
		const int c = c0 + threadIdx.x / SIDE;
		if (c0 + FA_THREADS / SIDE > COLS && c >= COLS) { break; }
		const int i = row_of(p, col0 + c), h = head * p.share + col0 + c - i * p.share;
		const bool there = c < cols && i < span.count;        // (others see nothing)
		float v[8];
		eight_f32(load8((const T *)p.q.data + b * p.q.stride_sequence + i * p.q.stride_token + h * p.q.stride_head + side * 8,
				there && side < NB * 4 ? 8 : 0, p.wide_q != 0), v);
		float most = 0.0f, part = 0.0f, factor, inverse;
		#pragma unroll
		for (int e = 0; e < 8; ++e) { most = max_nan(most, fabsf(v[e])); }
		#pragma unroll
		for (int m = 1; m < SIDE; m <<= 1) { most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, m)); }
		fit_f16(__float_as_uint(most) & 0x7fffffffu, factor, inverse);
		#pragma unroll
		for (int e = 0; e < 8; ++e)
		{
			v[e] *= factor;
			part += v[e];
		}
		#pragma unroll
		for (int m = 1; m < GB * 4; m <<= 1) { part += __shfl_xor_sync(0xffffffffu, part, m); }
		if (side < NB * 4 && side % (GB * 4) == 0) { s_qsum[side / (GB * 4) * COLS + c] = part; }
		if (side == 0)
		{
			s_qf[c] = inverse * p.scale_log2;
			s_to[c] = there ? min(span.end, span.at + i + 1) : 0;
			s_from[c] = there ? seen_from(p.window, span.at + i) : 0;
		}
		if (side < NB * 4)
		{
			float high[8], rest[8];
			#pragma unroll
			for (int e = 0; e < 8; ++e)
			{
				high[e] = v[e] * (e & 1 ? How::ODD : 1.0f);
				if (QP == 2) { split_f16(high[e], high[e], rest[e]); }
			}
			// the four lanes of a row read GB words each of a group: those of a place lie side by side
			unsigned char * at = s_q + c * S::Q_PITCH + (side / (4 * GB) * (4 * GB) + side % GB * 4 + side / GB % 4) * 16;
			*reinterpret_cast<uint4 *>(at) = make_uint4(pair_f16(high[0], high[4]), pair_f16(high[2], high[6]), pair_f16(high[1], high[5]), pair_f16(high[3], high[7]));
			if (QP == 2)
			{
				*reinterpret_cast<uint4 *>(at + COLS * S::Q_PITCH) = make_uint4(pair_f16(rest[0], rest[4]), pair_f16(rest[2], rest[6]), pair_f16(rest[1], rest[5]), pair_f16(rest[3], rest[7]));
			}
		}
	}
	__syncthreads();
	// Positions that every column of a token sees: no step inside them asks again
	const int row_first = row_of(p, col0), row_last = min(row_of(p, col0 + cols - 1), span.count - 1);
	const int all_to = min(span.end, span.at + row_first + 1), all_from = seen_from(p.window, span.at + row_last);

	float o[GROUPS][GB][2][NT][4] = {};                       // [group][word][even, odd channels][tile][channel of g: columns 2t, 2t+1; of g + 8]
	float lows[GROUPS][NT][2] = {};                           // sum(p * low_v) of this lane's positions
	// running maximum (log2; base: 0 while there is none), the scores that move it, sum(p) of this lane's positions
	float base[NT][2] = {}, limit[NT][2], total[NT][2] = {};
	#pragma unroll
	for (int nt = 0; nt < NT; ++nt) { limit[nt][0] = limit[nt][1] = -INFINITY; }
	// What p * scale_v of a group and column is multiplied by: brings the largest of those that count to 2^6 and more, so that what fp16 then
	// cuts off of any is 2^-31 of it.  No weight or scale has a say in a unit but those of the column and the group.
	for (int i = lane; i < GROUPS * COLS; i += 32) { s_unit[i] = power_of(FA_MOST_UNIT); }
	__syncwarp();
	const uint32_t pick = g < 4 ? 0x5410u : 0x7632u;          // the half of a word that holds this lane's channels

	int stage = 0;
	for (int step = begin + 2 * warp; step < end; step += 2 * FA_WARPS)
	{
		request((stage + FA_STAGES - 1) % FA_STAGES);
		copies_wait<FA_STAGES - 1>();
		__syncwarp();
		const unsigned char * at = ring + stage * S::STAGE;
		const uint32_t there = live >> (stage * 2) & 3;
		stage = (stage + 1) % FA_STAGES;
		const uint32_t * k_pairs = (const uint32_t *)(at + S::PAIRS_AT) + g * GROUPS, * v_pairs = k_pairs + 32 * GROUPS;

		// ---- scores
		float s[2][NT][4] = {};
		uint32_t sk[2][2][GROUPS];
		#pragma unroll
		for (int h = 0; h < 2; ++h)
		{
			#pragma unroll
			for (int r = 0; r < 2; ++r) { load_pairs<GROUPS>(sk[h][r], k_pairs + (h * 16 + r * 8) * GROUPS); }
		}
		#pragma unroll
		for (int gr = 0; gr < GROUPS; ++gr)
		{
			float acc[2][NT][4] = {};
			uint32_t w[2][2][GB];
			#pragma unroll
			for (int h = 0; h < 2; ++h)
			{
				#pragma unroll
				for (int r = 0; r < 2; ++r) { load_words<GB>(w[h][r], at + (h * 16 + r * 8 + g) * S::K_PITCH + gr * 16 * GB + t * 4 * GB); }
			}
			#pragma unroll
			for (int j = 0; j < GB; ++j)
			{
				uint4 qs[NT][QP];
				#pragma unroll
				for (int nt = 0; nt < NT; ++nt)
				{
					#pragma unroll
					for (int part = 0; part < QP; ++part) { qs[nt][part] = *(const uint4 *)(s_q + (part * COLS + nt * 8 + g) * S::Q_PITCH + (gr * GB + j) * 64 + t * 16); }
				}
				#pragma unroll
				for (int h = 0; h < 2; ++h)
				{
					const uint32_t w0 = w[h][0][j], w1 = w[h][1][j], w0_up = upper(w0), w1_up = upper(w1);
					const uint32_t even[4] = {even_codes<CENTRED>(w0), even_codes<CENTRED>(w1), even_codes<CENTRED>(w0_up), even_codes<CENTRED>(w1_up)};
					const uint32_t odd[4] = {odd_codes<CENTRED>(w0), odd_codes<CENTRED>(w1), odd_codes<CENTRED>(w0_up), odd_codes<CENTRED>(w1_up)};
					#pragma unroll
					for (int nt = 0; nt < NT; ++nt)
					{
						#pragma unroll
						for (int part = 0; part < QP; ++part)
						{
							mma_16816(acc[h][nt], even, qs[nt][part].x, qs[nt][part].y);
							mma_16816(acc[h][nt], odd, qs[nt][part].z, qs[nt][part].w);
						}
					}
				}
			}
			#pragma unroll
			for (int h = 0; h < 2; ++h)
			{
				float2 sl0 = halves(sk[h][0][gr]), sl1 = halves(sk[h][1][gr]);
				sl0.y += How::SHIFT * sl0.x;
				sl1.y += How::SHIFT * sl1.x;
				sl0.x *= How::UNIT;
				sl1.x *= How::UNIT;
				#pragma unroll
				for (int nt = 0; nt < NT; ++nt)
				{
					const float2 qsum = *(const float2 *)(s_qsum + gr * COLS + nt * 8 + t * 2);
					s[h][nt][0] += sl0.x * acc[h][nt][0] + sl0.y * qsum.x;
					s[h][nt][1] += sl0.x * acc[h][nt][1] + sl0.y * qsum.y;
					s[h][nt][2] += sl1.x * acc[h][nt][2] + sl1.y * qsum.x;
					s[h][nt][3] += sl1.x * acc[h][nt][3] + sl1.y * qsum.y;
				}
			}
		}
		#pragma unroll
		for (int nt = 0; nt < NT; ++nt)
		{
			const float2 qf = *(const float2 *)(s_qf + nt * 8 + t * 2);
			#pragma unroll
			for (int h = 0; h < 2; ++h)
			{
				s[h][nt][0] *= qf.x;
				s[h][nt][1] *= qf.y;
				s[h][nt][2] *= qf.x;
				s[h][nt][3] *= qf.y;
			}
		}

		// ---- what is not seen: neither its score nor its scales count, whatever they are
		uint32_t sv[2][2][GROUPS];
		#pragma unroll
		for (int h = 0; h < 2; ++h)
		{
			#pragma unroll
			for (int r = 0; r < 2; ++r) { load_pairs<GROUPS>(sv[h][r], v_pairs + (h * 16 + r * 8) * GROUPS); }
		}
		bool wild = false;                                    // a scale that one column sees and another does not is not finite
		const bool edge = step * 16 < all_from || step * 16 + 32 > all_to || there != 3;
		if (edge)
		{
			#pragma unroll
			for (int h = 0; h < 2; ++h)
			{
				#pragma unroll
				for (int r = 0; r < 2; ++r)
				{
					const int at_step = step + h, place = g + 8 * r;
					bool any = false;
					#pragma unroll
					for (int nt = 0; nt < NT; ++nt)
					{
						#pragma unroll
						for (int e = 0; e < 2; ++e)
						{
							const int c = nt * 8 + t * 2 + e;
							const bool seen = (there >> h & 1) && at_step < end && at_step * 16 + place >= s_from[c] && at_step * 16 + place < s_to[c];
							s[h][nt][2 * r + e] = seen ? s[h][nt][2 * r + e] : -INFINITY;
							any |= seen;
						}
					}
					#pragma unroll
					for (int gr = 0; gr < GROUPS; ++gr)
					{
						sv[h][r][gr] = any ? sv[h][r][gr] : 0;
						wild |= (sv[h][r][gr] & 0x7c00u) == 0x7c00u || (sv[h][r][gr] & 0x7c000000u) == 0x7c000000u;
					}
				}
			}
			wild = __any_sync(0xffffffffu, wild);
		}

		// ---- the maximum, where it has to move
		bool move = false;
		#pragma unroll
		for (int h = 0; h < 2; ++h)
		{
			#pragma unroll
			for (int nt = 0; nt < NT; ++nt)
			{
				#pragma unroll
				for (int e = 0; e < 4; ++e) { move |= !(s[h][nt][e] <= limit[nt][e & 1]); }           // (a NaN moves it, too)
			}
		}
		if (__any_sync(0xffffffffu, move))
		{
			#pragma unroll
			for (int nt = 0; nt < NT; ++nt)
			{
				float keep[2];                                    // what there is counts for that much of what it did: 2^-back down to half of that
				int back[2];
				#pragma unroll
				for (int e = 0; e < 2; ++e)
				{
					float m = -INFINITY;
					#pragma unroll
					for (int i = 0; i < 4; ++i)
					{
						// a NaN counts as an infinity: that makes the column's sums NaN
						float & v = s[i / 2][nt][i % 2 * 2 + e];
						v = v != v ? INFINITY : v;
						m = fmaxf(m, v);
					}
					m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
					m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
					m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
					// others may have moved theirs: a column's sums depend on its own scores alone
					keep[e] = 1.0f;
					back[e] = 0;
					if (m > limit[nt][e])
					{
						const bool fresh = limit[nt][e] == -INFINITY;
						keep[e] = fresh ? 0.0f : exp2_fast(base[nt][e] - m);
						back[e] = fresh ? 256 : (int)fminf(m - base[nt][e], 256.0f);
						base[nt][e] = m;
						limit[nt][e] = m + FA_SLACK;
					}
				}
				// A unit may grow as much, and the sum in it hardly changes; as far as these positions' weights let it.
				float w[2][4];
				#pragma unroll
				for (int i = 0; i < 8; ++i) { w[i / 4][i % 4] = exp2_fast(s[i / 4][nt][i % 4] - base[nt][i & 1]); }
				total[nt][0] *= keep[0];
				total[nt][1] *= keep[1];
				#pragma unroll
				for (int gr = 0; gr < GROUPS; ++gr)
				{
					const float2 most = most_of(w, sv, gr);
					float2 & unit = *(float2 *)(s_unit + gr * COLS + nt * 8 + t * 2);
					const int was[2] = {exponent_of(unit.x), exponent_of(unit.y)};
					const int now[2] = {unit_for(most.x, min(was[0] + back[0], FA_MOST_UNIT)), unit_for(most.y, min(was[1] + back[1], FA_MOST_UNIT))};
					const float by[2] = {keep[0] * power_of(127 + now[0] - was[0]), keep[1] * power_of(127 + now[1] - was[1])};
					__syncwarp();
					unit = make_float2(power_of(now[0]), power_of(now[1]));       // (the same from the eight lanes of a column)
					#pragma unroll
					for (int i = 0; i < GB * 8; ++i) { o[gr][i / 8][i / 4 % 2][nt][i % 4] *= by[i & 1]; }
					lows[gr][nt][0] *= keep[0];
					lows[gr][nt][1] *= keep[1];
				}
			}
			__syncwarp();
		}

		// ---- weights: 0 for what is not seen
		#pragma unroll
		for (int h = 0; h < 2; ++h)
		{
			#pragma unroll
			for (int nt = 0; nt < NT; ++nt)
			{
				#pragma unroll
				for (int e = 0; e < 4; ++e)
				{
					s[h][nt][e] = exp2_fast(s[h][nt][e] - base[nt][e & 1]);
					total[nt][e & 1] += s[h][nt][e];
				}
			}
		}

		// ---- values.  The tensor cores cut a sum off where fp32 rounds it, which adds up over a long run (60000 positions of codes 2 to 4: 3e-6
		// of what goes into the sums, and half a percent of the results): the products of 32 positions go into sums that start at 0, and those
		// are added to the others by fp32 additions.
		#pragma unroll
		for (int gr = 0; gr < GROUPS; ++gr)
		{
			uint32_t pv[2][NT][PP][2];
			{
				float2 unit[NT];
				#pragma unroll
				for (int nt = 0; nt < NT; ++nt) { unit[nt] = *(const float2 *)(s_unit + gr * COLS + nt * 8 + t * 2); }
				__half2 most = as_half2(0);
				#pragma unroll
				for (int h = 0; h < 2; ++h)
				{
					if (wild) { weigh<true, NT, PP>(pv[h], s[h], sv[h][0][gr], sv[h][1][gr], unit, most); }
					else { weigh<false, NT, PP>(pv[h], s[h], sv[h][0][gr], sv[h][1][gr], unit, most); }
				}
				const bool over = __half2float(__hmax(__low2half(most), __high2half(most))) >= (float)(1 << FA_MOST_P);
				if (__any_sync(0xffffffffu, over))
				{
					#pragma unroll
					for (int nt = 0; nt < NT; ++nt)
					{
						float w[2][4];
						#pragma unroll
						for (int i = 0; i < 8; ++i) { w[i / 4][i % 4] = s[i / 4][nt][i % 4]; }
						const float2 most = most_of(w, sv, gr);
						const int was[2] = {exponent_of(unit[nt].x), exponent_of(unit[nt].y)}, now[2] = {unit_for(most.x, was[0]), unit_for(most.y, was[1])};
						const float by[2] = {power_of(127 + now[0] - was[0]), power_of(127 + now[1] - was[1])};
						unit[nt] = make_float2(power_of(now[0]), power_of(now[1]));
						__syncwarp();
						*(float2 *)(s_unit + gr * COLS + nt * 8 + t * 2) = unit[nt];
						#pragma unroll
						for (int i = 0; i < GB * 8; ++i) { o[gr][i / 8][i / 4 % 2][nt][i % 4] *= by[i & 1]; }
					}
					__syncwarp();
					#pragma unroll
					for (int h = 0; h < 2; ++h) { weigh<true, NT, PP>(pv[h], s[h], sv[h][0][gr], sv[h][1][gr], unit, most); }
				}
			}
			#pragma unroll
			for (int h = 0; h < 2; ++h)
			{
				if (wild) { weigh_lows<true, NT>(lows[gr], s[h], sv[h][0][gr], sv[h][1][gr]); }
				else { weigh_lows<false, NT>(lows[gr], s[h], sv[h][0][gr], sv[h][1][gr]); }
			}
			constexpr int WORDS = GB == 4 ? 1 : GB;               // of a row at a time (131072 positions: 47.4 us, with all four, that spill, 49)
			#pragma unroll
			for (int j0 = 0; j0 < GB; j0 += WORDS)
			{
				uint32_t w[2][4][WORDS];
				#pragma unroll
				for (int h = 0; h < 2; ++h)
				{
					#pragma unroll
					for (int i = 0; i < 4; ++i)
					{
						load_words<WORDS>(w[h][i], at + S::V_AT + (h * 16 + i / 2 * 8 + i % 2 + 2 * t) * S::V_PITCH + gr * 16 * GB + (g & 3) * 4 * GB + j0 * 4);
					}
				}
				#pragma unroll
				for (int j = 0; j < WORDS; ++j)
				{
					float of_step[2][NT][4];                      // [even, odd channels]
					#pragma unroll
					for (int h = 0; h < 2; ++h)
					{
						const uint32_t x = __byte_perm(w[h][0][j], w[h][1][j], pick), y = __byte_perm(w[h][2][j], w[h][3][j], pick), x_up = upper(x), y_up = upper(y);
						const uint32_t even[4] = {even_codes<true>(x), even_codes<true>(x_up), even_codes<true>(y), even_codes<true>(y_up)};
						const uint32_t odd[4] = {odd_codes<true>(x), odd_codes<true>(x_up), odd_codes<true>(y), odd_codes<true>(y_up)};
						#pragma unroll
						for (int nt = 0; nt < NT; ++nt)
						{
							#pragma unroll
							for (int part = 0; part < PP; ++part)
							{
								if (h + part == 0)
								{
									mma_16816_first(of_step[0][nt], even, pv[h][nt][part][0], pv[h][nt][part][1]);
									mma_16816_first(of_step[1][nt], odd, pv[h][nt][part][0], pv[h][nt][part][1]);
								}
								else
								{
									mma_16816(of_step[0][nt], even, pv[h][nt][part][0], pv[h][nt][part][1]);
									mma_16816(of_step[1][nt], odd, pv[h][nt][part][0], pv[h][nt][part][1]);
								}
							}
						}
					}
					#pragma unroll
					for (int nt = 0; nt < NT; ++nt)
					{
						#pragma unroll
						for (int e = 0; e < 4; ++e)
						{
							o[gr][j0 + j][0][nt][e] += of_step[0][nt][e];
							o[gr][j0 + j][1][nt][e] += of_step[1][nt][e];
						}
					}
				}
			}
		}
		__syncwarp();
	}

	// The next kernel (the one that joins, too) may be launched once every CTA is through its steps.  Before, its CTAs would fill the SMs that
	// are done first, and go to work on those alone (64 sequences of up to 2048 tokens, one call behind the other, an earlier build: 40 us, 36
	// from here).
	pdl_trigger();

	// ---- the warps' sums meet
	copies_wait<0>();
	__syncwarp();
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
				s_m[warp * COLS + c] = limit[nt][e] == -INFINITY ? -INFINITY : base[nt][e];
				s_l[warp * COLS + c] = l;
			}
			#pragma unroll
			for (int gr = 0; gr < GROUPS; ++gr)
			{
				float low = lows[gr][nt][e];
				#pragma unroll
				for (int m = 4; m < 32; m <<= 1) { low += __shfl_xor_sync(0xffffffffu, low, m); }
				const float by = power_of(2 * 127 - exponent_of(s_unit[gr * COLS + c]));
				#pragma unroll
				for (int j = 0; j < GB; ++j)
				{
					float4 * to = (float4 *)(u + c * S::U_PITCH + (gr * 4 * GB + (g & 3) * GB + j) * 8 + (g >> 2) * 4);
					const auto & even = o[gr][j][0][nt], & odd = o[gr][j][1][nt];
					*to = make_float4(even[e] * by + low, odd[e] * by + low, even[2 + e] * by + low, odd[2 + e] * by + low);
				}
			}
		}
	}
	__syncthreads();
	// per column: what each warp's sums count for, the maximum and the total of all
	if (threadIdx.x < COLS)
	{
		const int c = threadIdx.x;
		float m = s_m[c], l = 0.0f;
		#pragma unroll
		for (int w = 1; w < FA_WARPS; ++w) { m = fmaxf(m, s_m[w * COLS + c]); }
		float by[FA_WARPS];
		#pragma unroll
		for (int w = 0; w < FA_WARPS; ++w)
		{
			by[w] = weight_of(s_m[w * COLS + c], m);
			l += by[w] == 0.0f ? 0.0f : by[w] * s_l[w * COLS + c];
		}
		#pragma unroll
		for (int w = 0; w < FA_WARPS; ++w) { s_by[w * COLS + c] = by[w]; }
		s_top[c] = m;
		s_all[c] = l;
	}
	__syncthreads();
	float * first_u = (float *)smem;
	constexpr int WARP_FLOATS = S::WARP / 4, quads = DIM / 4;
	const bool joined = p.partial == nullptr;
	float * partial = joined ? nullptr : p.partial + (((size_t)(b * p.c.kv_heads + head) * p.tiles + tile) * p.splits + split) * COLS * (DIM + 4);
	for (int c = threadIdx.x / quads, q = threadIdx.x % quads; c < cols; c += FA_THREADS / quads)
	{
		if (threadIdx.x >= FA_THREADS / quads * quads) { break; }
		float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
		#pragma unroll
		for (int w = 0; w < FA_WARPS; ++w)
		{
			// (what counts for nothing has seen nothing: its sums are 0)
			add_weighted(v, s_by[w * COLS + c], *(const float4 *)(first_u + w * WARP_FLOATS + c * S::U_PITCH + q * 4));
		}
		if (joined && p.splits == 1)
		{
			const int row = row_of(p, col0 + c);
			write_out<T>(p, b, row, head * p.share + col0 + c - row * p.share, q * 4, row >= span.count, s_top[c], s_all[c], v);
		}
		else if (joined) { *(float4 *)(first_u + c * S::U_PITCH + q * 4) = v; }
		else if (begin < end) { *(float4 *)(partial + c * DIM + q * 4) = v; }
	}

	// ---- the splits' sums meet
	if (!joined)
	{
		if (threadIdx.x < cols && begin < end)
		{
			partial[COLS * DIM + threadIdx.x] = s_top[threadIdx.x];
			partial[COLS * (DIM + 1) + threadIdx.x] = s_all[threadIdx.x];
		}
		return;
	}
	if (p.splits == 1) { return; }
	const cg::cluster_group cluster = cg::this_cluster();
	const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
	cluster.sync();
	for (int i = rank * FA_THREADS + threadIdx.x; i < cols * quads; i += ranks * FA_THREADS)
	{
		const int c = i / quads, q = i - c * quads, row = row_of(p, col0 + c), h = head * p.share + col0 + c - row * p.share;
		float m = -INFINITY, l = 0.0f;
		float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
		for (int r = 0; r < ranks; ++r) { m = fmaxf(m, cluster.map_shared_rank(s_top, r)[c]); }
		for (int r = 0; r < ranks; ++r)
		{
			const float by = weight_of(cluster.map_shared_rank(s_top, r)[c], m);
			if (by == 0.0f) { continue; }
			l += by * cluster.map_shared_rank(s_all, r)[c];
			add_weighted(v, by, *(const float4 *)(cluster.map_shared_rank(first_u, r) + c * S::U_PITCH + q * 4));
		}
		write_out<T>(p, b, row, h, q * 4, row >= span.count, m, l, v);
	}
	cluster.sync();                                           // nobody leaves while its sums are read
}

// Joins what the splits left, a block a column: what each split counts for is worked out once, then every warp adds up every eighth split,
// whose loads are all on their way at once.  Starts while the splits are still at work (its launch would take as long as its work).
constexpr int FJ_WARPS = 8, FJ_THREADS = 32 * FJ_WARPS, FJ_SPLITS = 1024;

template <class T>
__global__ void __launch_bounds__(FJ_THREADS)
four_attend_join_kernel(const AttendParams p, int cols_of_tile)
{
	pdl_wait();
	pdl_trigger();
	const int dim = p.c.dim, quads = dim / 4, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
	const int b = blockIdx.z, head = blockIdx.y, col = blockIdx.x, tile = col / cols_of_tile, c = col - tile * cols_of_tile;
	const int row = row_of(p, col), h = head * p.share + col - row * p.share;
	const int col0 = tile * cols_of_tile, cols = min(cols_of_tile, p.r.tokens * p.share - col0);
	const Span span = span_of(p, b, row_of(p, col0), row_of(p, col0 + cols - 1));
	const int per = steps_of_split(span, p.splits), used = (span.last - span.first + per - 1) / per;
	const size_t pitch = (size_t)cols_of_tile * (dim + 4);
	const float * from = p.partial + ((size_t)(b * p.c.kv_heads + head) * p.tiles + tile) * p.splits * pitch;
	const float * tops = from + cols_of_tile * dim + c, * totals = tops + cols_of_tile;
	__shared__ float s_by[FJ_SPLITS], s_m[FJ_WARPS], s_l[FJ_WARPS];
	__shared__ float4 s_v[FJ_WARPS][64];

	float m = -INFINITY, l = 0.0f;
	for (int s = threadIdx.x; s < used; s += FJ_THREADS)
	{
		const float top = tops[s * pitch];
		s_by[s] = top;
		m = fmaxf(m, top);
	}
	#pragma unroll
	for (int i = 1; i < 32; i <<= 1) { m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i)); }
	if (lane == 0) { s_m[warp] = m; }
	__syncthreads();
	#pragma unroll
	for (int w = 0; w < FJ_WARPS; ++w) { m = fmaxf(m, s_m[w]); }
	for (int s = threadIdx.x; s < used; s += FJ_THREADS)
	{
		const float by = weight_of(s_by[s], m);
		s_by[s] = by;
		l += by == 0.0f ? 0.0f : by * totals[s * pitch];
	}
	#pragma unroll
	for (int i = 1; i < 32; i <<= 1) { l += __shfl_xor_sync(0xffffffffu, l, i); }
	if (lane == 0) { s_l[warp] = l; }
	__syncthreads();
	float4 v[2] = {};
	#pragma unroll 8
	for (int s = warp; s < used; s += FJ_WARPS)
	{
		#pragma unroll
		for (int j = 0; j < 2; ++j)
		{
			if (lane + j * 32 < quads) { add_weighted(v[j], s_by[s], *(const float4 *)(from + s * pitch + c * dim + (lane + j * 32) * 4)); }
		}
	}
	s_v[warp][lane] = v[0];
	s_v[warp][lane + 32] = v[1];
	__syncthreads();
	for (int q = threadIdx.x; q < quads; q += FJ_THREADS)
	{
		l = 0.0f;
		float4 all = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
		#pragma unroll
		for (int w = 0; w < FJ_WARPS; ++w)
		{
			l += s_l[w];
			add_weighted(all, 1.0f, s_v[w][q]);
		}
		write_out<T>(p, b, row, h, q * 4, row >= span.count, m, l, all);
	}
}

// Tiles of columns and splits of a call.
struct AttendPlan
{
	int nt, tiles, splits;
	bool cluster;
};

template <class T, int NB, int GB, int NT>
static int launch_attend(const AttendParams & p, const AttendPlan & plan, cudaStream_t stream)
{
	constexpr size_t smem = AttendShape<NB, GB, NT, Parts<T>::Q>::SMEM;
	const auto kernel = four_attend_kernel<T, NB, GB, NT>;
	const int rc = ensure_dynamic_smem((const void *)kernel, smem);
	if (rc != XNOR_B200_OK) { return rc; }
	const int done = launch_four(kernel, dim3((unsigned)plan.splits, (unsigned)(p.c.kv_heads * plan.tiles), (unsigned)p.r.batch), FA_THREADS, smem,
			plan.cluster ? (unsigned)plan.splits : 1, stream, p);
	if (done != XNOR_B200_OK || plan.cluster) { return done; }
	return launch_four(four_attend_join_kernel<T>, dim3((unsigned)(p.r.tokens * p.share), (unsigned)p.c.kv_heads, (unsigned)p.r.batch), FJ_THREADS, 0, 1,
			stream, p, NT * 8);
}

template <class T, int NB, int GB>
static int launch_attend_columns(const AttendParams & p, const AttendPlan & plan, cudaStream_t stream)
{
	if constexpr (NB <= 4)
	{
		if (plan.nt == 2) { return launch_attend<T, NB, GB, 2>(p, plan, stream); }
		if (plan.nt == 3) { return launch_attend<T, NB, GB, 3>(p, plan, stream); }
	}
	return launch_attend<T, NB, GB, 1>(p, plan, stream);
}

// The kernel for a call's shape.
template <class T>
int launch_attend_shape(const AttendParams & p, const AttendPlan & plan, cudaStream_t stream)
{
	switch (p.c.dim / 32 * 8 + p.c.group / 32)                // (a group divides the dimension)
	{
		case 1 * 8 + 1: return launch_attend_columns<T, 1, 1>(p, plan, stream);
		case 2 * 8 + 1: return launch_attend_columns<T, 2, 1>(p, plan, stream);
		case 2 * 8 + 2: return launch_attend_columns<T, 2, 2>(p, plan, stream);
		case 3 * 8 + 1: return launch_attend_columns<T, 3, 1>(p, plan, stream);
		case 4 * 8 + 1: return launch_attend_columns<T, 4, 1>(p, plan, stream);
		case 4 * 8 + 2: return launch_attend_columns<T, 4, 2>(p, plan, stream);
		case 4 * 8 + 4: return launch_attend_columns<T, 4, 4>(p, plan, stream);
		case 5 * 8 + 1: return launch_attend_columns<T, 5, 1>(p, plan, stream);
		case 6 * 8 + 1: return launch_attend_columns<T, 6, 1>(p, plan, stream);
		case 6 * 8 + 2: return launch_attend_columns<T, 6, 2>(p, plan, stream);
		case 7 * 8 + 1: return launch_attend_columns<T, 7, 1>(p, plan, stream);
		case 8 * 8 + 1: return launch_attend_columns<T, 8, 1>(p, plan, stream);
		case 8 * 8 + 2: return launch_attend_columns<T, 8, 2>(p, plan, stream);
		default: return launch_attend_columns<T, 8, 4>(p, plan, stream);
	}
}

// One translation unit a type (four_attend_f32.cu and its like), which takes a third of the time to compile.
int launch_attend_f32(const AttendParams & p, const AttendPlan & plan, cudaStream_t stream);
int launch_attend_f16(const AttendParams & p, const AttendPlan & plan, cudaStream_t stream);
int launch_attend_bf16(const AttendParams & p, const AttendPlan & plan, cudaStream_t stream);

}  // namespace xnor
