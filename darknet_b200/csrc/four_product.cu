// Products of a few rows with a 4-bit matrix: out[r][i] = act( sum_j x[r][j] * (low[i][j/g] + scale[i][j/g] * code[i][j]) + bias[i] ).
//
// forward_connected_layer of Darknet (src-lib/connected_layer.cpp) with packed weights, one to some sixteen rows.  A group's sum is
// scale * sum(x * code) + low * sum(x): the codes go into the tensor cores as they lie (four_common.cuh), and scale and low come in once a
// group.  x is converted once a block of 256 neighbours, to fp16 next to a power of two of the block's own (fp32: to two fp16 parts,
// multiplied one after the other), which loses nothing of a 16-bit x down
// to some 2^-26 of the block's largest value, and next to nothing of that value below (fit_f16).
//
// A CTA has eight warps of 16 or 32 filters and a slice of the neighbours; each warp copies its own codes into a ring of its own, so that
// only the conversion of x, a turn ahead, is waited for.  The slices of the same filters are a cluster: their sums meet in shared memory, in
// a fixed order, so results do not vary.
//
// What bounds it: one row of 16384 x 16384 runs at 4.1 TB/s in bf16 (34.8 us; the copy rate is 6.5 TB/s), 3.7 in fp16 (38.1), 16 rows of bf16
// at 3.0 (47.6 us).  No unit is full (integer pipe 46 and 34 %, tensor pipe 23 and 38 %, issue slots 56 and 44 %, DRAM 42 and 35 %): 256 CTAs
// on 132 of 148 SMs with one or two steps of codes on their way, that come to a barrier every block.  Tried and slower by 16 rows: seven
// warps, whose 74 clusters do not fit at a time (66 us), barriers every other block with twice the room for x (52).  Up to 4096 x 4096
// (8 MB from the L2, 6 us) it is a chain of latencies: launch, x, codes, the cluster's sums.
#include <cooperative_groups.h>

#include <climits>

#include "four_common.cuh"

namespace xnor
{

namespace cg = cooperative_groups;

constexpr int FP_K = 256;                                 // neighbours of a block: one power of two for x, one step of the ring
constexpr int FP_X_BYTES = FP_K * 2 + 64;                 // a row's block of x: the pitch puts neighbouring rows 16 banks apart
constexpr int FP_CODE_PITCH = FP_K / 2;                   // a filter's block of codes

struct ProductParams
{
	const uint8_t * codes;
	const uint32_t * scales;      // (scale, low) pairs
	const void * x;
	const float * biases;
	void * out;
	long long ldx, ldo;
	int n, k, rows, leaky, wide;
	int row_bytes, groups;        // of one filter
	int slice;                    // blocks of 256 of one CTA of a cluster
	int steps;                    // of a warp's ring
	const unsigned char * ready;  // x as the kernel holds it in shared memory, made beforehand: [tile of rows][block of 256]
};

// NT: tiles of eight rows.  MT: tiles of 16 filters of a warp.  XB: blocks of x converted at a time.  READY: x was converted by a kernel
// of its own (four_x_kernel).
template <class T, int NT, int MT, int WARPS, int GROUP, int XB>
struct ProductShape
{
	static constexpr int PARTS = sizeof(T) == 4 ? 2 : 1, ROWS = NT * 8, THREADS = 32 * WARPS, FILTERS = 16 * MT * WARPS;
	static constexpr int GROUPS = FP_K / GROUP, SCALE_PITCH = GROUPS + 1;             // words; odd, so that eight filters lie in eight banks
	static constexpr int CODE_BYTES = 16 * MT * FP_CODE_PITCH, STEP_BYTES = CODE_BYTES + 16 * MT * SCALE_PITCH * 4;
	static constexpr int TASKS = (XB * ROWS + WARPS - 1) / WARPS;                     // rows' blocks that a warp converts
	// a buffer of x: [XB][part][row] blocks, [XB][row] powers of two, [XB][group][row] sums; behind the two of them a block of zeros,
	// which the columns of rows that are not there read
	__host__ __device__ static constexpr int x_bytes(int rows) { return XB * PARTS * rows * FP_X_BYTES; }
	__host__ __device__ static constexpr int buffer_bytes(int rows) { return x_bytes(rows) + XB * ROWS * 4 * (1 + GROUPS); }
	static size_t smem(int rows, int steps)
	{
		const size_t all = (size_t)WARPS * steps * STEP_BYTES + 2 * buffer_bytes(rows) + FP_X_BYTES, sums = (size_t)ROWS * (FILTERS + 1) * 4;
		return all > sums ? all : sums;
	}
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

// A row's block of 256 to its place in a buffer of x (a warp, a lane eight neighbours): fp16 parts, the power of two, the groups' sums.
template <class T, int GROUP, int ROWS>
__device__ __forceinline__ void convert_row(const Eight<T> & raw, unsigned char * buffer, int xb, int x_rows, int row, unsigned char * numbers, int blocks, int lane)
{
	using How = Codes<T>;
	constexpr int PARTS = sizeof(T) == 4 ? 2 : 1, W = GROUP / 32, GROUPS = FP_K / GROUP;
	float * inverses = (float *)numbers, * sums = inverses + blocks * ROWS;
	float v[8];
	eight_f32(raw, v);
	float most[4];                                                // (pairs of pairs: these chains are what a short call waits for)
	#pragma unroll
	for (int e = 0; e < 4; ++e) { most[e] = max_nan(fabsf(v[e]), fabsf(v[e + 4])); }
	most[0] = max_nan(max_nan(most[0], most[1]), max_nan(most[2], most[3]));
	const uint32_t largest = __reduce_max_sync(0xffffffffu, __float_as_uint(most[0]) & 0x7fffffffu);
	float factor, inverse;
	fit_f16(largest, factor, inverse);
	if (lane == 0) { inverses[xb * ROWS + row] = inverse; }
	// (what is not finite makes its own column of the products NaN, and the inverse does so anyway)
	float high[8], rest[8];
	#pragma unroll
	for (int e = 0; e < 8; ++e)
	{
		v[e] *= factor;
		high[e] = v[e] * (e & 1 ? How::ODD : 1.0f);
		if (PARTS == 2) { split_f16(high[e], high[e], rest[e]); }
	}
	// the sum at that power of two (that of the largest values passes fp32's range)
	float part = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
	#pragma unroll
	for (int m = 1; m < GROUP / 8; m <<= 1) { part += __shfl_xor_sync(0xffffffffu, part, m); }
	if (lane % (GROUP / 8) == 0) { sums[(xb * GROUPS + lane / (GROUP / 8)) * ROWS + row] = part; }
	unsigned char * at = buffer + (xb * PARTS * x_rows + row) * FP_X_BYTES + (lane / (4 * W) * (4 * W) + lane % W * 4 + lane / W % 4) * 16;
	*reinterpret_cast<uint4 *>(at) = make_uint4(pair_f16(high[0], high[4]), pair_f16(high[2], high[6]), pair_f16(high[1], high[5]), pair_f16(high[3], high[7]));
	if (PARTS == 2)
	{
		*reinterpret_cast<uint4 *>(at + x_rows * FP_X_BYTES) = make_uint4(pair_f16(rest[0], rest[4]), pair_f16(rest[2], rest[6]), pair_f16(rest[1], rest[5]), pair_f16(rest[3], rest[7]));
	}
}

// x converted once for all CTAs of a large product: a block of 256 neighbours of a tile of rows a CTA, as buffer_bytes() lays it out.
template <class T, int NT, int GROUP>
__global__ void __launch_bounds__(256)
four_x_kernel(const ProductParams p, unsigned char * ready)
{
	using S = ProductShape<T, NT, 2, 8, GROUP, 1>;
	const int row0 = blockIdx.y * S::ROWS, rows = min(S::ROWS, p.rows - row0), x_rows = min(S::ROWS, p.rows), lane = threadIdx.x % 32;
	unsigned char * buffer = ready + ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * S::buffer_bytes(x_rows);
	pdl_wait();
	pdl_trigger();                                            // the product may be launched; it waits for this kernel's end
	for (int row = threadIdx.x / 32; row < rows; row += 8)
	{
		const int k0 = blockIdx.x * FP_K + lane * 8;
		convert_row<T, GROUP, S::ROWS>(load8((const T *)p.x + (k0 < p.k ? (row0 + row) * p.ldx + k0 : 0), p.k - k0, p.wide != 0), buffer, 0, x_rows, row,
				buffer + S::x_bytes(x_rows), 1, lane);
	}
}

template <class T, int NT, int MT, int WARPS, int GROUP, int XB, bool READY>
__global__ void __launch_bounds__(32 * WARPS, 16 / WARPS)
four_product_kernel(const ProductParams p)
{
	using S = ProductShape<T, NT, MT, WARPS, GROUP, XB>;
	using How = Codes<T>;
	constexpr bool CENTRED = How::CENTRED;
	constexpr int PARTS = S::PARTS, ROWS = S::ROWS, GROUPS = S::GROUPS, W = GROUP / 32, WARP_FILTERS = 16 * MT;
	extern __shared__ __align__(128) unsigned char smem[];
	const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
	const cg::cluster_group cluster = cg::this_cluster();
	const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
	const int cta_filter = (blockIdx.x / ranks) * S::FILTERS, filter0 = cta_filter + warp * WARP_FILTERS;
	const int row0 = blockIdx.y * ROWS, rows = min(ROWS, p.rows - row0), x_rows = min(ROWS, p.rows);
	const int first = rank * p.slice, last = min(first + p.slice, (p.k + FP_K - 1) / FP_K);      // blocks of 256
	unsigned char * ring = smem + warp * p.steps * S::STEP_BYTES;
	unsigned char * buffers = smem + WARPS * p.steps * S::STEP_BYTES;
	const uint32_t ring_at = four_smem(ring);

	// Codes: a lane copies 16 bytes of every fourth filter.  Filters that are not there read the last one's, and are never stored.  In
	// shared memory the four lanes of a filter read W words each of a group: places are exchanged by the filter's number, so that the
	// filters that are read at a time lie in different banks.
	int ask = first, ask_stage = 0;
	const int my_byte = lane % 8 * 16, my_place = my_byte ^ (W == 4 ? lane / 8 % 2 * 64 : W == 2 ? lane / 8 * 32 : lane / 8 * 16);
	const uint8_t * code_from[4 * MT];
	#pragma unroll
	for (int j = 0; j < 4 * MT; ++j)
	{
		code_from[j] = p.codes + (size_t)min(filter0 + j * 4 + lane / 8, p.n - 1) * p.row_bytes + min(first * (FP_K / 2) + my_byte, p.row_bytes - 16);
	}
	constexpr int SCALE_COPIES = WARP_FILTERS * GROUPS / 32;
	const uint32_t * scale_from = p.scales + (size_t)min(filter0 + lane / GROUPS, p.n - 1) * p.groups + lane % GROUPS;
	auto request = [&]()
	{
		if (ask < last)
		{
			const uint32_t at = ring_at + ask_stage * S::STEP_BYTES, to = at + lane / 8 * FP_CODE_PITCH;
			const bool there = ask * (FP_K / 2) + my_byte < p.row_bytes;
			const int on = ask * (FP_K / 2) + my_byte + FP_K / 2 < p.row_bytes ? FP_K / 2 : 0;       // stays inside the filter
			#pragma unroll
			for (int j = 0; j < 4 * MT; ++j)
			{
				copy16(to + j * 4 * FP_CODE_PITCH + (W == 1 && j % 2 ? my_place ^ 64 : my_place), code_from[j], there);
				code_from[j] += on;
			}
			const bool there_group = ask * GROUPS + lane % GROUPS < p.groups;
			#pragma unroll
			for (int j = 0; j < SCALE_COPIES; ++j)
			{
				constexpr int EACH = 32 / GROUPS;             // filters that the lanes take at a time
				const uint32_t * from = scale_from + ask * GROUPS + (size_t)max(0, min(j * EACH, p.n - 1 - filter0 - lane / GROUPS)) * p.groups;
				copy4(at + S::CODE_BYTES + ((j * EACH + lane / GROUPS) * S::SCALE_PITCH + lane % GROUPS) * 4, there_group ? from : p.scales, there_group);
			}
			++ask;
			ask_stage = ask_stage + 1 == p.steps ? 0 : ask_stage + 1;
		}
		copies_close();
	};

	// x: a warp takes a row's block of 256, a lane eight neighbours; loaded a chunk ahead, converted when the chunk before is through
	Eight<T> raw[S::TASKS];
	auto load_x = [&](int chunk)
	{
		#pragma unroll
		for (int i = 0; i < S::TASKS; ++i)
		{
			const int task = i * WARPS + warp, xb = task / rows, row = task - xb * rows, k0 = (chunk + xb) * FP_K + lane * 8;
			const bool there = xb < XB && chunk + xb < last;
			raw[i] = load8((const T *)p.x + (there ? (row0 + row) * p.ldx + k0 : 0), there ? p.k - k0 : 0, p.wide != 0);
		}
	};
	auto convert_x = [&](int chunk, unsigned char * buffer)
	{
		#pragma unroll
		for (int i = 0; i < S::TASKS; ++i)
		{
			const int task = i * WARPS + warp, xb = task / rows, row = task - xb * rows;
			if (xb >= XB || chunk + xb >= last) { continue; }
			convert_row<T, GROUP, ROWS>(raw[i], buffer, xb, x_rows, row, buffer + S::x_bytes(x_rows), XB, lane);
		}
	};

	// x that was made beforehand: copied with the codes of its block
	auto copy_x = [&](int block, unsigned char * buffer)
	{
		const unsigned char * from = p.ready + ((size_t)blockIdx.y * ((p.k + FP_K - 1) / FP_K) + block) * S::buffer_bytes(x_rows);
		for (int i = threadIdx.x * 16; i < S::buffer_bytes(x_rows); i += S::THREADS * 16) { copy16(four_smem(buffer) + i, from + i, true); }
	};

	// (READY: this kernel's predecessor is four_x_kernel, which lets it start behind everything that wrote the weights)
	if (!READY)
	{
		pdl_wait();
		pdl_trigger();
		load_x(first);
	}
	for (int i = 0; i < p.steps - 1; ++i) { request(); }
	if (READY)
	{
		pdl_wait();
		pdl_trigger();
		if (first < last) { copy_x(first, buffers); }
		copies_close();
	}
	uint32_t * zeros = (uint32_t *)(buffers + 2 * S::buffer_bytes(x_rows));
	for (int i = threadIdx.x; i < FP_X_BYTES / 4; i += S::THREADS) { zeros[i] = 0; }
	if (!READY) { convert_x(first, buffers); }

	float sum[MT][NT][4] = {};
	int stage = 0, which = 0;
	for (int chunk = first; chunk < last; chunk += XB)
	{
		if (READY) { copies_wait<0>(); }
		__syncthreads();                                      // this chunk's x is there, and nobody reads the buffer of the one before
		const unsigned char * buffer = buffers + which * S::buffer_bytes(x_rows);
		which ^= 1;
		if (chunk + XB < last)
		{
			if (READY) { copy_x(chunk + 1, buffers + which * S::buffer_bytes(x_rows)); }
			else { load_x(chunk + XB); }
		}
		const float * inverses = (const float *)(buffer + S::x_bytes(x_rows)), * sums = inverses + XB * ROWS;
		#pragma unroll 1
		for (int xb = 0; xb < XB && chunk + xb < last; ++xb)
		{
			request();
			// of the copies asked for so far (a step each), all but the last steps - 1 have to be there
			if (!READY)
			{
				if (p.steps == 3) { copies_wait<2>(); }
				else { copies_wait<1>(); }
			}
			__syncwarp();
			const unsigned char * step = ring + stage * S::STEP_BYTES;
			stage = stage + 1 == p.steps ? 0 : stage + 1;
			const unsigned char * mine = step + g * FP_CODE_PITCH;
			const int place = t * W * 4 ^ (W == 4 ? g % 2 * 64 : W == 2 ? g % 4 * 32 : g * 16);
			const uint32_t * pairs = (const uint32_t *)(step + S::CODE_BYTES) + g * S::SCALE_PITCH;
			const unsigned char * x_from[NT][PARTS];
			#pragma unroll
			for (int nt = 0; nt < NT; ++nt)
			{
				#pragma unroll
				for (int part = 0; part < PARTS; ++part)
				{
					const bool there = nt * 8 + g < rows;
					x_from[nt][part] = (there ? buffer + ((xb * PARTS + part) * x_rows + nt * 8 + g) * FP_X_BYTES : (const unsigned char *)zeros) + t * 16;
				}
			}
			float of_block[MT][NT][4] = {};
			#pragma unroll
			for (int q = 0; q < GROUPS; ++q)
			{
				float acc[MT][NT][4] = {};
				uint32_t w[MT][2][W];
				#pragma unroll
				for (int mt = 0; mt < MT; ++mt)
				{
					#pragma unroll
					for (int r = 0; r < 2; ++r) { load_words<W>(w[mt][r], mine + (mt * 16 + r * 8) * FP_CODE_PITCH + (place ^ q * (GROUP / 2))); }
				}
				#pragma unroll
				for (int j = 0; j < W; ++j)
				{
					uint4 xs[NT][PARTS];
					#pragma unroll
					for (int nt = 0; nt < NT; ++nt)
					{
						#pragma unroll
						for (int part = 0; part < PARTS; ++part) { xs[nt][part] = *(const uint4 *)(x_from[nt][part] + (q * W + j) * 64); }
					}
					#pragma unroll
					for (int mt = 0; mt < MT; ++mt)
					{
						const uint32_t w0 = w[mt][0][j], w1 = w[mt][1][j], w0_up = upper(w0), w1_up = upper(w1);
						const uint32_t even[4] = {even_codes<CENTRED>(w0), even_codes<CENTRED>(w1), even_codes<CENTRED>(w0_up), even_codes<CENTRED>(w1_up)};
						const uint32_t odd[4] = {odd_codes<CENTRED>(w0), odd_codes<CENTRED>(w1), odd_codes<CENTRED>(w0_up), odd_codes<CENTRED>(w1_up)};
						#pragma unroll
						for (int nt = 0; nt < NT; ++nt)
						{
							#pragma unroll
							for (int part = 0; part < PARTS; ++part)
							{
								mma_16816(acc[mt][nt], even, xs[nt][part].x, xs[nt][part].y);
								mma_16816(acc[mt][nt], odd, xs[nt][part].z, xs[nt][part].w);
							}
						}
					}
				}
				#pragma unroll
				for (int mt = 0; mt < MT; ++mt)
				{
					float2 sl0 = halves(pairs[mt * 16 * S::SCALE_PITCH + q]), sl1 = halves(pairs[(mt * 16 + 8) * S::SCALE_PITCH + q]);
					sl0.y += How::SHIFT * sl0.x;
					sl1.y += How::SHIFT * sl1.x;
					sl0.x *= How::UNIT;
					sl1.x *= How::UNIT;
					#pragma unroll
					for (int nt = 0; nt < NT; ++nt)
					{
						const float2 xsum = *(const float2 *)(sums + (xb * GROUPS + q) * ROWS + nt * 8 + t * 2);
						of_block[mt][nt][0] = fmaf(sl0.x, acc[mt][nt][0], fmaf(sl0.y, xsum.x, of_block[mt][nt][0]));
						of_block[mt][nt][1] = fmaf(sl0.x, acc[mt][nt][1], fmaf(sl0.y, xsum.y, of_block[mt][nt][1]));
						of_block[mt][nt][2] = fmaf(sl1.x, acc[mt][nt][2], fmaf(sl1.y, xsum.x, of_block[mt][nt][2]));
						of_block[mt][nt][3] = fmaf(sl1.x, acc[mt][nt][3], fmaf(sl1.y, xsum.y, of_block[mt][nt][3]));
					}
				}
			}
			#pragma unroll
			for (int nt = 0; nt < NT; ++nt)
			{
				const float2 inverse = *(const float2 *)(inverses + xb * ROWS + nt * 8 + t * 2);
				#pragma unroll
				for (int mt = 0; mt < MT; ++mt)
				{
					sum[mt][nt][0] += inverse.x * of_block[mt][nt][0];
					sum[mt][nt][1] += inverse.y * of_block[mt][nt][1];
					sum[mt][nt][2] += inverse.x * of_block[mt][nt][2];
					sum[mt][nt][3] += inverse.y * of_block[mt][nt][3];
				}
			}
			__syncwarp();
		}
		if (!READY && chunk + XB < last) { convert_x(chunk + XB, buffers + which * S::buffer_bytes(x_rows)); }
	}

	// Columns of rows that are not there hold what shared memory held: never stored.
	copies_wait<0>();
	__syncthreads();
	float * s_out = (float *)smem;                                                    // [row][filters of the CTA + 1]
	constexpr int PITCH = S::FILTERS + 1;
	#pragma unroll
	for (int mt = 0; mt < MT; ++mt)
	{
		#pragma unroll
		for (int nt = 0; nt < NT; ++nt)
		{
			#pragma unroll
			for (int e = 0; e < 4; ++e) { s_out[(nt * 8 + t * 2 + (e & 1)) * PITCH + warp * WARP_FILTERS + mt * 16 + g + (e >> 1) * 8] = sum[mt][nt][e]; }
		}
	}
	cluster.sync();
	const int share = (S::FILTERS + ranks - 1) / ranks;                               // this CTA finishes some of the filters
	for (int i = threadIdx.x; i < rows * share; i += S::THREADS)
	{
		const int row = i / share, f = rank * share + i % share, filter = cta_filter + f;
		if (f >= S::FILTERS || filter >= p.n) { continue; }
		float v = 0.0f;
		for (int r = 0; r < ranks; ++r) { v += cluster.map_shared_rank(s_out, r)[row * PITCH + f]; }
		if (p.biases != nullptr) { v += p.biases[filter]; }
		if (p.leaky && !(v > 0.0f)) { v *= 0.1f; }
		((T *)p.out)[(row0 + row) * p.ldo + filter] = from_f32<T>(v);
	}
	cluster.sync();                                                                   // nobody leaves while its sums are read
}

// Large products of many rows: every CTA would convert all of x again, a fifth of its work.  By 16 rows of bf16 in groups of 128, us with a
// kernel for that / without: 2^24 weights 11.8 / 9.4, 2^26 18.3 / 19.4, 12288 x 8192 33.6 / 40.5, 2^27 27.5 / 32, 2^28 47.5 / 57 (groups of 32:
// 2^26 24.2 / 23.7, 12288 x 8192 48.9 / 47.8, 2^27 41 / 43, 2^28 74 / 80).  fp32 rows, whose parts are twice as much to copy, gain nothing:
// 8192 x 8192 by 12 rows 38 against 26.
static bool wants_ready(int n, int k, int dtype, int rows)
{
	return rows > 8 && dtype != XNOR_B200_F32 && (long long)n * k >= (1LL << 27);
}

template <class T, int NT, int MT, int WARPS, int GROUP, bool READY>
static int launch_product(ProductParams & p, void * scratch, cudaStream_t stream)
{
	constexpr int XB = NT == 1 && !READY ? 2 : 1;
	using S = ProductShape<T, NT, MT, WARPS, GROUP, XB>;
	const int tiles = (p.n + S::FILTERS - 1) / S::FILTERS, blocks = (p.k + FP_K - 1) / FP_K;
	const auto kernel = four_product_kernel<T, NT, MT, WARPS, GROUP, XB, READY>;
	// Slices: as few blocks as possible one after the other, with two CTAs on an SM at a time (and shared memory for two: two steps of
	// 256 filters, three of 128).  Clusters of 5 and 7 find fewer places.
	int ranks = 1, best = INT_MAX;
	for (const int r : {1, 2, 3, 4, 6, 8})
	{
		const long long waves = ((long long)tiles * r + 2 * sm_count() - 1) / (2 * sm_count());
		const long long cost = waves * ((blocks + r - 1) / r);
		if (r <= blocks && cost < best)
		{
			best = (int)cost;
			ranks = r;
		}
	}
	p.steps = MT == 2 ? 2 : 3;
	p.slice = (blocks + ranks - 1) / ranks;
	if (p.slice < p.steps) { p.steps = 2; }
	const size_t smem = S::smem(p.rows < S::ROWS ? p.rows : S::ROWS, p.steps);
	const int rc = ensure_dynamic_smem((const void *)kernel, smem);
	if (rc != XNOR_B200_OK) { return rc; }
	const unsigned row_tiles = (unsigned)((p.rows + NT * 8 - 1) / (NT * 8));
	if (READY)
	{
		p.ready = (const unsigned char *)scratch;
		const int x_rc = launch_four(four_x_kernel<T, NT, GROUP>, dim3((unsigned)blocks, row_tiles), 256, 0, 1, stream, p, (unsigned char *)scratch);
		if (x_rc != XNOR_B200_OK) { return x_rc; }
	}
	return launch_four(kernel, dim3((unsigned)(tiles * ranks), row_tiles), S::THREADS, smem, (unsigned)ranks, stream, p);
}

template <class T, int NT, int GROUP>
static int launch_product_shape(ProductParams & p, int dtype, void * scratch, cudaStream_t stream)
{
	if constexpr (sizeof(T) == 2)
	{
		if constexpr (NT == 2)
		{
			if (wants_ready(p.n, p.k, dtype, p.rows)) { return launch_product<T, NT, 2, 8, GROUP, true>(p, scratch, stream); }
		}
		// 256 filters of a CTA share its x and its loads of x, 128 fill the SMs where there are few, and are all that the registers of fp32
		// rows and the sums of small groups leave room for (us with 256 / 128, one row of bf16: 16384 x 16384 34.8 / 40.4, 8192 x 8192
		// 13.0 / 14.2, 4096 x 4096 7.4 / 6.2; groups of 32, 4096 x 16384 by 8 rows 17.4 / 16.9; fp32, 8192 x 8192 by 12 rows 28 / 26)
		const int blocks = (p.k + FP_K - 1) / FP_K;
		if constexpr (GROUP > 32)
		{
			if ((long long)((p.n + 255) / 256) * (blocks < 8 ? blocks : 8) >= 256) { return launch_product<T, NT, 2, 8, GROUP, false>(p, scratch, stream); }
		}
	}
	return launch_product<T, NT, 1, 8, GROUP, false>(p, scratch, stream);
}

template <class T, int NT>
static int launch_product_group(ProductParams & p, int dtype, int group, void * scratch, cudaStream_t stream)
{
	switch (group)
	{
		case 32: return launch_product_shape<T, NT, 32>(p, dtype, scratch, stream);
		case 64: return launch_product_shape<T, NT, 64>(p, dtype, scratch, stream);
		default: return launch_product_shape<T, NT, 128>(p, dtype, scratch, stream);
	}
}

template <class T>
static int launch_product_rows(ProductParams & p, int dtype, int group, void * scratch, cudaStream_t stream)
{
	if (p.rows <= 8) { return launch_product_group<T, 1>(p, dtype, group, scratch, stream); }
	return launch_product_group<T, 2>(p, dtype, group, scratch, stream);
}

// Bytes of one block of x of a tile of 16 rows as the kernel holds it.
static size_t ready_bytes(int group, int rows)
{
	const int x_rows = rows < 16 ? rows : 16;
	return (size_t)x_rows * FP_X_BYTES + 16 * 4 * (1 + FP_K / group);
}

}  // namespace xnor

using namespace xnor;

static int check_product(const xnor_b200_w4_desc * d, int dtype, int rows)
{
	if (d == nullptr) { return XNOR_B200_ERR_NULL; }
	if (d->n <= 0 || d->k <= 0 || !four_group_ok(d->group) || (d->activation != XNOR_B200_LINEAR && d->activation != XNOR_B200_LEAKY)
			|| !four_dtype_ok(dtype) || rows <= 0) { return XNOR_B200_ERR_INVALID; }
	if (d->k > XNOR_B200_W4_MAX_K || rows > XNOR_B200_W4_MAX_ROWS || d->n > XNOR_B200_W4_MAX_N) { return XNOR_B200_ERR_TOO_LARGE; }
	return XNOR_B200_OK;
}

extern "C" size_t xnor_b200_w4_scratch_bytes(const xnor_b200_w4_desc * d, int dtype, int rows)
{
	if (check_product(d, dtype, rows) != XNOR_B200_OK || !wants_ready(d->n, d->k, dtype, rows)) { return 0; }
	return (size_t)((rows + 15) / 16) * ((d->k + FP_K - 1) / FP_K) * ready_bytes(d->group, rows);
}

extern "C" int xnor_b200_w4_forward(const xnor_b200_w4_desc * d, const void * x, int dtype, int rows, long long ldx, const uint8_t * codes,
		const void * scales, const float * biases, void * output, long long ldo, void * scratch, size_t scratch_bytes, void * stream)
{
	if (d == nullptr || x == nullptr || codes == nullptr || scales == nullptr || output == nullptr) { return XNOR_B200_ERR_NULL; }
	const int rc = check_product(d, dtype, rows);
	if (rc != XNOR_B200_OK) { return rc; }
	if (ldx < 0 || ldo < d->n) { return XNOR_B200_ERR_INVALID; }
	const size_t size = four_size(dtype);
	if (((uintptr_t)codes & 15) != 0 || ((uintptr_t)scales & 3) != 0 || ((uintptr_t)biases & 3) != 0 || ((uintptr_t)x & (size - 1)) != 0
			|| ((uintptr_t)output & (size - 1)) != 0) { return XNOR_B200_ERR_ALIGNMENT; }
	if (wants_ready(d->n, d->k, dtype, rows))
	{
		if (scratch == nullptr) { return XNOR_B200_ERR_NULL; }
		if (scratch_bytes < xnor_b200_w4_scratch_bytes(d, dtype, rows)) { return XNOR_B200_ERR_SCRATCH; }
		if (((uintptr_t)scratch & 15) != 0) { return XNOR_B200_ERR_ALIGNMENT; }
	}
	ProductParams p = {};
	p.codes = codes;
	p.scales = (const uint32_t *)scales;
	p.x = x;
	p.biases = biases;
	p.out = output;
	p.ldx = ldx;
	p.ldo = ldo;
	p.n = d->n;
	p.k = d->k;
	p.rows = rows;
	p.leaky = d->activation == XNOR_B200_LEAKY;
	p.wide = ((uintptr_t)x & 15) == 0 && ldx * (long long)size % 16 == 0;
	p.row_bytes = (int)four_row_bytes(d->k);
	p.groups = (d->k + d->group - 1) / d->group;
	const cudaStream_t s = (cudaStream_t)stream;
	switch (dtype)
	{
		case XNOR_B200_F32: return launch_product_rows<float>(p, dtype, d->group, scratch, s);
		case XNOR_B200_F16: return launch_product_rows<__half>(p, dtype, d->group, scratch, s);
		default: return launch_product_rows<__nv_bfloat16>(p, dtype, d->group, scratch, s);
	}
}
