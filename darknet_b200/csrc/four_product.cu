// Products of a few rows with a 4-bit matrix: out[r][i] = act( sum_j x[r][j] * (low[i][j/g] + scale[i][j/g] * code[i][j]) + bias[i] ).
//
// forward_connected_layer of Darknet (src-lib/connected_layer.cpp) with packed weights, one to some sixteen rows.  Bound by the codes'
// way from memory.  A group's sum is scale * sum(x * code) + low * sum(x): the codes go into the tensor cores as they lie
// (four_common.cuh), a warp owning 16 filters, and scale and low come in once a group.  x is converted once a block of 256 neighbours, to
// fp16 next to a power of two of the block's own (fp32: to two fp16 parts, multiplied one after the other), which loses nothing of a
// 16-bit x.
//
// A CTA has four warps, 64 filters, and a slice of the neighbours; each warp copies its own codes into a ring of its own, so warps wait
// for nobody.  The slices of the same filters are a cluster: their sums meet in shared memory, in a fixed order, so results do not vary.
#include <cooperative_groups.h>

#include "four_common.cuh"

namespace xnor
{

namespace cg = cooperative_groups;

constexpr int FP_WARPS = 4, FP_THREADS = 32 * FP_WARPS, FP_ROWS = 16 * FP_WARPS;
constexpr int FP_K = 256;                                 // neighbours of a block: one power of two for x, one step of the ring
constexpr int FP_STEPS = 6;                               // steps of a warp's ring
constexpr int FP_CODE_BYTES = 16 * FP_K / 2;              // a step's codes of a warp
constexpr int FP_SCALE_PITCH = FP_K / 32 + 1;             // words; odd, so that eight filters lie in eight banks
constexpr int FP_STEP_BYTES = FP_CODE_BYTES + 16 * FP_SCALE_PITCH * 4;
constexpr int FP_X_BYTES = FP_K * 2 + 64;                 // a row's block of x: the pitch puts neighbouring rows 16 banks apart

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
};

// NT: tiles of eight rows.  XB: blocks of x in shared memory at a time.
template <class T, int NT, int GROUP, int XB>
__global__ void __launch_bounds__(FP_THREADS)
four_product_kernel(const ProductParams p)
{
	constexpr int PARTS = sizeof(T) == 4 ? 2 : 1, ROWS = NT * 8, GROUPS = FP_K / GROUP, GROUP_BLOCKS = GROUP / 32;
	using How = Codes<T>;
	constexpr bool CENTRED = How::CENTRED;
	extern __shared__ __align__(128) unsigned char smem[];
	unsigned char * s_x = smem + FP_WARPS * FP_STEPS * FP_STEP_BYTES;                 // [XB][part][row][FP_X_BYTES]
	float * s_inverse = (float *)(s_x + XB * PARTS * ROWS * FP_X_BYTES);              // [XB][row]
	float * s_sum = s_inverse + XB * ROWS;                                            // [XB][group][row]
	const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
	const cg::cluster_group cluster = cg::this_cluster();
	const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
	const int filter0 = (blockIdx.x / ranks) * FP_ROWS + warp * 16;
	const int row0 = blockIdx.y * ROWS, rows = min(ROWS, p.rows - row0);
	const int first = rank * p.slice, last = min(first + p.slice, (p.k + FP_K - 1) / FP_K);      // blocks of 256
	unsigned char * ring = smem + warp * FP_STEPS * FP_STEP_BYTES;
	const uint32_t ring_at = four_smem(ring);

	auto request = [&](int block)
	{
		if (block < last)
		{
			const uint32_t at = ring_at + (block - first) % FP_STEPS * FP_STEP_BYTES;
			#pragma unroll
			for (int j = 0; j < 4; ++j)
			{
				const int r = j * 4 + lane / 8, c = lane % 8, byte = block * (FP_K / 2) + c * 16;
				const bool there = filter0 + r < p.n && byte < p.row_bytes;
				copy16(at + r * 128 + ((c ^ (r & 7)) * 16), p.codes + (there ? (size_t)(filter0 + r) * p.row_bytes + byte : 0), there);
			}
			#pragma unroll
			for (int i = lane; i < 16 * GROUPS; i += 32)
			{
				const int r = i / GROUPS, q = i % GROUPS, group = block * GROUPS + q;
				const bool there = filter0 + r < p.n && group < p.groups;
				copy4(at + FP_CODE_BYTES + (r * FP_SCALE_PITCH + q) * 4, p.scales + (there ? (size_t)(filter0 + r) * p.groups + group : 0), there);
			}
		}
		copies_close();
	};
	#pragma unroll
	for (int i = 0; i < FP_STEPS - 1; ++i) { request(first + i); }

	float sum[NT][4] = {};
	for (int chunk = first; chunk < last; chunk += XB)
	{
		if (chunk != first) { __syncthreads(); }
		// x: a warp takes a row's block of 256, a lane eight neighbours
		const int blocks = min(XB, last - chunk);
		for (int i = warp; i < blocks * rows; i += FP_WARPS)
		{
			const int xb = i / rows, row = i - xb * rows, k0 = (chunk + xb) * FP_K + lane * 8;
			float v[8];
			const int there = min(8, p.k - k0);
			if (there > 0) { load8((const T *)p.x + (row0 + row) * p.ldx + k0, there, p.wide != 0, v); }
			else
			{
				#pragma unroll
				for (int e = 0; e < 8; ++e) { v[e] = 0.0f; }
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
			for (int m = 1; m < GROUP / 8; m <<= 1) { part += __shfl_xor_sync(0xffffffffu, part, m); }
			if (lane % (GROUP / 8) == 0) { s_sum[(xb * GROUPS + lane / (GROUP / 8)) * ROWS + row] = part; }
			float factor, inverse;
			fit_f16(largest, factor, inverse);
			if (lane == 0) { s_inverse[xb * ROWS + row] = inverse * How::UNIT; }
			float high[8], rest[8];
			#pragma unroll
			for (int e = 0; e < 8; ++e)
			{
				const float f = factor == 0.0f ? 0.0f : v[e] * factor * (e & 1 ? How::ODD : 1.0f);
				split_f16(f, high[e], rest[e]);
			}
			unsigned char * at = s_x + ((xb * PARTS) * ROWS + row) * FP_X_BYTES + lane * 16;
			*reinterpret_cast<uint4 *>(at) = make_uint4(pair_f16(high[0], high[4]), pair_f16(high[2], high[6]), pair_f16(high[1], high[5]), pair_f16(high[3], high[7]));
			if (PARTS == 2)
			{
				*reinterpret_cast<uint4 *>(at + ROWS * FP_X_BYTES) = make_uint4(pair_f16(rest[0], rest[4]), pair_f16(rest[2], rest[6]), pair_f16(rest[1], rest[5]), pair_f16(rest[3], rest[7]));
			}
		}
		__syncthreads();
		for (int xb = 0; xb < blocks; ++xb)
		{
			request(chunk + xb + FP_STEPS - 1);
			copies_wait<FP_STEPS - 1>();
			__syncwarp();
			const unsigned char * step = ring + (chunk + xb - first) % FP_STEPS * FP_STEP_BYTES;
			const uint32_t * pairs = (const uint32_t *)(step + FP_CODE_BYTES);
			float of_block[NT][4] = {};
			#pragma unroll
			for (int q = 0; q < GROUPS; ++q)
			{
				float acc[NT][4] = {};
				#pragma unroll
				for (int j = 0; j < GROUP_BLOCKS; ++j)
				{
					const int b = q * GROUP_BLOCKS + j;
					const uint32_t w0 = *(const uint32_t *)(step + g * 128 + ((b ^ g) * 16) + t * 4);
					const uint32_t w1 = *(const uint32_t *)(step + (g + 8) * 128 + ((b ^ g) * 16) + t * 4);
					const uint32_t even[4] = {even_codes<CENTRED>(w0), even_codes<CENTRED>(w1), even_codes<CENTRED>(w0 >> 8), even_codes<CENTRED>(w1 >> 8)};
					const uint32_t odd[4] = {odd_codes<CENTRED>(w0), odd_codes<CENTRED>(w1), odd_codes<CENTRED>(w0 >> 8), odd_codes<CENTRED>(w1 >> 8)};
					#pragma unroll
					for (int nt = 0; nt < NT; ++nt)
					{
						#pragma unroll
						for (int part = 0; part < PARTS; ++part)
						{
							uint4 xs = make_uint4(0, 0, 0, 0);
							if (nt * 8 + g < rows)
							{
								xs = *(const uint4 *)(s_x + ((xb * PARTS + part) * ROWS + nt * 8 + g) * FP_X_BYTES + (b * 4 + t) * 16);
							}
							mma_16816(acc[nt], even, xs.x, xs.y);
							mma_16816(acc[nt], odd, xs.z, xs.w);
						}
					}
				}
				float2 sl0 = halves(pairs[g * FP_SCALE_PITCH + q]), sl1 = halves(pairs[(g + 8) * FP_SCALE_PITCH + q]);
				sl0.y += How::SHIFT * sl0.x;
				sl1.y += How::SHIFT * sl1.x;
				#pragma unroll
				for (int nt = 0; nt < NT; ++nt)
				{
					const float2 xsum = *(const float2 *)(s_sum + (xb * GROUPS + q) * ROWS + nt * 8 + t * 2);
					of_block[nt][0] += sl0.x * acc[nt][0];
					of_block[nt][1] += sl0.x * acc[nt][1];
					of_block[nt][2] += sl1.x * acc[nt][2];
					of_block[nt][3] += sl1.x * acc[nt][3];
					sum[nt][0] += sl0.y * xsum.x;
					sum[nt][1] += sl0.y * xsum.y;
					sum[nt][2] += sl1.y * xsum.x;
					sum[nt][3] += sl1.y * xsum.y;
				}
			}
			#pragma unroll
			for (int nt = 0; nt < NT; ++nt)
			{
				const float2 inverse = *(const float2 *)(s_inverse + xb * ROWS + nt * 8 + t * 2);
				sum[nt][0] += inverse.x * of_block[nt][0];
				sum[nt][1] += inverse.y * of_block[nt][1];
				sum[nt][2] += inverse.x * of_block[nt][2];
				sum[nt][3] += inverse.y * of_block[nt][3];
			}
			__syncwarp();
		}
	}

	// Columns of rows that are not there hold what shared memory held: never stored.
	copies_wait<0>();
	__syncthreads();
	float * s_out = (float *)smem;                                                    // [row][64 filters + 1]
	constexpr int PITCH = FP_ROWS + 1;
	#pragma unroll
	for (int nt = 0; nt < NT; ++nt)
	{
		#pragma unroll
		for (int e = 0; e < 4; ++e) { s_out[(nt * 8 + t * 2 + (e & 1)) * PITCH + warp * 16 + g + (e >> 1) * 8] = sum[nt][e]; }
	}
	cluster.sync();
	const int share = FP_ROWS / ranks;                                                // this CTA finishes some of the 64 filters
	for (int i = threadIdx.x; i < rows * share; i += FP_THREADS)
	{
		const int row = i / share, f = rank * share + i % share, filter = (blockIdx.x / ranks) * FP_ROWS + f;
		if (filter >= p.n) { continue; }
		float v = 0.0f;
		for (int r = 0; r < ranks; ++r) { v += cluster.map_shared_rank(s_out, r)[row * PITCH + f]; }
		if (p.biases != nullptr) { v += __ldg(p.biases + filter); }
		if (p.leaky && !(v > 0.0f)) { v *= 0.1f; }
		((T *)p.out)[(row0 + row) * p.ldo + filter] = from_f32<T>(v);
	}
	cluster.sync();                                                                   // nobody leaves while its sums are read
}

template <class T, int NT, int GROUP>
static int launch_product(ProductParams & p, cudaStream_t stream)
{
	constexpr int PARTS = sizeof(T) == 4 ? 2 : 1, XB = 4 / NT / PARTS < 1 ? 1 : 4 / NT / PARTS;
	const int tiles = (p.n + FP_ROWS - 1) / FP_ROWS, blocks = (p.k + FP_K - 1) / FP_K;
	int ranks = 1;
	while (ranks < 8 && tiles * ranks < 4 * sm_count() && blocks >= 2 * ranks) { ranks *= 2; }
	p.slice = (blocks + ranks - 1) / ranks;
	const size_t smem = (size_t)FP_WARPS * FP_STEPS * FP_STEP_BYTES + (size_t)XB * PARTS * NT * 8 * FP_X_BYTES
			+ (size_t)XB * NT * 8 * 4 * (1 + FP_K / GROUP);
	const auto kernel = four_product_kernel<T, NT, GROUP, XB>;
	const int rc = ensure_dynamic_smem((const void *)kernel, smem);
	if (rc != XNOR_B200_OK) { return rc; }
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = dim3((unsigned)(tiles * ranks), (unsigned)((p.rows + NT * 8 - 1) / (NT * 8)), 1);
	cfg.blockDim = dim3(FP_THREADS, 1, 1);
	cfg.dynamicSmemBytes = smem;
	cfg.stream = stream;
	cudaLaunchAttribute attr[1];
	attr[0].id = cudaLaunchAttributeClusterDimension;
	attr[0].val.clusterDim.x = (unsigned)ranks;
	attr[0].val.clusterDim.y = 1;
	attr[0].val.clusterDim.z = 1;
	cfg.attrs = attr;
	cfg.numAttrs = 1;
	const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
	return e == cudaSuccess ? check_launch() : cuda_fail(e);
}

template <class T, int NT>
static int launch_product_group(ProductParams & p, int group, cudaStream_t stream)
{
	switch (group)
	{
		case 32: return launch_product<T, NT, 32>(p, stream);
		case 64: return launch_product<T, NT, 64>(p, stream);
		default: return launch_product<T, NT, 128>(p, stream);
	}
}

template <class T>
static int launch_product_rows(ProductParams & p, int group, cudaStream_t stream)
{
	if (p.rows <= 8) { return launch_product_group<T, 1>(p, group, stream); }
	return launch_product_group<T, 2>(p, group, stream);
}

}  // namespace xnor

using namespace xnor;

extern "C" int xnor_b200_w4_forward(const xnor_b200_w4_desc * d, const void * x, int dtype, int rows, long long ldx, const uint8_t * codes,
		const void * scales, const float * biases, void * output, long long ldo, void * stream)
{
	if (d == nullptr || x == nullptr || codes == nullptr || scales == nullptr || output == nullptr) { return XNOR_B200_ERR_NULL; }
	if (d->n <= 0 || d->k <= 0 || !four_group_ok(d->group) || (d->activation != XNOR_B200_LINEAR && d->activation != XNOR_B200_LEAKY)
			|| !four_dtype_ok(dtype) || rows <= 0 || ldx < 0 || ldo < d->n) { return XNOR_B200_ERR_INVALID; }
	if (d->k > XNOR_B200_W4_MAX_K || rows > XNOR_B200_W4_MAX_ROWS || d->n > XNOR_B200_W4_MAX_N) { return XNOR_B200_ERR_TOO_LARGE; }
	const size_t size = four_size(dtype);
	if (((uintptr_t)codes & 15) != 0 || ((uintptr_t)scales & 3) != 0 || ((uintptr_t)biases & 3) != 0 || ((uintptr_t)x & (size - 1)) != 0
			|| ((uintptr_t)output & (size - 1)) != 0) { return XNOR_B200_ERR_ALIGNMENT; }
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
		case XNOR_B200_F32: return launch_product_rows<float>(p, d->group, s);
		case XNOR_B200_F16: return launch_product_rows<__half>(p, d->group, s);
		default: return launch_product_rows<__nv_bfloat16>(p, d->group, s);
	}
}
