// Shared pieces of the four-bit operators (four_rows.cu, four_product.cu, four_attend.cu): element types, the tensor-core product of
// codes, and the way codes become its operands.
//
// Format: groups of 32, 64 or 128 neighbours of a row; per group fp16 (scale, low); value = low + scale * code.  Byte b of a row holds
// code 2b in its low four bits, code 2b + 1 in its high four: a 32-bit word holds codes 0..7 of eight neighbours, code i at bit 4i.
//
// Codes reach the tensor cores as they are: the word masked with 0x000F000F is two fp16 subnormals, code 0 and code 4, each code * 2^-24
// exactly; masked with 0x00F000F0 it is codes 1 and 5 times 2^-20; shifted down by eight the same masks give 2 and 6, 3 and 7.  So eight
// codes cost five integer operations and no conversion, the products are exact, and their sums are fp32.  The other operand pairs the
// same neighbours, the odd ones divided by 16, and the factor 2^24 goes into the group's scale (not into the power of two of the other
// operand's values: times 2^24 that passes fp32's range where they are 2^117 and more).
//
// fp32 and fp16 calls take code - 8 instead, as value = (low + 8 * scale) + scale * (code - 8): the sums of a group's two terms, which rounding
// (and the tensor cores' cutting off) is relative to, then hardly cancel.  1024 + code in fp16 is the same mask with the exponent's bits set
// (the common way from small integers to floats), one addition takes 1032 off; 1024 + 16 * code, times 1/16, less 72.  Four more operations
// for eight codes (2 to 10 % of a product's time: 16384 x 16384 by one row 38.2 and 34.7 us, by 16 51.7 and 47.6), and a product of 1024 fp32
// values is 2e-7 off where it was 1.3e-6; of fp16 results 0.02 % are not the nearest to the exact ones where 1.9 % were not (4096 x 4096; the
// sums in plain fp32: 0.15 %).
// bf16 results are too coarse to show it (16384 x 16384: 0.17 %, in plain fp32 0.13 %).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "xnor_common.cuh"

namespace xnor
{

// How calls of a type take their codes: what a code in the operand has to be multiplied by, odd neighbours' codes by ODD times that, and
// what is added to low as a part of the scale.
template <class T> struct Codes
{
	static constexpr bool CENTRED = !__is_same(T, __nv_bfloat16);
	static constexpr float UNIT = CENTRED ? 1.0f : 16777216.0f, ODD = CENTRED ? 1.0f : 0.0625f, SHIFT = CENTRED ? 8.0f : 0.0f;
};

__host__ __device__ __forceinline__ size_t four_row_bytes(int k) { return (size_t)((k + 31) / 32) * 16; }
inline bool four_group_ok(int g) { return g == 32 || g == 64 || g == 128; }
inline bool four_dtype_ok(int t) { return t == XNOR_B200_F32 || t == XNOR_B200_F16 || t == XNOR_B200_BF16; }
inline size_t four_size(int t) { return t == XNOR_B200_F32 ? 4 : 2; }

#ifdef __CUDACC__

// Every kernel of a call but the load-time ones starts with pdl_wait() and pdl_trigger() and is launched through this: its CTAs take their
// places while the kernel in front of it on the stream finishes, and do nothing before it has.  A decoding step is a chain of such kernels.
// So what a call reads may still be written while its kernels are there already: they read it by ordinary loads, not by those (__ldg, a
// __restrict__ pointer) that are for memory which nobody writes as long as the kernel lives.
// cluster: CTAs of a cluster, along x.
template <class Kernel, class... Args>
int launch_four(Kernel kernel, dim3 grid, unsigned threads, size_t smem, unsigned cluster, cudaStream_t stream, const Args & ... args)
{
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = grid;
	cfg.blockDim = dim3(threads, 1, 1);
	cfg.dynamicSmemBytes = smem;
	cfg.stream = stream;
	cudaLaunchAttribute attr[2];
	attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
	attr[0].val.programmaticStreamSerializationAllowed = 1;
	attr[1].id = cudaLaunchAttributeClusterDimension;
	attr[1].val.clusterDim.x = cluster;
	attr[1].val.clusterDim.y = 1;
	attr[1].val.clusterDim.z = 1;
	cfg.attrs = attr;
	cfg.numAttrs = cluster > 1 ? 2 : 1;
	const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
	return e == cudaSuccess ? check_launch() : cuda_fail(e);
}

// The smaller and the larger value; NaN where there is one.
__device__ __forceinline__ float min_nan(float a, float b)
{
	float r;
	asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
	return r;
}
__device__ __forceinline__ float max_nan(float a, float b)
{
	float r;
	asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
	return r;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight neighbours as they lie in memory.
template <class T> struct Eight { uint4 raw[sizeof(T) / 2]; };

// Eight neighbours from p, of which the first `there` exist (the others read as 0); wide: p is aligned to 16 bytes.
template <class T>
__device__ __forceinline__ Eight<T> load8(const T * p, int there, bool wide)
{
	Eight<T> v;
	if (wide && there >= 8)
	{
		v.raw[0] = reinterpret_cast<const uint4 *>(p)[0];
		if (sizeof(T) == 4) { v.raw[sizeof(T) / 2 - 1] = reinterpret_cast<const uint4 *>(p)[1]; }
		return v;
	}
	uint32_t * w = reinterpret_cast<uint32_t *>(v.raw);
	#pragma unroll
	for (int i = 0; i < 8; ++i)
	{
		if (sizeof(T) == 4) { w[i] = i < there ? reinterpret_cast<const uint32_t *>(p)[i] : 0; continue; }
		const uint32_t h = i < there ? reinterpret_cast<const uint16_t *>(p)[i] : 0;
		if (i % 2 == 0) { w[i / 2] = h; }
		else { w[i / 2] |= h << 16; }
	}
	return v;
}

template <class T>
__device__ __forceinline__ void eight_f32(const Eight<T> & e, float (&v)[8])
{
	const T * p = reinterpret_cast<const T *>(e.raw);
	#pragma unroll
	for (int i = 0; i < 8; ++i) { v[i] = to_f32(p[i]); }
}

template <class T>
__device__ __forceinline__ void store8(T * p, bool wide, const float (&v)[8])
{
	if (wide)
	{
		uint4 raw[sizeof(T) / 2];
		T * e = reinterpret_cast<T *>(raw);
		#pragma unroll
		for (int i = 0; i < 8; ++i) { e[i] = from_f32<T>(v[i]); }
		reinterpret_cast<uint4 *>(p)[0] = raw[0];
		if (sizeof(T) == 4) { reinterpret_cast<uint4 *>(p)[1] = raw[sizeof(T) / 2 - 1]; }
		return;
	}
	#pragma unroll
	for (int i = 0; i < 8; ++i) { p[i] = from_f32<T>(v[i]); }
}

// d += a * b over 16 neighbours: a 16 rows, b 8 columns, both fp16; fp32 sums.  The operand comes from packed words in registers, which
// only the warp-wide instruction takes; it runs at 0.85 products a ns and SM (measured), where the codes of one product take 3 to 6 ns
// to arrive from memory.
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
	asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
			: "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// d = a * b
__device__ __forceinline__ void mma_16816_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
	asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
			: "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ uint32_t pair_f16(float a, float b)
{
	const __half2 h = __floats2half2_rn(a, b);
	return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ __half2 as_half2(uint32_t w) { return *reinterpret_cast<const __half2 *>(&w); }
__device__ __forceinline__ uint32_t as_word(__half2 h) { return *reinterpret_cast<const uint32_t *>(&h); }

// The low four bits of each half (even), or the next four (odd), as a pair of an operand; upper: the codes of the high byte of each half, for
// either.  Written as the instructions they are: left to itself the compiler shifts once for every mask, and the integer pipe is what
// these kernels wait for.
__device__ __forceinline__ uint32_t upper(uint32_t w)
{
	uint32_t r;
	asm("shr.u32 %0, %1, 8;" : "=r"(r) : "r"(w));
	return r;
}
template <uint32_t MASK, bool CENTRED>
__device__ __forceinline__ uint32_t masked(uint32_t w)
{
	uint32_t r;
	if (CENTRED) { asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "n"(MASK), "r"(0x64006400u)); }
	else { asm("and.b32 %0, %1, %2;" : "=r"(r) : "r"(w), "n"(MASK)); }
	return r;
}
template <bool CENTRED>
__device__ __forceinline__ uint32_t even_codes(uint32_t w)
{
	const uint32_t r = masked<0x000F000Fu, CENTRED>(w);
	return CENTRED ? as_word(__hadd2(as_half2(r), as_half2(0xE408E408u))) : r;
}
template <bool CENTRED>
__device__ __forceinline__ uint32_t odd_codes(uint32_t w)
{
	const uint32_t r = masked<0x00F000F0u, CENTRED>(w);
	return CENTRED ? as_word(__hfma2(as_half2(r), as_half2(0x2C002C00u), as_half2(0xD480D480u))) : r;
}

__device__ __forceinline__ float2 halves(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }

// Copies to shared memory that run by themselves; there == false writes zeros (and reads nothing).
__device__ __forceinline__ void copy16(uint32_t smem, const void * g, bool there)
{
	asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(smem), "l"(g), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t smem, const void * g, bool there)
{
	asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" :: "r"(smem), "l"(g), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_close() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(LEFT) : "memory"); }

__device__ __forceinline__ uint32_t four_smem(const void * p) { return (uint32_t)__cvta_generic_to_shared(p); }

// Power of two that brings values of this largest magnitude (its bits) to [2^13, 2^14), and its inverse: fp16 then holds all 11 bits of
// anything down to 2^-27 of the largest, and its error is at most 2^-38 of the largest below that.  Odd neighbours of bf16 calls, divided by
// 16: 2^-23 and 2^-34; bf16's own 8 bits are all there down to 2^-26 of the largest (even neighbours: 2^-30).  An infinity or a NaN: the
// factor is 0 and the inverse NaN, so that every sum over the values is NaN.
__device__ __forceinline__ void fit_f16(uint32_t largest, float & factor, float & inverse)
{
	const uint32_t e = max(largest >> 23, 14u);
	factor = e < 255 ? __uint_as_float((267 - e) << 23) : 0.0f;
	inverse = e < 255 ? __uint_as_float((e - 13) << 23) : __uint_as_float(0x7fc00000u);
}

// A value as fp16 parts: their sum is within 2^-22 of it (relatively, down to where fit_f16's bound takes over).
__device__ __forceinline__ void split_f16(float v, float & high, float & low)
{
	high = __half2float(__float2half_rn(v));
	low = v - high;
}

#endif

}  // namespace xnor
