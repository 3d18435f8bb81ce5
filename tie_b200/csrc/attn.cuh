// What the two attention kernels (attn.cu, attn_tc.cu) share: their arguments, and how work is shared out among CTAs.
#pragma once

#include "kv_cache.cuh"

namespace tie {

// p is held times a power of two.  2^14 where its parts are fp16, which then reach down to 2^-38 of the largest; 2^-15 where they are bf16,
// whose values may be as large as fp32's: 2^15 keys with the largest p and the largest values still have a sum.
template <int KIND>
constexpr float ATTN_P_SHIFT = KIND == TIE_CUDA_KV_BF16 ? -15.0f : 14.0f;
constexpr float ATTN_LOG2E = 1.4426950408889634f;
constexpr int ATTN_UNIT = 128;	       // keys: what an item's work is counted in
constexpr int ATTN_MAX_ROWS = 128;     // query rows of a tile, at most

// An item that begins in a CTA and goes on in others: parts, and the rows they are of (n_rows: of the sequence and head; 0: none).
struct AttnJoin {
	int n, tok0, head, row0, n_rows;
};

struct AttnArgs {
	const float *q;
	float *out;
	int n_head, group;  // group: query heads per key/value head
	float scale_log2e;
	float *part;
	unsigned *count;
	AttnJoin *join;
};

// What a CTA leaves for a shared item of ROWS rows: its sums ([row][D] in attn.cu, [D / 4][row][4] in attn_tc.cu), then the maxima, the
// sums of p.
__host__ __device__ constexpr size_t attn_part_floats(int rows)
{
	return (size_t)rows * (128 + 2);
}

// Q8's value factors meet p in 16-bit parts, as shares of a unit: a power of two, of the largest factor.  The parts reach down to
// 2^-38 of it, so that a row must not share the unit of a factor that it does not see: in tiles that not every row sees in full, and
// whose factors lie further apart than ATTN_WIDE (up to there p of 1 keeps 2^-31 in its parts), each row has a unit of its own.
constexpr float ATTN_LEAST_UNIT = 0x1p-126f, ATTN_WIDE = 0x1p8f;
// Sums of Q8's products, not yet divided by the sum of p, are held 2^34 times smaller, so that 2^20 keys with factors of 2^120 do not
// pass fp32's range: 2^14 lie in the values' operand (int8_pair_low), 2^20 in the unit, which leaves factors of 2^-106 and more all bits.
constexpr float ATTN_Q8_DOWN = 0x1p-20f, ATTN_Q8_UP = 0x1p34f;
__device__ __forceinline__ float attn_unit_of(float top)
{
	return __uint_as_float(min(max(__float_as_uint(top) & 0x7f800000u, 0x00800000u), 253u << 23));
}
// of a unit, or of the inverse of one
__device__ __forceinline__ float attn_unit_inverse(float unit)
{
	return __uint_as_float((254u << 23) - __float_as_uint(unit));
}

// The work of a launch: items = (sequence, key/value head, tile of query rows), each of as many units as its keys take;
// CTA b of G does units [U b / G, U (b + 1) / G), whatever items these belong to.  An item within one CTA is finished there;
// the CTAs that share one leave (maximum, sum, rows) behind, and the last to be done adds them up in the order of the
// CTAs, so that the result does not depend on which was last.
struct AttnWork {
	long long start[KV_MAX_SEQ + 1];  // units (or items) in front of a sequence
	long long warp_sum[32];
	int last;
};

__device__ __forceinline__ long long attn_items(const KvView &kv, const AttnArgs &a, const SeqView &q, int rows)
{
	return ((long long)q.n_tok * a.group + rows - 1) / rows * kv.n_head_kv;  // (rows: a constant)
}
__device__ __forceinline__ int attn_units(const SeqView &q)
{
	return (q.kv_len + q.n_tok + ATTN_UNIT - 1) / ATTN_UNIT;
}

// Fills w.start with the running sums of `of(sequence)`, by all threads of the CTA.
template <int THREADS, class F>
__device__ __forceinline__ void attn_share_work(AttnWork &w, const KvView &kv, const StepView &st, F of)
{
	constexpr int PER = (KV_MAX_SEQ + THREADS - 1) / THREADS;
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
	if (st.n_seq == 1) {
		if (threadIdx.x == 0) {
			w.start[0] = 0;
			w.start[1] = of(kv_sequence(st, kv.page_shift, 0));
		}
		__syncthreads();
		return;
	}
	long long mine[PER], sum = 0;
#pragma unroll
	for (int i = 0; i < PER; i++) {
		const int s = threadIdx.x * PER + i;
		mine[i] = s < st.n_seq ? of(kv_sequence(st, kv.page_shift, s)) : 0;
		sum += mine[i];
	}
	long long incl = sum;
#pragma unroll
	for (int o = 1; o < 32; o <<= 1) {
		const long long v = __shfl_up_sync(0xffffffffu, incl, o);
		if (lane >= o)
			incl += v;
	}
	if (lane == 31)
		w.warp_sum[warp] = incl;
	__syncthreads();
	long long at = incl - sum;
	for (int i = 0; i < warp; i++)
		at += w.warp_sum[i];
#pragma unroll
	for (int i = 0; i < PER; i++) {
		const int s = threadIdx.x * PER + i;
		if (s <= st.n_seq)
			w.start[s] = at;
		at += mine[i];
	}
	if (threadIdx.x == THREADS - 1 && THREADS * PER <= st.n_seq)
		w.start[st.n_seq] = at;
	__syncthreads();
}

// The sequence of unit (or item) u: the last that starts at or in front of it.
__device__ __forceinline__ int attn_sequence_of(const AttnWork &w, int n_seq, long long u)
{
	int lo = 0, hi = n_seq - 1;
	while (lo < hi) {
		const int mid = (lo + hi + 1) >> 1;
		if (w.start[mid] <= u)
			lo = mid;
		else
			hi = mid - 1;
	}
	return lo;
}

// a / b for a, b > 0: mostly of numbers that 32 bits hold, where it is several times as fast
__device__ __forceinline__ long long attn_div(long long a, long long b)
{
	return (a | b) >> 32 ? a / b : (long long)((unsigned)a / (unsigned)b);
}

// The CTA that has unit u of `total`.
__device__ __forceinline__ int attn_cta_of(long long u, long long total, int n_cta)
{
	return (int)attn_div((u + 1) * n_cta - 1, total);
}

// 2^x to 2^-22, results below 2^-126 zero
__device__ __forceinline__ float exp2_ftz(float x)
{
	float r;
	asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
	return r;
}

__device__ __forceinline__ bool nonfinite16(uint32_t w, uint32_t exponent)
{
	return (w & exponent) == exponent || (w >> 16 & exponent) == exponent;
}
// Two of the four signed bytes of a word whose bytes were XORed with 0x80 as halves, exactly: byte + 128 becomes the
// mantissa of 1024 + byte + 128.
template <uint32_t SEL>
__device__ __forceinline__ uint32_t int8_pair(uint32_t x_biased)
{
	const uint32_t h = __byte_perm(x_biased, 0x64646464u, SEL);
	const __half2 v = __hsub2(*reinterpret_cast<const __half2 *>(&h), __half2half2(__ushort_as_half(0x6480)));  // 1152
	return *reinterpret_cast<const uint32_t *>(&v);
}

// The same, times 2^-14 (fp16's least normal number, so that 1 stays one).
template <uint32_t SEL>
__device__ __forceinline__ uint32_t int8_pair_low(uint32_t x_biased)
{
	const uint32_t h = __byte_perm(x_biased, 0x64646464u, SEL);
	const __half2 v = __hfma2(*reinterpret_cast<const __half2 *>(&h), __half2half2(__ushort_as_half(0x0400)), __half2half2(__ushort_as_half(0xac80)));  // -1152 * 2^-14
	return *reinterpret_cast<const uint32_t *>(&v);
}

int attn_maps(tie_cuda_ctx *c, const KvView &kv, int elem, int head_dim, int box_bytes, int box_rows, CUtensorMapSwizzle swizzle, CUtensorMap *map);
// attn_tc.cu: tiles of 128 rows on tcgen05
int attn_tc_setup(tie_cuda_ctx *c);
int launch_attn_tc(tie_cuda_ctx *c, const KvView &kv, const StepView &st, int kind, int head_dim, const AttnArgs &a);

}  // namespace tie
