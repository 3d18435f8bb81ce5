// What goes into the paged key/value cache and what comes back out of it: norms of q and k for each head, rotation and
// rounding to the cache's type in one pass over a step's q, k and v (model_qwen3.c:303-389 runs them one after the other on the
// host, engine.c:263-862), and the reverse of the last.  Both move each byte once and are bound by HBM or, for a few tokens,
// by one chain of loads.
#include <float.h>
#include <math.h>

#include <type_traits>

#include "kernels.cuh"
#include "kv_cache.cuh"

namespace tie {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;

struct RopeTable {
	double turns[64];  // base^(-2i/D) / 2 pi: turns per position of pair i
};

struct QkvArgs {
	const float *q, *k, *v;
	long long q_stride, k_stride, v_stride;
	const float *q_norm_w, *k_norm_w;
	float *q_out;
	int n_head;
	float eps;
	int rotate, interleaved;
};

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
	for (int o = 16; o; o >>= 1)
		v += __shfl_xor_sync(0xffffffffu, v, o);
	return v;
}

// N consecutive values of a row (N = 2 or 4)
template <int N>
__device__ __forceinline__ void load_row(float (&x)[N], const float *p)
{
	if constexpr (N == 4) {
		const float4 v = __ldcs(reinterpret_cast<const float4 *>(p));
		x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
	} else {
		const float2 v = __ldcs(reinterpret_cast<const float2 *>(p));
		x[0] = v.x, x[1] = v.y;
	}
}
template <int N>
__device__ __forceinline__ void store_row(float *p, const float (&x)[N])
{
	if constexpr (N == 4)
		*reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
	else
		*reinterpret_cast<float2 *>(p) = make_float2(x[0], x[1]);
}

// A row of the cache, by a warp.  F16 and BF16 round to nearest (beyond +-65504 F16 holds infinities); Q8 is
// rint(x / s) with s = max|x| / 127, both divisions as IEEE has them so that a file of one machine reads the same on
// another.  A row with an infinity or NaN reads back as NaN throughout; one whose s would not be a normal number, as zeros.
template <int KIND, int N>
__device__ __forceinline__ void store_cache_row(uint8_t *rows, float *scales, long long row, const float (&x)[N], int lane)
{
	if constexpr (KIND == TIE_CUDA_KV_Q8) {
		float top = 0.0f;
		bool fine = true;
#pragma unroll
		for (int i = 0; i < N; i++) {
			top = fmaxf(top, fabsf(x[i]));
			fine = fine && fabsf(x[i]) <= FLT_MAX;
		}
		top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
		fine = __all_sync(0xffffffffu, fine);
		float s = __fdiv_rn(top, 127.0f);
		s = s >= FLT_MIN ? s : 0.0f;
		uint32_t packed = 0;
#pragma unroll
		for (int i = 0; i < N; i++) {
			const int q = fine && s > 0.0f ? max(-127, min(127, __float2int_rn(__fdiv_rn(x[i], s)))) : 0;
			packed |= (uint32_t)(q & 0xff) << (8 * i);
		}
		uint8_t *p = rows + row * (32 * N) + lane * N;
		if constexpr (N == 4)
			*reinterpret_cast<uint32_t *>(p) = packed;
		else
			*reinterpret_cast<uint16_t *>(p) = (uint16_t)packed;
		if (lane == 0)
			scales[row] = fine ? s : __int_as_float(0x7fc00000);
	} else {
		uint32_t w[N / 2];
#pragma unroll
		for (int i = 0; i < N / 2; i++) {
			if constexpr (KIND == TIE_CUDA_KV_F16) {
				const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
				w[i] = *reinterpret_cast<const uint32_t *>(&h);
			} else {
				const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
				w[i] = *reinterpret_cast<const uint32_t *>(&h);
			}
		}
		uint8_t *p = rows + (row * (32 * N) + lane * N) * 2;
		if constexpr (N == 4)
			*reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
		else
			*reinterpret_cast<uint32_t *>(p) = w[0];
	}
}

// One CTA: one token; a warp takes a head row at a time (a lane D / 32 neighbouring values), blockIdx.y shares the rows of a
// token out where tokens alone would leave SMs idle.  Angles are formed once per CTA, in 64 bits and in turns, so that only the
// fraction of a turn is rounded to 32: at position 100,000 a 32-bit angle would be off by up to 0.004.
template <int KIND, int D>
__global__ void __launch_bounds__(THREADS) qk_norm_rope_rows(const KvView kv, const StepView st, const QkvArgs a, const __grid_constant__ RopeTable rope)
{
	constexpr int N = D / 32, HALF = D / 2;
	__shared__ float2 s_turn[HALF];	 // cos, sin
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = blockIdx.x;
	const int s = kv_find_sequence(st, t, lane);
	if (s < 0)
		return;	 // a row behind the last sequence
	const SeqView seq = kv_sequence(st, kv.page_shift, s);
	const int i = t - seq.tok0;
	const bool fits = i >= 0 && i < seq.n_tok;  // (reported by kv_sequence where it does not)
	const int slot = fits ? seq.kv_len + i : 0;
	if (a.rotate && threadIdx.x < HALF) {
		const int pos = st.pos ? st.pos[t] : slot;
		const double turns = pos * rope.turns[threadIdx.x], part = turns - rint(turns);
		float2 cs;
		sincospif((float)(2.0 * part), &cs.y, &cs.x);
		s_turn[threadIdx.x] = cs;
	}
	const int page = st.page_table[(long long)s * st.max_pages + (slot >> kv.page_shift)];
	__syncthreads();
	const int rows = a.n_head + 2 * kv.n_head_kv, step = WARPS * gridDim.y;
	for (int r = blockIdx.y * WARPS + warp; r < rows; r += step) {
		const int which = r < a.n_head ? 0 : r < a.n_head + kv.n_head_kv ? 1 : 2;
		const int head = which == 0 ? r : which == 1 ? r - a.n_head : r - a.n_head - kv.n_head_kv;
		const float *src = which == 0 ? a.q + t * a.q_stride : which == 1 ? a.k + t * a.k_stride : a.v + t * a.v_stride;
		float x[N];
		load_row(x, src + head * D + lane * N);
		const float *w = which == 0 ? a.q_norm_w : which == 1 ? a.k_norm_w : nullptr;
		if (w) {
			float ss = 0.0f;
#pragma unroll
			for (int j = 0; j < N; j++)
				ss = fmaf(x[j], x[j], ss);
			const float inv = 1.0f / sqrtf(warp_sum(ss) / D + a.eps);
#pragma unroll
			for (int j = 0; j < N; j++)
				x[j] = x[j] * __ldg(w + lane * N + j) * inv;
		}
		if (which < 2 && a.rotate) {
			if (a.interleaved) {  // pairs (2i, 2i + 1)
#pragma unroll
				for (int j = 0; j < N; j += 2) {
					const float2 cs = s_turn[(lane * N + j) / 2];
					const float x0 = x[j], x1 = x[j + 1];
					x[j] = x0 * cs.x - x1 * cs.y;
					x[j + 1] = x1 * cs.x + x0 * cs.y;
				}
			} else {  // pairs (i, i + D / 2): the other half of the row is 16 lanes away
#pragma unroll
				for (int j = 0; j < N; j++) {
					const float2 cs = s_turn[(lane & 15) * N + j];
					const float other = __shfl_xor_sync(0xffffffffu, x[j], 16);
					x[j] = x[j] * cs.x + (lane < 16 ? -other : other) * cs.y;
				}
			}
		}
		if (which == 0) {
			store_row(a.q_out + ((long long)t * a.n_head + head) * D + lane * N, x);
			continue;
		}
		const long long first = fits ? kv_page_row(kv, st, page, head) : -1;
		if (first < 0)
			continue;
		const long long row = first + (slot & ((1 << kv.page_shift) - 1));
		if (which == 1)
			store_cache_row<KIND>(kv.k, kv.k_scale, row, x, lane);
		else
			store_cache_row<KIND>(kv.v, kv.v_scale, row, x, lane);
	}
}

// 8 consecutive values of a row of the cache.
template <int KIND, int D>
struct CacheOctet {
	uint4 raw;
	float scale = 1.0f;
	__device__ __forceinline__ void load(const uint8_t *rows, const float *scales, long long row, int at)
	{
		if constexpr (KIND == TIE_CUDA_KV_Q8) {
			const uint2 v = __ldcs(reinterpret_cast<const uint2 *>(rows + row * D + at * 8));
			raw = make_uint4(v.x, v.y, 0, 0);
			scale = scales[row];
		} else {
			raw = __ldcs(reinterpret_cast<const uint4 *>(rows + (row * D + at * 8) * 2));
		}
	}
	__device__ __forceinline__ void values(float (&x)[8]) const
	{
		const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
		for (int i = 0; i < 4; i++) {
			if constexpr (KIND == TIE_CUDA_KV_Q8) {
				const uint32_t b = w[i >> 1] >> (16 * (i & 1));
				x[2 * i] = (float)(int8_t)(b & 0xff) * scale;
				x[2 * i + 1] = (float)(int8_t)((b >> 8) & 0xff) * scale;
			} else if constexpr (KIND == TIE_CUDA_KV_F16) {
				const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
				x[2 * i] = f.x, x[2 * i + 1] = f.y;
			} else {
				x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
			}
		}
	}
};

template <typename O>
__device__ __forceinline__ void store_octet(O *p, const float (&x)[8])
{
	if constexpr (sizeof(O) == 4) {
		__stcs(reinterpret_cast<float4 *>(p), make_float4(x[0], x[1], x[2], x[3]));
		__stcs(reinterpret_cast<float4 *>(p) + 1, make_float4(x[4], x[5], x[6], x[7]));
	} else {
		uint32_t w[4];
#pragma unroll
		for (int i = 0; i < 4; i++) {
			if constexpr (std::is_same<O, __half>::value) {
				const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
				w[i] = *reinterpret_cast<const uint32_t *>(&h);
			} else {
				const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
				w[i] = *reinterpret_cast<const uint32_t *>(&h);
			}
		}
		__stcs(reinterpret_cast<uint4 *>(p), make_uint4(w[0], w[1], w[2], w[3]));
	}
}

// One CTA: READ_TOKENS tokens of one head, keys (blockIdx.z 0) or values; D / 8 threads a row, READ_U rows in flight per thread.
constexpr int READ_TOKENS = 64;
template <int KIND, int D, typename O>
__global__ void __launch_bounds__(THREADS) kv_read_rows(const KvView kv, const StepView st, O *k_out, O *v_out)
{
	constexpr int PER_ROW = D / 8, AT_ONCE = THREADS / PER_ROW, U = READ_TOKENS / AT_ONCE;
	__shared__ long long s_row[READ_TOKENS];
	const int head = blockIdx.y, t0 = blockIdx.x * READ_TOKENS;
	if (threadIdx.x < READ_TOKENS) {  // each token's row, by a thread
		const int t = t0 + threadIdx.x;
		long long row = -1;
		const int s = t < st.n_tokens ? kv_find_sequence_alone(st, t) : -1;
		if (s >= 0) {
			const SeqView seq = kv_sequence(st, kv.page_shift, s);
			const int i = t - seq.tok0, slot = seq.kv_len + i;
			if (i >= 0 && i < seq.n_tok) {
				row = kv_page_row(kv, st, st.page_table[(long long)s * st.max_pages + (slot >> kv.page_shift)], head);
				if (row >= 0)
					row += slot & ((1 << kv.page_shift) - 1);
			}
		}
		s_row[threadIdx.x] = row;
	}
	__syncthreads();
	const uint8_t *rows = blockIdx.z ? kv.v : kv.k;
	const float *scales = blockIdx.z ? kv.v_scale : kv.k_scale;
	O *out = blockIdx.z ? v_out : k_out;
	const int at = threadIdx.x % PER_ROW, first = threadIdx.x / PER_ROW;
	CacheOctet<KIND, D> o[U];
#pragma unroll
	for (int u = 0; u < U; u++) {
		const long long row = s_row[first + u * AT_ONCE];
		if (row >= 0)
			o[u].load(rows, scales, row, at);
	}
#pragma unroll
	for (int u = 0; u < U; u++) {
		const int b = first + u * AT_ONCE;
		if (s_row[b] < 0)
			continue;
		float x[8];
		o[u].values(x);
		store_octet(out + ((long long)(t0 + b) * kv.n_head_kv + head) * D + at * 8, x);
	}
}

template <int KIND, int D>
int launch_read_as(tie_cuda_ctx *c, const KvView &kv, const StepView &st, void *k_out, void *v_out, int out_type)
{
	const dim3 grid((st.n_tokens + READ_TOKENS - 1) / READ_TOKENS, kv.n_head_kv, 2);
	if (out_type == TIE_CUDA_KV_F32)
		kv_read_rows<KIND, D, float><<<grid, THREADS, 0, c->stream>>>(kv, st, static_cast<float *>(k_out), static_cast<float *>(v_out));
	else if (out_type == TIE_CUDA_KV_F16)
		kv_read_rows<KIND, D, __half><<<grid, THREADS, 0, c->stream>>>(kv, st, static_cast<__half *>(k_out), static_cast<__half *>(v_out));
	else
		kv_read_rows<KIND, D, __nv_bfloat16>
			<<<grid, THREADS, 0, c->stream>>>(kv, st, static_cast<__nv_bfloat16 *>(k_out), static_cast<__nv_bfloat16 *>(v_out));
	TIE_CUDA_LAUNCHED(c);
	return TIE_CUDA_OK;
}

}  // namespace

int launch_qk_norm_rope(tie_cuda_ctx *c, const KvView &kv, const StepView &st, int kind, int head_dim, const tie_cuda_attn_qkv &in)
{
	QkvArgs a = {in.q, in.k, in.v, in.q_stride, in.k_stride, in.v_stride, in.q_norm_w, in.k_norm_w, in.q_out, in.n_head, in.norm_eps, in.rope_base > 0.0f, in.rope_interleaved};
	RopeTable rope = {};
	if (a.rotate)
		for (int i = 0; i < head_dim / 2; i++)
			rope.turns[i] = (double)(powl((long double)in.rope_base, -2.0L * i / head_dim) / (2.0L * 3.14159265358979323846264338327950288L));
	// rows of a token go to as many CTAs as it takes to have two per SM
	const int rows = in.n_head + 2 * kv.n_head_kv, most = (rows + WARPS - 1) / WARPS;
	const int want = (2 * c->sm_count + st.n_tokens - 1) / st.n_tokens;
	const dim3 grid(st.n_tokens, want < most ? want : most);
#define TIE_GO(KIND, D) qk_norm_rope_rows<KIND, D><<<grid, THREADS, 0, c->stream>>>(kv, st, a, rope)
	if (head_dim == 128)
		kind == TIE_CUDA_KV_F16 ? TIE_GO(TIE_CUDA_KV_F16, 128) : kind == TIE_CUDA_KV_BF16 ? TIE_GO(TIE_CUDA_KV_BF16, 128) : TIE_GO(TIE_CUDA_KV_Q8, 128);
	else
		kind == TIE_CUDA_KV_F16 ? TIE_GO(TIE_CUDA_KV_F16, 64) : kind == TIE_CUDA_KV_BF16 ? TIE_GO(TIE_CUDA_KV_BF16, 64) : TIE_GO(TIE_CUDA_KV_Q8, 64);
#undef TIE_GO
	TIE_CUDA_LAUNCHED(c);
	return TIE_CUDA_OK;
}

int launch_kv_read(tie_cuda_ctx *c, const KvView &kv, const StepView &st, int kind, int head_dim, void *k_out, void *v_out, int out_type)
{
#define TIE_GO(KIND) (head_dim == 128 ? launch_read_as<KIND, 128>(c, kv, st, k_out, v_out, out_type) : launch_read_as<KIND, 64>(c, kv, st, k_out, v_out, out_type))
	return kind == TIE_CUDA_KV_F16 ? TIE_GO(TIE_CUDA_KV_F16) : kind == TIE_CUDA_KV_BF16 ? TIE_GO(TIE_CUDA_KV_BF16) : TIE_GO(TIE_CUDA_KV_Q8);
#undef TIE_GO
}

}  // namespace tie
