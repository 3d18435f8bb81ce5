// What goes into the paged key/value cache and what comes back out of it: norms of q and k for each head, rotation and
// rounding to the cache's type in one pass over a step's q, k and v (model_qwen3.c:303-389 runs them one after the other on the
// host, engine.c:263-862), and the reverse of the last.  Both move each byte once and are bound by HBM or, for a few tokens,
// by one chain of loads.
#include <float.h>
#include <math.h>
#include <string.h>

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

// A row of q, k or v, by D / 8 lanes: lane l has the values 4 l .. 4 l + 3 and as many D / 2 further on, so that both halves of
// every pair of the rotation, of either kind, are its own (with the row over 32 lanes a pair's halves were 16 lanes
// apart: 9 shuffles a row where there are 2 now).
template <int D>
struct Row {
	static constexpr int LANES = D / 8, AT_ONCE = 32 / LANES;  // rows a warp has at once
	float v[8];
	__device__ __forceinline__ void load(const float *p, int l)
	{
		const float4 a = __ldcs(reinterpret_cast<const float4 *>(p + 4 * l)), b = __ldcs(reinterpret_cast<const float4 *>(p + D / 2 + 4 * l));
		v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
	}
	__device__ __forceinline__ void store(float *p, int l) const
	{
		*reinterpret_cast<float4 *>(p + 4 * l) = make_float4(v[0], v[1], v[2], v[3]);
		*reinterpret_cast<float4 *>(p + D / 2 + 4 * l) = make_float4(v[4], v[5], v[6], v[7]);
	}
	__device__ __forceinline__ void norm(const float *w, float eps, int l)
	{
		float ss = 0.0f;
#pragma unroll
		for (int j = 0; j < 8; j++)
			ss = fmaf(v[j], v[j], ss);
#pragma unroll
		for (int o = LANES / 2; o; o >>= 1)
			ss += __shfl_xor_sync(0xffffffffu, ss, o);
		const float inv = rsqrtf(ss * (1.0f / D) + eps);
#pragma unroll
		for (int j = 0; j < 8; j++)
			v[j] = w ? v[j] * __ldg(w + (j < 4 ? 4 * l + j : D / 2 + 4 * l + j - 4)) * inv : v[j];
	}
	// turn[j]: interleaved, of pair (2 j, 2 j + 1) of v; else of pair (j, j + 4)
	__device__ __forceinline__ void rotate(const float2 (&turn)[4], bool interleaved)
	{
#pragma unroll
		for (int j = 0; j < 4; j++) {
			float &a = interleaved ? v[2 * j] : v[j], &b = interleaved ? v[2 * j + 1] : v[j + 4];
			const float x = a, y = b;
			a = x * turn[j].x - y * turn[j].y;
			b = y * turn[j].x + x * turn[j].y;
		}
	}
};

// A row of the cache.  F16 and BF16 round to nearest (beyond +-65504 F16 holds infinities); Q8 is rint(x / s) with
// s = max|x| / 127, both divisions as IEEE has them so that a file of one machine reads the same on another.  A row with an
// infinity or NaN reads back as NaN throughout; one whose s would not be a normal number, as zeros.
// All lanes of the warp come here; a row is stored where `row` is not negative.
template <int KIND, int D>
__device__ __forceinline__ void store_cache_row(uint8_t *rows, float *scales, long long row, const float (&v)[8], int l)
{
	uint32_t w[4];
	if constexpr (KIND == TIE_CUDA_KV_Q8) {
		uint32_t top = 0;  // the largest magnitude, as the number that its bits are (NaN above infinity)
#pragma unroll
		for (int j = 0; j < 8; j++)
			top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
#pragma unroll
		for (int o = Row<D>::LANES / 2; o; o >>= 1)
			top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
		const bool fine = top < 0x7f800000u;
		float s = __fdiv_rn(__uint_as_float(top), 127.0f);
		s = s >= FLT_MIN ? s : 0.0f;
		w[0] = w[1] = 0;
		if (fine && s > 0.0f)
#pragma unroll
			for (int j = 0; j < 8; j++)
				w[j >> 2] |= (uint32_t)(max(-127, min(127, __float2int_rn(__fdiv_rn(v[j], s)))) & 0xff) << (8 * (j & 3));
		if (row < 0)
			return;
		*reinterpret_cast<uint32_t *>(rows + row * D + 4 * l) = w[0];
		*reinterpret_cast<uint32_t *>(rows + row * D + D / 2 + 4 * l) = w[1];
		if (l == 0)
			scales[row] = fine ? s : __int_as_float(0x7fc00000);
	} else {
		if (row < 0)
			return;
#pragma unroll
		for (int j = 0; j < 4; j++) {
			if constexpr (KIND == TIE_CUDA_KV_F16) {
				const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
				w[j] = *reinterpret_cast<const uint32_t *>(&h);
			} else {
				const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
				w[j] = *reinterpret_cast<const uint32_t *>(&h);
			}
		}
		*reinterpret_cast<uint2 *>(rows + (row * D + 4 * l) * 2) = make_uint2(w[0], w[1]);
		*reinterpret_cast<uint2 *>(rows + (row * D + D / 2 + 4 * l) * 2) = make_uint2(w[2], w[3]);
	}
}

// One CTA: one token (4096 tokens with 32 heads of q and 4 each of k and v, BF16: 30.7 us, 5.2 TB/s; one token: 11.8 us, launch and
// call); a warp takes two or four head rows at a time, the next ones requested before those in hand are worked on,
// the first before anything is known of the token; blockIdx.y shares the rows of a token out where tokens alone would leave
// SMs idle.  Two warps find the token's place for all and form its angles, in 64 bits and in turns, so that only the
// fraction of a turn is rounded to 32: at position 100,000 a 32-bit angle would be off by up to 0.004.
constexpr int WRITE_THREADS = 128, WRITE_WARPS = WRITE_THREADS / 32;
template <int KIND, int D>
__global__ void __launch_bounds__(WRITE_THREADS) qk_norm_rope_rows(const KvView kv, const StepView st, const QkvArgs a, const __grid_constant__ RopeTable rope)
{
	using R = Row<D>;
	constexpr int HALF = D / 2;
	__shared__ float2 s_turn[HALF];	 // cos, sin
	__shared__ int s_place[2];	 // slot (-1: has none), page
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = blockIdx.x, l = lane % R::LANES;
	const int rows = a.n_head + 2 * kv.n_head_kv, step = WRITE_WARPS * gridDim.y * R::AT_ONCE;
	int r = (blockIdx.y * WRITE_WARPS + warp) * R::AT_ONCE + lane / R::LANES;
	auto load = [&](int r, R &x) {
		if (r < a.n_head)
			x.load(a.q + t * a.q_stride + r * D, l);
		else if (r < rows)
			x.load(r < a.n_head + kv.n_head_kv ? a.k + t * a.k_stride + (r - a.n_head) * D : a.v + t * a.v_stride + (r - a.n_head - kv.n_head_kv) * D, l);
	};
	R next;
#pragma unroll
	for (int j = 0; j < 8; j++)
		next.v[j] = 0.0f;
	load(r, next);
	if (warp < 2) {
		const int s = kv_find_sequence(st, t, lane);
		int slot = -1, page = 0;
		if (s >= 0) {
			const SeqView seq = kv_sequence(st, kv.page_shift, s);
			const int i = t - seq.tok0;
			if (i >= 0 && i < seq.n_tok) {  // (reported by kv_sequence where it does not fit)
				slot = seq.kv_len + i;
				page = st.page_table[(long long)s * st.max_pages + (slot >> kv.page_shift)];
			}
			if (a.rotate && slot >= 0 && threadIdx.x < HALF) {
				const int pos = st.pos ? st.pos[t] : slot;
				const double turns = pos * rope.turns[threadIdx.x], part = turns - rint(turns);
				float2 cs;
				sincospif((float)(2.0 * part), &cs.y, &cs.x);
				s_turn[threadIdx.x] = cs;
			}
		}
		if (threadIdx.x == 0) {
			s_place[0] = slot;
			s_place[1] = page;
		}
	}
	__syncthreads();
	const int slot = s_place[0], page = s_place[1];
	if (slot < 0)
		return;	 // a row that no sequence has, or has no slot for
	const int in_page = slot & ((1 << kv.page_shift) - 1);
	float2 turn[4];
	if (a.rotate)
#pragma unroll
		for (int j = 0; j < 4; j++)
			turn[j] = s_turn[!a.interleaved ? 4 * l + j : j < 2 ? 2 * l + j : HALF / 2 + 2 * l + j - 2];
#pragma unroll 1
	for (int r_warp = r - lane / R::LANES; r_warp < rows; r_warp += step, r += step) {
		R x = next;
		load(r + step, next);
		const bool is_q = r < a.n_head, is_v = r >= a.n_head + kv.n_head_kv;
		x.norm(is_q ? a.q_norm_w : is_v ? nullptr : a.k_norm_w, a.eps, l);
		if (a.rotate && !is_v) {
			if (a.interleaved)
				x.rotate(turn, true);
			else
				x.rotate(turn, false);
		}
		if (is_q)
			x.store(a.q_out + ((long long)t * a.n_head + r) * D, l);
		if (r_warp + R::AT_ONCE <= a.n_head)
			continue;  // (of these rows none is the cache's)
		const int head = is_v ? r - a.n_head - kv.n_head_kv : r - a.n_head;
		const long long page_row = !is_q && r < rows ? kv_page_row(kv, st, page, head) : -1;
		store_cache_row<KIND, D>(is_v ? kv.v : kv.k, is_v ? kv.v_scale : kv.k_scale, page_row < 0 ? -1 : page_row + in_page, x.v, l);
	}
}

// A row's N = D / 32 values of a lane, as the cache holds them.
template <int KIND, int N>
struct CacheValues {
	uint32_t raw[KIND == TIE_CUDA_KV_Q8 ? 1 : N / 2];
	float scale;
	__device__ __forceinline__ void load(const uint8_t *rows, const float *scales, long long row, int lane)
	{
		if constexpr (KIND == TIE_CUDA_KV_Q8) {
			const uint8_t *p = rows + row * (32 * N) + lane * N;
			raw[0] = N == 4 ? __ldcs(reinterpret_cast<const uint32_t *>(p)) : __ldcs(reinterpret_cast<const uint16_t *>(p));
			scale = __ldg(scales + row);
		} else {
			const uint8_t *p = rows + (row * (32 * N) + lane * N) * 2;
			if constexpr (N == 4) {
				const uint2 v = __ldcs(reinterpret_cast<const uint2 *>(p));
				raw[0] = v.x, raw[1] = v.y;
			} else {
				raw[0] = __ldcs(reinterpret_cast<const uint32_t *>(p));
			}
		}
	}
	__device__ __forceinline__ float value(int i) const
	{
		if constexpr (KIND == TIE_CUDA_KV_Q8)
			return (float)(int8_t)(raw[0] >> (8 * i) & 0xff) * scale;
		const uint32_t w = raw[i >> 1], h = i & 1 ? w >> 16 : w & 0xffffu;
		return KIND == TIE_CUDA_KV_F16 ? __half2float(__ushort_as_half((unsigned short)h)) : __uint_as_float(h << 16);
	}
};

template <typename O, int N>
__device__ __forceinline__ void store_values(O *p, const float (&x)[N])
{
	if constexpr (sizeof(O) == 4) {
		if constexpr (N == 4)
			__stcs(reinterpret_cast<float4 *>(p), make_float4(x[0], x[1], x[2], x[3]));
		else
			__stcs(reinterpret_cast<float2 *>(p), make_float2(x[0], x[1]));
	} else {
		uint32_t w[N / 2];
#pragma unroll
		for (int i = 0; i < N / 2; i++) {
			if constexpr (std::is_same<O, __half>::value) {
				const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
				w[i] = *reinterpret_cast<const uint32_t *>(&h);
			} else {
				const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
				w[i] = *reinterpret_cast<const uint32_t *>(&h);
			}
		}
		if constexpr (N == 4)
			__stcs(reinterpret_cast<uint2 *>(p), make_uint2(w[0], w[1]));
		else
			__stcs(reinterpret_cast<uint32_t *>(p), w[0]);
	}
}

// One CTA: READ_TOKENS tokens of one head, keys (blockIdx.z 0) or values.  A warp takes a row at a time, so that its stores are
// whole rows (8 values a thread, two stores of 16 bytes 32 apart: 134 us for 120000 slots of Q8 to fp32, now 109, 5.6 TB/s), READ_U of them in flight.
constexpr int READ_TOKENS = 64, READ_U = READ_TOKENS / WARPS;
template <int KIND, int D, typename O>
__global__ void __launch_bounds__(THREADS) kv_read_rows(const KvView kv, const StepView st, O *k_out, O *v_out)
{
	constexpr int N = D / 32;
	__shared__ long long s_row[READ_TOKENS];
	const int head = blockIdx.y, t0 = blockIdx.x * READ_TOKENS, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
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
	CacheValues<KIND, N> o[READ_U];
#pragma unroll
	for (int u = 0; u < READ_U; u++) {
		const long long row = s_row[warp * READ_U + u];
		if (row >= 0)
			o[u].load(rows, scales, row, lane);
	}
#pragma unroll
	for (int u = 0; u < READ_U; u++) {
		const int b = warp * READ_U + u;
		if (s_row[b] < 0)
			continue;
		float x[N];
#pragma unroll
		for (int i = 0; i < N; i++)
			x[i] = o[u].value(i);
		store_values(out + ((long long)(t0 + b) * kv.n_head_kv + head) * D + lane * N, x);
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
	RopeTable rope;
	if (a.rotate) {
		// (a context's layers have one base: the 64 powers of a call took the host longer than the launch)
		tie_cuda_ctx::RopeTurns &known = c->rope;
		if (known.base != in.rope_base || known.head_dim != head_dim) {
			for (int i = 0; i < head_dim / 2; i++)
				known.turns[i] = (double)(powl((long double)in.rope_base, -2.0L * i / head_dim) / (2.0L * 3.14159265358979323846264338327950288L));
			known.base = in.rope_base;
			known.head_dim = head_dim;
		}
		memcpy(rope.turns, known.turns, sizeof(rope.turns));
	}
	// rows of a token go to as many CTAs as it takes to have two per SM
	const int rows = in.n_head + 2 * kv.n_head_kv, at_once = WRITE_WARPS * 32 / (head_dim / 8), most = (rows + at_once - 1) / at_once;
	const int want = (2 * c->sm_count + st.n_tokens - 1) / st.n_tokens;
	const dim3 grid(st.n_tokens, want < most ? want : most);
#define TIE_GO(KIND, D) qk_norm_rope_rows<KIND, D><<<grid, WRITE_THREADS, 0, c->stream>>>(kv, st, a, rope)
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
