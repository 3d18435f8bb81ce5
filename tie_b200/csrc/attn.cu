// Attention of a step's tokens over the paged cache (engine.c:794-862 does it per head and token on the host):
//
//   out[t][h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale * q[t][h].k_j - max),
//
// j over the slots in front of the step and the step's own tokens that t sees (its tree mask, or those up to itself); a
// token that sees nothing gets zeros.  One pass over keys and values with a running maximum and sum.
#include <float.h>

#include "attn.cuh"
#include "decode_common.cuh"
#include "kernels.cuh"
#include "mma_dot.cuh"
#include "tc_ptx.cuh"

namespace tie {
namespace {

constexpr int WARPS = 8, WORKERS = 32 * WARPS;	// warps and threads that work on keys
constexpr int ASKERS = 4, EACH = WARPS / ASKERS, THREADS = WORKERS + 32 * ASKERS;  // warps that request keys and values for them
constexpr int MAX_ROWS = 16;  // query rows of a CTA's tile

template <int KIND, int D>
struct Cfg {
	static constexpr bool Q8 = KIND == TIE_CUDA_KV_Q8;
	static constexpr int ROW = Q8 ? D : 2 * D;  // bytes of a head row of the cache
	static constexpr int GROUP = ROW == 256 ? 16 : 32;  // keys a warp takes at a time
	static constexpr int HALVES = GROUP / 16;
	static constexpr int BOX_BYTES = ROW < 128 ? ROW : 128;	// of a row, side by side in a TMA box; what is further comes behind: [64 dims][row]
	static constexpr int PANEL = GROUP * 128;
	static_assert(ROW <= 128 || HALVES == 1, "a box is a group's rows");
	static constexpr int STAGE = 2 * GROUP * ROW, STAGES = STAGE > 4096 ? 3 : 6;
	static constexpr int FACTORS = Q8 ? 2 * GROUP * 4 : 0;	// of a stage's keys, then of its values: behind all warps' stages
	static_assert(STAGE % 1024 == 0, "the swizzle is by address");
	// parts of an fp32 operand: bf16 3 x 8 bits, fp16 2 x 11; Q8's queries are 3 bytes (whole numbers of 24 bits, sums exact)
	static constexpr int PARTS = KIND == TIE_CUDA_KV_BF16 ? 3 : 2, Q_PARTS = Q8 ? 3 : PARTS, Q_STEP = Q8 ? 32 : 16;
	// where TMA puts a 16-byte chunk of a row: eight consecutive keys' chunks of a column lie in eight different bank groups
	__device__ static __forceinline__ int place(int row, int ch)
	{
		if (ROW == 64)
			return row * 64 + ((ch ^ (row >> 1 & 3)) << 4);
		return (ch >> 3) * PANEL + row * 128 + (((ch & 7) ^ (row & 7)) << 4);
	}
};

__device__ __forceinline__ void workers_sync()
{
	asm volatile("bar.sync 1, %0;" ::"n"(WORKERS) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr)
{
	asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr)
{
	asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
		     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
		     : "r"(addr)
		     : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v)
{
	uint32_t r;
	asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
	return r;
}
__device__ __forceinline__ void mma_16816_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
	asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
	    : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
	    : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <int KIND>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
	if constexpr (KIND == TIE_CUDA_KV_BF16)
		mma_16816_bf16(c, a[0], a[1], a[2], a[3], b0, b1);
	else
		mma_16816(c, a[0], a[1], a[2], a[3], b0, b1);
}

__device__ __forceinline__ void mma_bytes(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
	asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
	    : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
	    : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// (a, b) as PARTS pairs of 16-bit parts, the largest first, that add up to them (to 22 bits in fp16, all 24 in bf16).
template <int KIND, int PARTS>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&part)[PARTS])
{
#pragma unroll
	for (int p = 0; p < PARTS; p++) {
		if constexpr (KIND == TIE_CUDA_KV_BF16) {
			const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
			part[p] = *reinterpret_cast<const uint32_t *>(&h);
			a -= __bfloat162float(h.x);
			b -= __bfloat162float(h.y);
		} else {
			const __half2 h = __floats2half2_rn(a, b);
			part[p] = *reinterpret_cast<const uint32_t *>(&h);
			a -= __half2float(h.x);
			b -= __half2float(h.y);
		}
	}
}

// The groups in flight of each worker warp.
template <int KIND, int D>
struct Ring {
	using C = Cfg<KIND, D>;
	uint64_t full[WARPS][C::STAGES], empty[WARPS][C::STAGES];
	unsigned there[WARPS][C::STAGES];  // which 16 keys of a group have a page
};

// The pieces of work of a CTA, one after the other.
struct Piece {
	SeqView seq;
	int s, head, row0, unit0, unit1, item_units, key_end;
	long long first_unit;  // of the item
};
template <int ROWS>
__device__ __forceinline__ Piece piece_at(long long u, long long u_end, const AttnWork &work, const KvView &kv, const StepView &st, const AttnArgs &a)
{
	Piece p;
	p.s = attn_sequence_of(work, st.n_seq, u);
	p.seq = kv_sequence(st, kv.page_shift, p.s);
	p.item_units = attn_units(p.seq);
	const int tiles = (p.seq.n_tok * a.group + ROWS - 1) / ROWS;
	const long long in_seq = u - work.start[p.s], item = attn_div(in_seq, p.item_units);
	p.unit0 = (int)(in_seq - item * p.item_units);
	p.unit1 = (int)min((long long)p.item_units, p.unit0 + (u_end - u));
	p.first_unit = u - p.unit0;
	p.head = (int)attn_div(item, tiles);
	p.row0 = (int)(item - (long long)p.head * tiles) * ROWS;
	// a tile's last row sees the furthest unless a tree says otherwise
	p.key_end = p.seq.kv_len + (st.tree ? p.seq.n_tok : min((p.row0 + ROWS - 1) / a.group, p.seq.n_tok - 1) + 1);
	return p;
}

// The last warps: a lane requests a worker's groups, a TMA box per page for keys and for values, as its slots get free, and runs
// ahead of the workers into the next piece while they join the one before.  A request holds up the warp that makes it for about a
// hundred cycles: each worker for itself, it was 900 a group of 32 keys; one warp for all eight, 80 us instead of 73 for 48
// sequences of 5000.
template <int KIND, int D, int ROWS>
__device__ __forceinline__ void request(Ring<KIND, D> *ring, uint32_t stages, uint32_t factors, long long u, long long u_end, const AttnWork &work, const KvView &kv,
					const StepView &st, const AttnArgs &a, const CUtensorMap *k_map, const CUtensorMap *v_map, int worker, bool mine)
{
	using C = Cfg<KIND, D>;
	const int in_page = (1 << kv.page_shift) - 1;
	const bool one = (1 << kv.page_shift) >= C::GROUP;
	uint32_t n = 0;
	while (u < u_end) {
		const Piece p = piece_at<ROWS>(u, u_end, work, kv, st, a);
		const int *pages = st.page_table + (long long)p.s * st.max_pages;
		const int g0 = p.unit0 * (ATTN_UNIT / C::GROUP) + worker, g_end = min(p.unit1 * (ATTN_UNIT / C::GROUP), (p.key_end + C::GROUP - 1) / C::GROUP);
		int next[C::HALVES];
		auto pages_of = [&](int g) {
#pragma unroll
			for (int h = 0; h < C::HALVES; h++)
				next[h] = mine && g < g_end && g * C::GROUP + 16 * h < p.key_end ? pages[(g * C::GROUP + 16 * h) >> kv.page_shift] : 0;
		};
		pages_of(g0);
		for (int g = g0; mine && g < g_end; g += WARPS, n++) {
			long long row[C::HALVES];
			unsigned ok = 0;
#pragma unroll
			for (int h = 0; h < C::HALVES; h++) {
				const int key = g * C::GROUP + 16 * h;
				row[h] = key < p.key_end ? kv_page_row(kv, st, next[h], p.head) : -1;
				ok |= (row[h] >= 0 ? 1u : 0u) << h;
				row[h] += key & in_page;
			}
			pages_of(g + WARPS);
			const uint32_t slot = n % C::STAGES, bar = ptx::smem_u32(&ring->full[worker][slot]);
			if (n >= C::STAGES)
				dec_wait(ptx::smem_u32(&ring->empty[worker][slot]), st.status, (n / C::STAGES & 1u) ^ 1u);
			ring->there[worker][slot] = ok;
			const int rows = one ? ((ok & 1) ? C::GROUP : 0) : 16 * __popc(ok);
			ptx::mbar_arrive_expect_tx(bar, rows * (2 * C::ROW + (C::Q8 ? 8 : 0)));
			const uint32_t to = stages + (worker * C::STAGES + slot) * C::STAGE;
#pragma unroll
			for (int h = 0; h < C::HALVES; h++) {
				if (!(ok >> h & 1) || (h && one))
					continue;
				const uint32_t k_to = to + h * 16 * C::BOX_BYTES, v_to = k_to + C::GROUP * C::ROW;
				ptx::tma_load_3d(k_to, k_map, bar, 0, (int)row[h], 0);
				ptx::tma_load_3d(v_to, v_map, bar, 0, (int)row[h], 0);
				if constexpr (C::Q8) {
					const uint32_t f = factors + (worker * C::STAGES + slot) * C::FACTORS + 64 * h, bytes = one ? C::GROUP * 4 : 64;
					bulk_g2s(f, kv.k_scale + row[h], bytes, bar);
					bulk_g2s(f + 4 * C::GROUP, kv.v_scale + row[h], bytes, bar);
				}
			}
		}
		u += p.unit1 - p.unit0;
	}
}

// One warp's state over the groups of keys it takes: S^T = K Q^T and O^T = V^T P^T on m16n8k16, keys (then dims) on the
// 16-row side, query rows on the 8-column side, so that a single token's 8 heads fill the columns.  A lane holds rows
// 2c and 2c + 1 (c = lane % 4) of each block of 8.
template <int KIND, int D, int NB>
struct Warp {
	using C = Cfg<KIND, D>;
	static constexpr int KS = D / C::Q_STEP, MB = D / 16, H = C::HALVES;
	uint32_t q[NB][C::Q_PARTS][KS][2];
	float row_scale[NB][2];	 // scale * log2 e, and what the row's parts were divided by
	float acc[NB][MB][4];	 // Q8: in units of v_unit, apart: over the row's multiple of p (`more`)
	float m[NB][2], l[NB][2];  // running maximum (of the whole column), sum (of this lane's keys)
	float v_unit;		 // Q8: of the largest value factor so far (attn_unit_of)
	bool apart;		 // Q8: rows have units of their own

	__device__ __forceinline__ void begin(const AttnArgs &a, const SeqView &seq, int head_kv, int row0, int lane)
	{
		const int g = lane >> 2, c = lane & 3;
		const int n_rows = seq.n_tok * a.group;
#pragma unroll
		for (int nb = 0; nb < NB; nb++) {
			const int r = row0 + nb * 8 + g;
			const bool there = r < n_rows;
			const int tok = there ? r / a.group : 0;
			const float *src = a.q + ((long long)(seq.tok0 + tok) * a.n_head + head_kv * a.group + (there ? r - tok * a.group : 0)) * D;
			float top = 0.0f, up = 1.0f;
			if constexpr (C::Q8) {
				// Whole numbers of -127 * 2^16 .. 127 * 2^16 in units of the row's largest, as three signed bytes: bytes against bytes
				// need no expansion of the keys and their sums are exact.
				float4 v[KS][2];
#pragma unroll
				for (int j = 0; j < KS; j++)
#pragma unroll
					for (int h = 0; h < 2; h++) {
						const float4 f = there ? *reinterpret_cast<const float4 *>(src + 32 * j + 16 * h + 4 * c) : make_float4(0, 0, 0, 0);
						v[j][h] = f;
						top = fmaxf(fmaxf(fmaxf(top, fabsf(f.x)), fmaxf(fabsf(f.y), fabsf(f.z))), fabsf(f.w));
					}
				top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
				top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
				constexpr float MOST = 127.0f * 65536.0f;
				// (a row below 2^-100 of anything is brought up by two factors, since the inverse of its largest is no fp32 number)
				const float lift = top < 0x1p-100f ? 0x1p100f : 1.0f;
				const float down = top > 0.0f ? MOST / (top * lift) : 0.0f;
				up = top * (1.0f / MOST);
				bool odd = false;
#pragma unroll
				for (int j = 0; j < KS; j++)
#pragma unroll
					for (int h = 0; h < 2; h++) {
						const float x[4] = {v[j][h].x, v[j][h].y, v[j][h].z, v[j][h].w};
						uint32_t n[4];
#pragma unroll
						for (int i = 0; i < 4; i++) {
							odd = odd || !(fabsf(x[i]) <= FLT_MAX);
							// + 128 in each byte makes signed digits of them
							n[i] = (uint32_t)__float2int_rn(x[i] * lift * down) + 0x00808080u;
						}
#pragma unroll
						for (int p = 0; p < 3; p++) {  // the highest byte first
							const uint32_t s = p == 0 ? 0x0062 : p == 1 ? 0x0051 : 0x0040;
							q[nb][p][j][h] = (__byte_perm(n[0], n[1], s) & 0xffffu | __byte_perm(n[2], n[3], s) << 16) ^ 0x80808080u;
						}
					}
				// (by all lanes, whatever their own: a || would leave the shuffle out where it is true, and the others waiting)
				int any = odd;
				any |= __shfl_xor_sync(0xffffffffu, any, 1);
				any |= __shfl_xor_sync(0xffffffffu, any, 2);
				up = any ? __int_as_float(0x7fc00000) : up;  // a row with an infinity or NaN has no scores
			} else {
				float2 v[KS][2];
#pragma unroll
				for (int j = 0; j < KS; j++) {
					v[j][0] = there ? *reinterpret_cast<const float2 *>(src + 16 * j + 2 * c) : make_float2(0, 0);
					v[j][1] = there ? *reinterpret_cast<const float2 *>(src + 16 * j + 8 + 2 * c) : make_float2(0, 0);
#pragma unroll
					for (int h = 0; h < 2; h++)
						top = fmaxf(top, fmaxf(fabsf(v[j][h].x), fabsf(v[j][h].y)));
				}
				// fp16 parts: the row is brought to 1 .. 2 by a power of two (any fp32 row then keeps its 22 bits)
				float down = 1.0f;
				if constexpr (KIND != TIE_CUDA_KV_BF16) {
					top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
					top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
					const int e = min(max((int)(__float_as_uint(top) >> 23), 1), 253);
					if (top > 0.0f) {
						down = __uint_as_float((unsigned)(254 - e) << 23);
						up = __uint_as_float((unsigned)e << 23);
					}
				}
#pragma unroll
				for (int j = 0; j < KS; j++)
#pragma unroll
					for (int h = 0; h < 2; h++) {
						uint32_t part[C::PARTS];
						split_pair<KIND>(v[j][h].x * down, v[j][h].y * down, part);
#pragma unroll
						for (int p = 0; p < C::PARTS; p++)
							q[nb][p][j][h] = part[p];
					}
			}
#pragma unroll
			for (int i = 0; i < 2; i++) {
				row_scale[nb][i] = __shfl_sync(0xffffffffu, up, (2 * c + i) * 4) * a.scale_log2e;
				m[nb][i] = -INFINITY;
				l[nb][i] = 0.0f;
			}
#pragma unroll
			for (int mb = 0; mb < MB; mb++)
#pragma unroll
				for (int i = 0; i < 4; i++)
					acc[nb][mb][i] = 0.0f;
		}
		v_unit = ATTN_LEAST_UNIT;
		apart = false;
	}

	// The group of keys from key0 on, in shared memory at `stage`; keys at or behind key_end, and 16 of them whose bit of `there`
	// is not set, are nobody's.  more[..].w, while the rows have units of their own: what a row's p are multiplied by, v_unit over its unit.
	__device__ __forceinline__ void group(const AttnArgs &a, const StepView &st, const SeqView &seq, uint32_t stage, uint32_t factors, int key0, int key_end, unsigned there, int row0,
					      float4 *more, int lane)
	{
		const int g = lane >> 2, c = lane & 3;
		const uint32_t ks = stage, vs = stage + C::GROUP * C::ROW;
		float s[H][NB][4];
#pragma unroll
		for (int h = 0; h < H; h++) {
			const int krow = 16 * h + (lane & 15), kch = lane >> 4;
			if constexpr (C::Q8) {
				int part[NB][3][4];
#pragma unroll
				for (int nb = 0; nb < NB; nb++)
#pragma unroll
					for (int p = 0; p < 3; p++)
#pragma unroll
						for (int i = 0; i < 4; i++)
							part[nb][p][i] = 0;
#pragma unroll
				for (int j = 0; j < KS; j++) {
					uint32_t r[4];
					ldsm4(r, ks + C::place(krow, 2 * j + kch));
#pragma unroll
					for (int nb = 0; nb < NB; nb++)
#pragma unroll
						for (int p = 0; p < 3; p++)
							mma_bytes(part[nb][p], r, q[nb][p][j][0], q[nb][p][j][1]);
				}
#pragma unroll
				for (int nb = 0; nb < NB; nb++)
#pragma unroll
					for (int i = 0; i < 4; i++)
						s[h][nb][i] = fmaf((float)part[nb][0][i], 65536.0f, (float)(part[nb][1][i] * 256 + part[nb][2][i])) * row_scale[nb][i & 1];
			} else {
				float part[NB][C::PARTS][4];  // a chain each: the tensor cores cut every sum off
#pragma unroll
				for (int nb = 0; nb < NB; nb++)
#pragma unroll
					for (int p = 0; p < C::PARTS; p++)
#pragma unroll
						for (int i = 0; i < 4; i++)
							part[nb][p][i] = 0.0f;
#pragma unroll
				for (int j = 0; j < KS; j++) {
					uint32_t r[4];
					ldsm4(r, ks + C::place(krow, 2 * j + kch));
#pragma unroll
					for (int nb = 0; nb < NB; nb++)
#pragma unroll
						for (int p = 0; p < C::PARTS; p++)
							mma<KIND>(part[nb][p], r, q[nb][p][j][0], q[nb][p][j][1]);
				}
#pragma unroll
				for (int nb = 0; nb < NB; nb++)
#pragma unroll
					for (int i = 0; i < 4; i++) {
						float v = part[nb][C::PARTS - 1][i];
#pragma unroll
						for (int p = C::PARTS - 2; p >= 0; p--)
							v += part[nb][p][i];
						s[h][nb][i] = v * row_scale[nb][i & 1];
					}
			}
		}
		const bool masked = there != (1u << H) - 1u || key0 + C::GROUP > min(seq.kv_len, key_end);
		float f[H][2], unit_change = 1.0f;  // Q8: factors of the values, in units of v_unit
		if constexpr (C::Q8) {
			float top = 0.0f;
#pragma unroll
			for (int h = 0; h < H; h++)
#pragma unroll
				for (int i = 0; i < 2; i++) {
					const int k = 16 * h + 8 * i + g;
					const uint32_t at = factors + 4 * k;
					float kf;
					asm volatile("ld.shared.f32 %0, [%1];" : "=f"(kf) : "r"(at) : "memory");
					asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f[h][i]) : "r"(at + 4 * C::GROUP) : "memory");
#pragma unroll
					for (int nb = 0; nb < NB; nb++) {
						s[h][nb][2 * i] *= kf;
						s[h][nb][2 * i + 1] *= kf;
					}
					// (nobody's factor is none; an infinite one is as little a number as NaN, and NaN does not reach the largest)
					f[h][i] = key0 + k < key_end && (there >> h & 1) ? f[h][i] : 0.0f;
					f[h][i] = fabsf(f[h][i]) <= FLT_MAX ? f[h][i] : __int_as_float(0x7fc00000);
					top = fmaxf(top, fabsf(f[h][i]));
				}
			const float unit = attn_unit_of(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top))));
			if (unit > v_unit) {
				unit_change = v_unit * attn_unit_inverse(unit);
				v_unit = unit;
			}
			const float inv = attn_unit_inverse(v_unit);
#pragma unroll
			for (int h = 0; h < H; h++)
#pragma unroll
				for (int i = 0; i < 2; i++)
					f[h][i] *= inv;
		}
		if (masked) {
#pragma unroll
			for (int nb = 0; nb < NB; nb++)
#pragma unroll
				for (int i = 0; i < 2; i++) {
					const int r = row0 + nb * 8 + 2 * c + i, tok = min(r / a.group, seq.n_tok - 1);
					unsigned long long bits = 0;
					if (st.tree)
						bits = st.tree[seq.tok0 + tok];
#pragma unroll
					for (int h = 0; h < H; h++)
#pragma unroll
						for (int k = 0; k < 2; k++) {
							const int key = key0 + 16 * h + g + 8 * k, j = key - seq.kv_len;
							const bool sees =
								(there >> h & 1) && key < key_end && (j < 0 || (st.tree ? j < KV_MAX_TREE && (bits >> j & 1) : j <= tok));
							if (!sees)
								s[h][nb][2 * k + i] = -INFINITY;
						}
				}
		}
		if constexpr (C::Q8) {
			if (masked || apart) {
				bool far = false;
#pragma unroll
				for (int h = 0; h < H; h++)
#pragma unroll
					for (int i = 0; i < 2; i++)
						far = far || !(fabsf(f[h][i]) * ATTN_WIDE >= 1.0f || f[h][i] == 0.0f);  // (or no number)
				if (__builtin_expect(__any_sync(0xffffffffu, far), 0)) {
					if (!apart && lane < 8 * NB)
						more[lane].w = 1.0f;
					__syncwarp();
					apart = true;
					// (in the products below 0 times what is no number is 0, for the rows that do not see it)
#pragma unroll
					for (int h = 0; h < H; h++)
#pragma unroll
						for (int nb = 0; nb < NB; nb++)
#pragma unroll
							for (int i = 0; i < 4; i++)
								l[nb][i & 1] = s[h][nb][i] != -INFINITY && f[h][i >> 1] != f[h][i >> 1] ? f[h][i >> 1] : l[nb][i & 1];
				}
			}
		}
		uint32_t b[NB][H][C::PARTS][2];  // P^T as the second operand
		float alpha[NB][2];
#pragma unroll
		for (int nb = 0; nb < NB; nb++) {
			float base[2];
#pragma unroll
			for (int i = 0; i < 2; i++) {
				float top = m[nb][i];
#pragma unroll
				for (int h = 0; h < H; h++)
					top = fmaxf(top, fmaxf(s[h][nb][i], s[h][nb][2 + i]));
				top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
				top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
				top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
				base[i] = (top == -INFINITY ? 0.0f : top) - ATTN_P_SHIFT<KIND>;
				alpha[nb][i] = m[nb][i] == -INFINITY ? 0.0f : exp2_ftz(m[nb][i] - top);
				m[nb][i] = top;
				l[nb][i] *= alpha[nb][i];
			}
#pragma unroll
			for (int h = 0; h < H; h++) {
#pragma unroll
				for (int i = 0; i < 4; i++)
					s[h][nb][i] = exp2_ftz(s[h][nb][i] - base[i & 1]);
#pragma unroll
				for (int i = 0; i < 2; i++)
					l[nb][i] += s[h][nb][i] + s[h][nb][2 + i];
			}
			if constexpr (C::Q8) {
				if (__builtin_expect(apart, 0)) {
#pragma unroll
					for (int i = 0; i < 2; i++) {
						float most = 0.0f;
#pragma unroll
						for (int h = 0; h < H; h++)
#pragma unroll
							for (int k = 0; k < 2; k++)
								most = fmaxf(most, s[h][nb][2 * k + i] == 0.0f ? 0.0f : fabsf(f[h][k]));
						most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 4));
						most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 8));
						most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
						const float was = unit_change * attn_unit_inverse(more[nb * 8 + 2 * c + i].w);  // the row's unit, as a share of v_unit
						const float m = attn_unit_inverse(fmaxf(was, attn_unit_of(most)));
						alpha[nb][i] *= was * m;
						__syncwarp();
						if (lane < 4)
							more[nb * 8 + 2 * lane + i].w = m;
						// (a factor that is no number is nothing to a row that does not see it)
#pragma unroll
						for (int h = 0; h < H; h++)
#pragma unroll
							for (int k = 0; k < 2; k++)
								s[h][nb][2 * k + i] = s[h][nb][2 * k + i] == 0.0f ? 0.0f : s[h][nb][2 * k + i] * (f[h][k] * m);
					}
				} else {
					alpha[nb][0] *= unit_change;
					alpha[nb][1] *= unit_change;
#pragma unroll
					for (int h = 0; h < H; h++)
#pragma unroll
						for (int i = 0; i < 4; i++)
							s[h][nb][i] *= f[h][i >> 1];
				}
			}
#pragma unroll
			for (int h = 0; h < H; h++)
#pragma unroll
				for (int k = 0; k < 2; k++) {
					uint32_t part[C::PARTS];
					split_pair<KIND>(s[h][nb][2 * k], s[h][nb][2 * k + 1], part);
#pragma unroll
					for (int p = 0; p < C::PARTS; p++)
						b[nb][h][p][k] = transpose8x8(part[p]);
				}
		}
		if constexpr (!C::Q8) {
			// 0 * infinity is not nothing: where a group that not every row sees holds values that are no numbers, nobody's (stale
			// slots) become zeros, and the products of the others are made one by one
			bool odd = false, cleared = false;
			if (masked) {
				constexpr uint32_t EXPONENT = KIND == TIE_CUDA_KV_F16 ? 0x7c00u : 0x7f80u;
				for (int i = lane; i < C::GROUP * C::ROW / 4; i += 32) {
					const int k = (4 * i & (C::PANEL - 1)) >> 7;
					uint32_t w;
					asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(vs + 4 * i) : "memory");
					if (!nonfinite16(w, EXPONENT))
						continue;
					if (key0 + k < key_end && (there >> (k >> 4) & 1)) {
						odd = true;
					} else {
						asm volatile("st.shared.u32 [%0], %1;" ::"r"(vs + 4 * i), "r"(0u) : "memory");
						cleared = true;
					}
				}
				if (cleared)
					ptx::fence_proxy_async_smem();	// (the next values come in over these stores)
				odd = __any_sync(0xffffffffu, odd);
				__syncwarp();
			}
			if (odd) {
				one_by_one(a, st, seq, vs, s, alpha, key0, key_end, there, row0, lane);
				return;
			}
		}
#pragma unroll
		for (int mb = 0; mb < MB; mb += C::Q8 ? 2 : 1) {
			uint32_t f[C::Q8 ? 2 : 1][H][4];
#pragma unroll
			for (int h = 0; h < H; h++) {
				if constexpr (C::Q8) {
					uint32_t r[4];	// (keys 0-7, 8-15) of 16 dims, then of the next 16; a unit of 16 bits is two neighbouring dims
					ldsm4_trans(r, vs + C::place(16 * h + (lane & 15), mb + (lane >> 4)));
#pragma unroll
					for (int i = 0; i < 4; i++)
						r[i] ^= 0x80808080u;
#pragma unroll
					for (int k = 0; k < 2; k++) {
						f[k][h][0] = int8_pair_low<0x4240>(r[2 * k]);
						f[k][h][1] = int8_pair_low<0x4341>(r[2 * k]);
						f[k][h][2] = int8_pair_low<0x4240>(r[2 * k + 1]);
						f[k][h][3] = int8_pair_low<0x4341>(r[2 * k + 1]);
					}
				} else {
					ldsm4_trans(f[0][h], vs + C::place(16 * h + (lane & 7) + 8 * (lane >> 4), 2 * mb + (lane >> 3 & 1)));
				}
			}
			// acc = acc * alpha + (the group's products, summed up from zero, lo parts first: the tensor cores cut sums off)
#pragma unroll
			for (int k = 0; k < (C::Q8 ? 2 : 1); k++)
#pragma unroll
				for (int nb = 0; nb < NB; nb++) {
					float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
					for (int p = C::PARTS - 1; p >= 0; p--)
#pragma unroll
						for (int h = 0; h < H; h++)
							mma<KIND>(d, f[k][h], b[nb][h][p][0], b[nb][h][p][1]);
#pragma unroll
					for (int i = 0; i < 4; i++)
						acc[nb][mb + k][i] = fmaf(acc[nb][mb + k][i], alpha[nb][i & 1], d[i]);
				}
		}
	}

	// dim of acc[..][mb][i]
	__device__ static __forceinline__ int dim(int mb, int i, int lane)
	{
		return C::Q8 ? 16 * mb + 2 * (lane >> 2) + (i >> 1) : 16 * mb + (lane >> 2) + 8 * (i >> 1);
	}

	__device__ __forceinline__ void one_by_one(const AttnArgs &a, const StepView &st, const SeqView &seq, uint32_t vs, const float (&p)[H][NB][4],
						   const float (&alpha)[NB][2], int key0, int key_end, unsigned there, int row0, int lane)
	{
		int tok[NB][2];
		unsigned long long bits[NB][2];
#pragma unroll
		for (int nb = 0; nb < NB; nb++)
#pragma unroll
			for (int i = 0; i < 2; i++) {
				tok[nb][i] = min((row0 + nb * 8 + 2 * (lane & 3) + i) / a.group, seq.n_tok - 1);
				bits[nb][i] = st.tree ? st.tree[seq.tok0 + tok[nb][i]] : 0;
			}
#pragma unroll
		for (int nb = 0; nb < NB; nb++)
#pragma unroll
			for (int mb = 0; mb < MB; mb++)
#pragma unroll
				for (int i = 0; i < 4; i++)
					acc[nb][mb][i] *= alpha[nb][i & 1];
#pragma unroll 1
		for (int k = 0; k < C::GROUP && key0 + k < key_end; k++) {
			if (!(there >> (k >> 4) & 1))
				continue;
			const int j = key0 + k - seq.kv_len;
			float pk[NB][2];
			bool sees[NB][2];
#pragma unroll
			for (int nb = 0; nb < NB; nb++)
#pragma unroll
				for (int i = 0; i < 2; i++) {
					float mine = k & 8 ? p[0][nb][2 + i] : p[0][nb][i];
					if (H == 2 && k >= 16)
						mine = k & 8 ? p[H - 1][nb][2 + i] : p[H - 1][nb][i];
					pk[nb][i] = __shfl_sync(0xffffffffu, mine, (k & 7) * 4 + (lane & 3));
					sees[nb][i] = j < 0 || (st.tree ? j < KV_MAX_TREE && (bits[nb][i] >> j & 1) : j <= tok[nb][i]);
				}
#pragma unroll
			for (int mb = 0; mb < MB; mb++)
#pragma unroll
				for (int h = 0; h < 2; h++) {
					const int d = dim(mb, 2 * h, lane);
					uint16_t raw;
					asm volatile("ld.shared.u16 %0, [%1];" : "=h"(raw) : "r"(vs + C::place(k, d >> 3) + 2 * (d & 7)) : "memory");
					const float v = KIND == TIE_CUDA_KV_F16 ? __half2float(__ushort_as_half(raw)) : __uint_as_float((uint32_t)raw << 16);
#pragma unroll
					for (int nb = 0; nb < NB; nb++)
#pragma unroll
						for (int i = 0; i < 2; i++)
							if (sees[nb][i])
								acc[nb][mb][2 * h + i] = fmaf(pk[nb][i], v, acc[nb][mb][2 * h + i]);
				}
		}
	}
};

template <int KIND, int D, int NB>
constexpr size_t smem_bytes()
{
	using C = Cfg<KIND, D>;
	return (size_t)WARPS * C::STAGES * (C::STAGE + C::FACTORS) + (size_t)WARPS / 2 * 8 * D * 4 + 1024;
}

// One CTA per SM, each an equal share of the launch's units of 128 keys; a worker warp takes every eighth group of 16 or 32 keys
// through a ring of its own, so that no warp waits for another until the sums are joined.  Bound by HBM where there is much
// to read (48 tokens over 20,000 slots each, F16: 313 us, 6.3 TB/s; over 5000: 73 us, 5.2 TB/s; one token over 100,003, Q8: 31
// us, 3.4 TB/s: 4 us until the first keys are there, 8 from the last ones to the joined row) and by one chain of latencies
// where there is little (one token over 500: 11.0 us, launch and call included).
template <int KIND, int D, int NB>
__global__ void __launch_bounds__(THREADS, 1) attn_rows(const KvView kv, const StepView st, const AttnArgs a, const __grid_constant__ CUtensorMap k_map,
							const __grid_constant__ CUtensorMap v_map)
{
	using C = Cfg<KIND, D>;
	constexpr int ROWS = 8 * NB, D4 = D / 4, UNIT_GROUPS = ATTN_UNIT / C::GROUP;
	extern __shared__ uint8_t smem_raw[];
	__shared__ AttnWork work;
	__shared__ Ring<KIND, D> ring;
	__shared__ float4 s_row[WARPS][ROWS];  // each warp's: maximum of a row, sum of p, unit of the sums; `more` of Warp::group
	__shared__ float2 s_all[ROWS];	       // maximum and sum of p of all
	__shared__ float s_w[ROWS][WARPS];		      // what a warp's sums count for
	const uint32_t stages = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u, factors = stages + WARPS * C::STAGES * C::STAGE;
	// [half of the warps][8 rows][D]: sums on their way together
	float *sums = reinterpret_cast<float *>(smem_raw + (factors - ptx::smem_u32(smem_raw)) + WARPS * C::STAGES * C::FACTORS);
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, cta = blockIdx.x;
	if (threadIdx.x == 0) {
		for (int w = 0; w < WARPS; w++)
			for (int i = 0; i < C::STAGES; i++) {
				ptx::mbar_init(ptx::smem_u32(&ring.full[w][i]), 1);
				ptx::mbar_init(ptx::smem_u32(&ring.empty[w][i]), 1);
			}
		ptx::fence_barrier_init();
		ptx::fence_proxy_async_smem();
	}
	attn_share_work<THREADS>(work, kv, st, [&](const SeqView &q) { return attn_items(kv, a, q, ROWS) * attn_units(q); });
	const long long total = work.start[st.n_seq];
	const int n_cta = (int)min((long long)gridDim.x, total);  // (each of them has a unit at least)
	if (cta >= n_cta)
		return;
	const long long u_begin = attn_div(total * cta, n_cta), u_end = attn_div(total * (cta + 1), n_cta);
	if (warp >= WARPS) {
		const int worker = (warp - WARPS) * EACH + lane % EACH;
		request<KIND, D, ROWS>(&ring, stages, factors, u_begin, u_end, work, kv, st, a, &k_map, &v_map, worker, lane < EACH);
		return;
	}
	Warp<KIND, D, NB> w;
	uint32_t taken = 0;
	for (long long u = u_begin; u < u_end;) {
		const Piece p = piece_at<ROWS>(u, u_end, work, kv, st, a);
		const SeqView seq = p.seq;
		if (st.tree && seq.n_tok > KV_MAX_TREE && threadIdx.x == 0)
			kv_report(st, ST_BAD_STEP);
		const int g_end = min(p.unit1 * UNIT_GROUPS, (p.key_end + C::GROUP - 1) / C::GROUP);
		w.begin(a, seq, p.head, p.row0, lane);
		for (int g = p.unit0 * UNIT_GROUPS + warp; g < g_end; g += WARPS, taken++) {
			const uint32_t slot = taken % C::STAGES, at = warp * C::STAGES + slot;
			dec_wait(ptx::smem_u32(&ring.full[warp][slot]), st.status, taken / C::STAGES & 1u);
			w.group(a, st, seq, stages + at * C::STAGE, factors + at * C::FACTORS, g * C::GROUP, p.key_end, ring.there[warp][slot], p.row0, s_row[warp], lane);
			__syncwarp();
			if (lane == 0)
				ptx::mbar_arrive(ptx::smem_u32(&ring.empty[warp][slot]));
		}

		// the warps' keys together
#pragma unroll
		for (int nb = 0; nb < NB; nb++)
#pragma unroll
			for (int i = 0; i < 2; i++) {
				float sum = w.l[nb][i];
				sum += __shfl_xor_sync(0xffffffffu, sum, 4);
				sum += __shfl_xor_sync(0xffffffffu, sum, 8);
				sum += __shfl_xor_sync(0xffffffffu, sum, 16);
				if (lane < 4) {
					float4 &to = s_row[warp][nb * 8 + 2 * lane + i];
					to = make_float4(w.m[nb][i], sum, !C::Q8 ? 1.0f : ATTN_Q8_DOWN * (w.apart ? w.v_unit * attn_unit_inverse(to.w) : w.v_unit), 0.0f);
				}
			}
		auto weigh = [&](int r) {
			float top = -INFINITY, sum = 0.0f;
#pragma unroll
			for (int i = 0; i < WARPS; i++)
				top = fmaxf(top, s_row[i][r].x);
#pragma unroll
			for (int i = 0; i < WARPS; i++) {
				const float4 v = s_row[i][r];
				const float f = v.x == -INFINITY ? 0.0f : exp2_ftz(v.x - top);
				s_w[r][i] = C::Q8 ? f * v.z : f;
				sum = fmaf(v.y, f, sum);
			}
			s_all[r] = make_float2(top, sum);
		};
		workers_sync();
		if (threadIdx.x < ROWS)
			weigh(threadIdx.x);
		workers_sync();
		const bool whole = p.unit0 == 0 && p.unit1 == p.item_units;
		const int n_rows = seq.n_tok * a.group;
		float *part = a.part + (2 * cta + (p.unit0 == 0 ? 1 : 0)) * attn_part_floats(MAX_ROWS);
		auto out_row = [&](int r) {
			const int tok = r / a.group;
			return a.out + ((long long)(seq.tok0 + tok) * a.n_head + p.head * a.group + (r - tok * a.group)) * D;
		};
		auto finished = [](float4 y, float sum) {
			const float inv = sum == 0.0f ? 0.0f : (C::Q8 ? ATTN_Q8_UP : 1.0f) / sum;
			return make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
		};
		// 8 rows: the later warps' sums to the earlier ones, and these by all threads (4 dims of a row each)
		auto together = [&](auto give, auto take) {
#pragma unroll
			for (int half = 1; half >= 0; half--) {
				if ((warp >= WARPS / 2) == (half == 1))
					give(sums + warp % (WARPS / 2) * 8 * D, half == 0);
				workers_sync();
			}
			for (int i = threadIdx.x; i < 8 * D4; i += WORKERS) {
				float4 y = make_float4(0, 0, 0, 0);
#pragma unroll
				for (int k = 0; k < WARPS / 2; k++) {
					const float4 v = *reinterpret_cast<const float4 *>(sums + (k * 8 + i / D4) * D + i % D4 * 4);
					y = make_float4(y.x + v.x, y.y + v.y, y.z + v.z, y.w + v.w);
				}
				take(i / D4, i % D4 * 4, y);
			}
			workers_sync();
		};
#pragma unroll
		for (int nb = 0; nb < NB; nb++)
			together(
				[&](float *to, bool add) {
#pragma unroll
					for (int i = 0; i < 2; i++) {
						const int r = 2 * (lane & 3) + i;
						const float f = s_w[nb * 8 + r][warp];
#pragma unroll
						for (int mb = 0; mb < D / 16; mb++)
#pragma unroll
							for (int h = 0; h < 2; h++) {
								float &d = to[r * D + w.dim(mb, 2 * h, lane)];
								const float v = w.acc[nb][mb][2 * h + i] * f;
								d = add ? d + v : v;
							}
					}
				},
				[&](int r8, int col, float4 y) {
					const int r = nb * 8 + r8;
					if (!whole) {
						*reinterpret_cast<float4 *>(part + r * D + col) = y;
					} else if (p.row0 + r < n_rows) {
						*reinterpret_cast<float4 *>(out_row(p.row0 + r) + col) = finished(y, s_all[r].y);
					}
				});
		if (!whole) {
			if (threadIdx.x < ROWS)
				reinterpret_cast<float2 *>(part + MAX_ROWS * 128)[threadIdx.x] = s_all[threadIdx.x];
			// the CTAs of the item: those of its first and last unit, and all between
			const int c0 = attn_cta_of(p.first_unit, total, n_cta), c1 = attn_cta_of(p.first_unit + p.item_units - 1, total, n_cta), n = c1 - c0 + 1;
			__threadfence();
			workers_sync();
			if (threadIdx.x == 0)
				work.last = atomicAdd(a.count + c0, 1u) == (unsigned)(c1 - c0);
			workers_sync();
			if (work.last) {
				// Joined in the order of the CTAs: warp w takes parts w, w + 8 .. of 8 rows (a lane 4 dims), then the warps' sums.
				__threadfence();
				auto at = [&](int i) { return a.part + (size_t)(2 * (c0 + i) + (i == 0 ? 1 : 0)) * attn_part_floats(MAX_ROWS); };
				constexpr int PER = 32 / D4, STEPS = 8 / PER;  // rows at once
#pragma unroll 1
				for (int nb = 0; nb < NB; nb++) {
					float4 sum[STEPS];
					float top[STEPS], l[STEPS];
#pragma unroll
					for (int k = 0; k < STEPS; k++) {
						sum[k] = make_float4(0, 0, 0, 0);
						top[k] = -INFINITY;
						l[k] = 0.0f;
					}
					for (int i = warp; i < n; i += WARPS) {
						const float *src = at(i);
						float4 v[STEPS];
						float2 of[STEPS];
#pragma unroll
						for (int k = 0; k < STEPS; k++) {
							const int r = nb * 8 + k * PER + lane / D4;
							v[k] = __ldcg(reinterpret_cast<const float4 *>(src + r * D) + lane % D4);
							of[k] = __ldcg(reinterpret_cast<const float2 *>(src + MAX_ROWS * 128) + r);
						}
#pragma unroll
						for (int k = 0; k < STEPS; k++) {
							const float next = fmaxf(top[k], of[k].x);
							const float f = of[k].x == -INFINITY ? 0.0f : exp2_ftz(of[k].x - next), o = top[k] == -INFINITY ? 0.0f : exp2_ftz(top[k] - next);
							top[k] = next;
							l[k] = fmaf(of[k].y, f, l[k] * o);
							sum[k] = make_float4(fmaf(v[k].x, f, sum[k].x * o), fmaf(v[k].y, f, sum[k].y * o), fmaf(v[k].z, f, sum[k].z * o),
									     fmaf(v[k].w, f, sum[k].w * o));
						}
					}
#pragma unroll
					for (int k = 0; k < STEPS; k++)
						if (lane % D4 == 0)
							s_row[warp][k * PER + lane / D4] = make_float4(top[k], l[k], 1.0f, 0.0f);
					workers_sync();
					if (threadIdx.x < 8)
						weigh(threadIdx.x);
					workers_sync();
					together(
						[&](float *to, bool add) {
#pragma unroll
							for (int k = 0; k < STEPS; k++) {
								const int r = k * PER + lane / D4;
								const float f = s_w[r][warp];
								float4 *d = reinterpret_cast<float4 *>(to + r * D) + lane % D4;
								const float4 o = add ? *d : make_float4(0, 0, 0, 0);
								*d = make_float4(fmaf(sum[k].x, f, o.x), fmaf(sum[k].y, f, o.y), fmaf(sum[k].z, f, o.z), fmaf(sum[k].w, f, o.w));
							}
						},
						[&](int r8, int col, float4 y) {
							const int r = p.row0 + nb * 8 + r8;
							if (r >= n_rows)
								return;
							*reinterpret_cast<float4 *>(out_row(r) + col) = finished(y, s_all[r8].y);
						});
				}
				if (threadIdx.x == 0)
					a.count[c0] = 0;  // at rest again
			}
		}
		u += p.unit1 - p.unit0;
	}
}

template <int KIND, int D, int NB>
int go(tie_cuda_ctx *c, const KvView &kv, const StepView &st, const AttnArgs &a)
{
	using C = Cfg<KIND, D>;
	CUtensorMap map[2];
	const int rc = attn_maps(c, kv, C::Q8 ? 1 : 2, D, C::BOX_BYTES, C::GROUP, C::ROW == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, map);
	if (rc)
		return rc;
	attn_rows<KIND, D, NB><<<c->sm_count, THREADS, smem_bytes<KIND, D, NB>(), c->stream>>>(kv, st, a, map[0], map[1]);
	TIE_CUDA_LAUNCHED(c);
	return TIE_CUDA_OK;
}
template <int KIND, int D, int NB>
int allow_smem(tie_cuda_ctx *c)
{
	TIE_CUDA_TRY(c, cudaFuncSetAttribute(attn_rows<KIND, D, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes<KIND, D, NB>()));
	return TIE_CUDA_OK;
}
template <int KIND>
int allow_smem_all(tie_cuda_ctx *c)
{
	int rc = allow_smem<KIND, 128, 1>(c);
	rc = rc ? rc : allow_smem<KIND, 128, 2>(c);
	rc = rc ? rc : allow_smem<KIND, 64, 1>(c);
	return rc ? rc : allow_smem<KIND, 64, 2>(c);
}
template <int KIND>
int go_kind(tie_cuda_ctx *c, const KvView &kv, const StepView &st, int head_dim, bool two, const AttnArgs &a)
{
	if (head_dim == 128)
		return two ? go<KIND, 128, 2>(c, kv, st, a) : go<KIND, 128, 1>(c, kv, st, a);
	return two ? go<KIND, 64, 2>(c, kv, st, a) : go<KIND, 64, 1>(c, kv, st, a);
}

}  // namespace

// Maps of keys and values: boxes of up to box_rows rows of a page x the whole row, box_bytes of it side by side (the shared-memory
// row that is swizzled), the next box_bytes of all rows behind these; of pages with fewer rows, one of these panels a box.
int attn_maps(tie_cuda_ctx *c, const KvView &kv, int elem, int head_dim, int box_bytes, int box_rows, CUtensorMapSwizzle swizzle, CUtensorMap *map)
{
	const size_t rows = ((size_t)kv.n_pages * kv.n_head_kv) << kv.page_shift;
	const int n = 1 << kv.page_shift < box_rows ? 1 << kv.page_shift : box_rows;
	const CUtensorMapDataType type = elem == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
	for (int i = 0; i < 2; i++) {
		const int rc = tc_encode_panels(c, &map[i], type, elem, i ? kv.v : kv.k, rows, head_dim, box_bytes / elem, n,
						n == box_rows ? head_dim * elem / box_bytes : 1, swizzle);
		if (rc)
			return rc;
	}
	return TIE_CUDA_OK;
}

size_t attn_scratch_floats(const tie_cuda_ctx *c)
{
	return 2 * c->sm_count * attn_part_floats(ATTN_MAX_ROWS);
}

int attn_setup(tie_cuda_ctx *c)
{
	int rc = allow_smem_all<TIE_CUDA_KV_F16>(c);
	rc = rc ? rc : allow_smem_all<TIE_CUDA_KV_BF16>(c);
	rc = rc ? rc : allow_smem_all<TIE_CUDA_KV_Q8>(c);
	return rc ? rc : attn_tc_setup(c);
}

int launch_attn(tie_cuda_ctx *c, const KvView &kv, const StepView &st, int kind, int head_dim, const float *q, float *out, int n_head, float scale)
{
	AttnArgs a = {q, out, n_head, n_head / kv.n_head_kv, scale * ATTN_LOG2E, c->s.attn_part, c->s.attn_count, c->s.attn_join};
	// Rows of a sequence and key/value head, on average: up to 8 and up to 16 in tiles of that.  More go in tiles of 128, which
	// read the cache once for all of them but take 22 us for the least: where the page table has no room for more slots than
	// leave a tile of 16 rows and 128 keys to each SM, those are done sooner (12 tokens of 8 heads, F16: 12.9 us where tiles of
	// 128 take 27.8 with 100 slots in front, 17.9 and 23.3 with 500, 30.8 and 23.6 with 1000, 29.3 and 24.4 with 2000).  What the host
	// does not see decides neither: a table of 4096 slots over 100 used ones takes the 27.8.
	// A step of both kinds goes one way as a whole.  A piece of 512 beside single tokens, F16 / Q8, over the sum of both by
	// themselves: 47 over 4000 slots 171 us of 172 / 224 of 170; 250 over 1000 (tiles) 187 of 156 / 212 of 142; 700 over 1000 (few rows)
	// 751 of 306 / 624 of 270.
	const long long rows = ((long long)st.n_tokens * a.group + st.n_seq - 1) / st.n_seq;
	if (rows > 16) {
		const long long tiles = ((long long)st.n_tokens * a.group + 15) / 16 + st.n_seq - 1;
		const long long units = (((long long)st.max_pages << kv.page_shift) + ATTN_UNIT - 1) / ATTN_UNIT;
		if (tiles * kv.n_head_kv * units > c->sm_count)
			return launch_attn_tc(c, kv, st, kind, head_dim, a);
	}
	const bool two = rows > 8;
	if (kind == TIE_CUDA_KV_F16)
		return go_kind<TIE_CUDA_KV_F16>(c, kv, st, head_dim, two, a);
	if (kind == TIE_CUDA_KV_BF16)
		return go_kind<TIE_CUDA_KV_BF16>(c, kv, st, head_dim, two, a);
	return go_kind<TIE_CUDA_KV_Q8>(c, kv, st, head_dim, two, a);
}

}  // namespace tie
