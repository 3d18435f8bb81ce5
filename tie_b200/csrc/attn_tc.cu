// Attention over the paged cache for sequences with many query rows per key/value head (trees of drafted tokens, prompt
// pieces): tiles of 128 rows x 128 keys on tcgen05.
//
//   S = Q K^T, P = exp2(S - max), O = P V      rows (token, head of the group) on the 128 lanes of tensor memory
//
// fp32 results need more than one 16-bit operand per value: Q and P are fp16 hi + lo (22 bits), two MMAs each, against
// keys and values that are exact in fp16 (F16; Q8's whole numbers; BF16 rows brought to fp16 by a power of two), the factors
// of rows applied in fp32.  The products of a tile start from zero and are added to fp32 registers: the tensor cores cut
// every sum off, which over a long cache would add up.
//
// One CTA per SM, 512 threads:
//   * two warpgroups of softmax threads, a thread per row, take key tiles in turn, each with a running maximum, sum and
//     output row of its own (joined at the end), so that one's exponentials run under the other's MMAs;
//   * two warps load keys, two values: cp.async into the swizzled operand layout (pages of 16 slots and more, zeros behind
//     the last key), expanded to fp16 in place where the cache has another type;
//   * one thread issues the MMAs.  Q and P are operands in tensor memory (a step of shared memory then feeds only the 128
//     keys or dims of its other operand: half of what the memory delivers); P's parts of 16 keys take the columns of these keys' scores.
// Tensor memory: Q 128 columns, two score tiles, O: all 512.  Every wait is bounded, as in tensor.cu; after a
// time-out no wait waits any more and all roles run to their ends.
#include <float.h>

#include "attn.cuh"
#include "kernels.cuh"
#include "tc_ptx.cuh"

namespace tie {
namespace {

constexpr int ROWS = ATTN_MAX_ROWS, TILE = ATTN_UNIT;
constexpr int THREADS = 512, SOFT_THREADS = 256, LOAD_THREADS = 64;
constexpr int W_KEYS = 8, W_VALUES = 10, W_MMA = 12;  // first warps of the roles behind the softmax warps
constexpr int SOFT_REGS = 192, LOAD_REGS = 80, MMA_REGS = 48;
static_assert(2 * SOFT_REGS + LOAD_REGS + MMA_REGS <= 512, "a launch of 512 threads holds 128 registers a thread");
constexpr int COL_Q = 0, COL_S = 128, COL_O = 384;
constexpr uint32_t PANEL = TILE * 128;	// bytes of 64 dims of a tile: 128 rows of 128 bytes
constexpr long long WAIT_CYCLES = 1ll << 30;

struct Shared {
	uint64_t k_full[2], k_free[2], v_full[2], v_free[2];
	uint64_t s_full[2], p_full[2], o_full[2], o_free, q_full, fin;  // (o_full: a warpgroup's own, so that it waits for every phase)
	// What the softmax threads need to know of a tile's keys outlives its operand slot, which is free once the scores are
	// made.  Tile n + 4 is requested after the scores of n + 2, these after the products of n, whose P then has been made.
	uint64_t f_full[4];
	uint32_t bad[4];	  // groups of 16 keys of a tile whose page does not exist
	alignas(16) float k_scale[4][TILE];
	alignas(16) float v_raw[2][TILE], v_scale[2][TILE];
	float v_top[2];
	uint32_t odd[2][2];	  // a masked tile's values hold one that is no number (per loading warp)
	uint32_t tmem_base, abort;
	float load_max[2][2];
	float q_max[2][ROWS];
	float2 ml[2][ROWS];
};

// The n-th piece of work of this CTA: an item, or (few items: shared) some units of one.
struct Piece {
	SeqView seq;
	int s, head, row0;
	int unit0, unit1, item_units;
	int n_tiles;	// from unit0 on: tiles that some row of the item sees keys of
	int key_end;	// first key that nobody sees
	int all_see;	// keys in front of this one are seen by every row
};
struct Walk {
	bool shared;
	long long total, u, u_end;
	int n_cta, round;
};

__device__ __forceinline__ void finish_piece(Piece &p, const StepView &st, const AttnArgs &a)
{
	const int first_tok = p.row0 / a.group, last_tok = min((p.row0 + ROWS - 1) / a.group, p.seq.n_tok - 1);
	p.key_end = p.seq.kv_len + (st.tree ? p.seq.n_tok : last_tok + 1);
	p.all_see = p.seq.kv_len + (st.tree ? 0 : first_tok + 1);
	p.n_tiles = max(0, min(p.unit1, (p.key_end + TILE - 1) / TILE) - p.unit0);
}

__device__ bool next_piece(Walk &w, Piece &p, const AttnWork &work, const KvView &kv, const StepView &st, const AttnArgs &a)
{
	if (w.shared) {
		if (w.u >= w.u_end)
			return false;
		p.s = attn_sequence_of(work, st.n_seq, w.u);
		p.seq = kv_sequence(st, kv.page_shift, p.s);
		const int tiles = (int)(((long long)p.seq.n_tok * a.group + ROWS - 1) / ROWS);
		p.item_units = attn_units(p.seq);
		const long long in_seq = w.u - work.start[p.s], item = in_seq / p.item_units;
		p.unit0 = (int)(in_seq - item * p.item_units);
		p.unit1 = (int)min((long long)p.item_units, p.unit0 + (w.u_end - w.u));
		p.head = (int)(item / tiles);
		p.row0 = (int)(item % tiles) * ROWS;
		w.u += p.unit1 - p.unit0;
	} else {
		// whole items, a sequence's last rows (the ones that see most) first, there and back over the CTAs
		long long i;
		do {
			if ((long long)w.round * w.n_cta >= w.total)
				return false;
			i = (w.round & 1) ? (long long)(w.round + 1) * w.n_cta - 1 - blockIdx.x : (long long)w.round * w.n_cta + blockIdx.x;
			w.round++;
		} while (i >= w.total);
		p.s = attn_sequence_of(work, st.n_seq, i);
		p.seq = kv_sequence(st, kv.page_shift, p.s);
		const int tiles = (int)(((long long)p.seq.n_tok * a.group + ROWS - 1) / ROWS);
		const int in_seq = (int)(i - work.start[p.s]);
		p.row0 = (tiles - 1 - in_seq / kv.n_head_kv) * ROWS;
		p.head = in_seq % kv.n_head_kv;
		p.unit0 = 0;
		p.unit1 = p.item_units = attn_units(p.seq);
	}
	finish_piece(p, st, a);
	return true;
}

template <int KIND, int D>
struct Tile {
	static constexpr bool SCALED = KIND != TIE_CUDA_KV_F16;
	static constexpr int ROW = KIND == TIE_CUDA_KV_Q8 ? D : 2 * D;	// bytes of a head row of the cache
	static constexpr int CHUNKS = ROW / 16;
	static constexpr uint32_t BYTES = TILE * D * 2;
	// where a 16-byte chunk of row r's fp16 values lies in the operand tile
	__device__ static __forceinline__ uint32_t place(int r, int ch) { return (ch >> 3) * PANEL + r * 128 + (((ch & 7) ^ (r & 7)) << 4); }
	// ... and where it comes in: packed bytes lie in the last panel until they are expanded
	__device__ static __forceinline__ uint32_t raw(int r, int ch)
	{
		return KIND == TIE_CUDA_KV_Q8 ? (D == 128 ? PANEL : 0u) + r * 128 + ((ch ^ (r & 7)) << 4) : place(r, ch);
	}
};

__device__ __forceinline__ uint4 lds128(uint32_t at)
{
	uint4 v;
	asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
	return v;
}
__device__ __forceinline__ void sts128(uint32_t at, uint4 v)
{
	asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
template <int ID, int N>
__device__ __forceinline__ void bar_sync()
{
	asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(N) : "memory");
}

// Bounded; true once the barrier's phase is complete.
struct Waiter {
	volatile uint32_t *abort;
	unsigned *status;
	__device__ __forceinline__ bool operator()(uint64_t &bar, uint32_t parity) const
	{
		const uint32_t b = ptx::smem_u32(&bar);
		if (ptx::mbar_try_wait(b, parity))
			return true;
		const long long t0 = clock64();
		while (!ptx::mbar_try_wait_suspend(b, parity, 20000u)) {
			if (*abort)
				return false;
			if (clock64() - t0 > WAIT_CYCLES) {
				atomicOr(status, ST_WAIT_TIMEOUT);
				*abort = 1;
				return false;
			}
		}
		return true;
	}
};

// fp16 hi and lo of a pair
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo)
{
	const __half2 h = __floats2half2_rn(a, b);
	const float2 f = __half22float2(h);
	const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
	hi = *reinterpret_cast<const uint32_t *>(&h);
	lo = *reinterpret_cast<const uint32_t *>(&l);
}

// The loading warps of keys (VALUES false) or values: 64 threads.
template <int KIND, int D, bool VALUES>
struct Loader {
	using T = Tile<KIND, D>;
	const KvView &kv;
	const StepView &st;
	Shared *sh;
	uint32_t ring;	// two operand tiles
	int t, lane;

	// Requests tile `unit` of piece p, this CTA's n-th.
	__device__ __forceinline__ void issue(const Piece &p, int unit, uint32_t n)
	{
		const uint32_t slot = n & 1u;
		const uint8_t *rows = VALUES ? kv.v : kv.k;
		const int key0 = unit * TILE, page_mask = (1 << kv.page_shift) - 1, grp = lane & 7;
		// a lane finds the row of one group of 16 keys
		long long first = -1;
		const int gkey = key0 + grp * 16;
		if (gkey < p.key_end) {
			first = kv_page_row(kv, st, st.page_table[(long long)p.s * st.max_pages + (gkey >> kv.page_shift)], p.head);
			if (first >= 0)
				first += gkey & page_mask;
		}
		const uint32_t bad = __ballot_sync(0xffffffffu, gkey < p.key_end && first < 0) & 0xffu;
		if (!VALUES && t == 0)
			sh->bad[n & 3u] = bad;
		const uint32_t dst = ring + slot * T::BYTES;
		constexpr int AT_ONCE = LOAD_THREADS / T::CHUNKS, PASSES = TILE / AT_ONCE, PER_GROUP = 16 / AT_ONCE;
		const int ch = t % T::CHUNKS, r0 = t / T::CHUNKS;
#pragma unroll
		for (int i = 0; i < PASSES; i++) {
			const int r = r0 + i * AT_ONCE;
			const long long row = __shfl_sync(0xffffffffu, first, AT_ONCE <= 16 ? i / (PER_GROUP ? PER_GROUP : 1) : r >> 4);
			const bool in = row >= 0 && key0 + r < p.key_end;
			cp_async16_or_zero(dst + T::raw(r, ch), rows + (in ? (row + (r & 15)) * T::ROW + ch * 16 : 0), in);
		}
		if constexpr (KIND == TIE_CUDA_KV_Q8) {
			const float *scales = VALUES ? kv.v_scale : kv.k_scale;
			const uint32_t to = ptx::smem_u32(VALUES ? sh->v_raw[slot] : sh->k_scale[n & 3u]);
#pragma unroll
			for (int i = 0; i < 2; i++) {
				const int r = t + LOAD_THREADS * i;
				const long long row = __shfl_sync(0xffffffffu, first, r >> 4);
				const bool in = row >= 0 && key0 + r < p.key_end;
				cp_async4_or_zero(to + 4 * r, scales + (in ? row + (r & 15) : 0), in);
			}
		}
		ptx::cp_async_commit();
	}

	// The n-th tile has come in (this thread's part of it): makes it the operand and hands it over.
	__device__ __forceinline__ void finish(const Piece &p, int unit, uint32_t n)
	{
		const uint32_t slot = n & 1u;
		const uint32_t at = ring + slot * T::BYTES;
		constexpr int AT_ONCE = LOAD_THREADS / T::CHUNKS, PASSES = TILE / AT_ONCE;
		const int ch = t % T::CHUNKS, r0 = t / T::CHUNKS;
		const bool masked = (unit + 1) * TILE > p.all_see;
		float *scale = VALUES ? sh->v_raw[slot] : sh->k_scale[n & 3u];
		bool odd = false;
		if constexpr (KIND == TIE_CUDA_KV_Q8) {
#pragma unroll
			for (int i0 = 0; i0 < PASSES; i0 += 4) {
				uint4 v[4];
#pragma unroll
				for (int i = 0; i < 4; i++)
					v[i] = lds128(at + T::raw(r0 + (i0 + i) * AT_ONCE, ch));
				__syncwarp();  // a row's bytes are all in registers before its values overwrite them
#pragma unroll
				for (int i = 0; i < 4; i++) {
					const int r = r0 + (i0 + i) * AT_ONCE;
					const uint32_t b[4] = {v[i].x ^ 0x80808080u, v[i].y ^ 0x80808080u, v[i].z ^ 0x80808080u, v[i].w ^ 0x80808080u};
					sts128(at + T::place(r, 2 * ch), make_uint4(int8_pair<0x4140>(b[0]), int8_pair<0x4342>(b[0]), int8_pair<0x4140>(b[1]), int8_pair<0x4342>(b[1])));
					sts128(at + T::place(r, 2 * ch + 1), make_uint4(int8_pair<0x4140>(b[2]), int8_pair<0x4342>(b[2]), int8_pair<0x4140>(b[3]), int8_pair<0x4342>(b[3])));
				}
			}
		} else {
			constexpr uint32_t EXPONENT = KIND == TIE_CUDA_KV_F16 ? 0x7c00u : 0x7f80u;
			if (KIND == TIE_CUDA_KV_BF16 || (VALUES && masked)) {
#pragma unroll 4
				for (int i = 0; i < PASSES; i++) {
					const int r = r0 + i * AT_ONCE;
					const uint4 v = lds128(at + T::raw(r, ch));
					uint32_t w[4] = {v.x, v.y, v.z, v.w};
					bool change = KIND == TIE_CUDA_KV_BF16;
					if (VALUES && masked) {
#pragma unroll
						for (int j = 0; j < 4; j++)
							if (nonfinite16(w[j], EXPONENT)) {  // (its products are made by the rows that see it)
								w[j] &= ((w[j] & EXPONENT) == EXPONENT ? 0u : 0xffffu) | ((w[j] >> 16 & EXPONENT) == EXPONENT ? 0u : 0xffff0000u);
								odd = change = true;
							}
					}
					if constexpr (KIND == TIE_CUDA_KV_BF16) {
						uint32_t top = 0;  // largest magnitudes of even and odd values, infinities and NaN left out
#pragma unroll
						for (int j = 0; j < 4; j++) {
							uint32_t m = w[j] & 0x7fff7fffu;
							if (nonfinite16(w[j], EXPONENT))
								m &= ((m & EXPONENT) == EXPONENT ? 0u : 0xffffu) | ((m >> 16 & EXPONENT) == EXPONENT ? 0u : 0xffff0000u);
							top = __vmaxu2(top, m);
						}
#pragma unroll
						for (int o = T::CHUNKS / 2; o; o >>= 1)
							top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
						// the largest to 2^14 .. 2^15: 8 bits are exact down to 2^-32 of it
						const int e = max((int)(max(top & 0xffffu, top >> 16) >> 7), 15);
						const float f = __uint_as_float((uint32_t)(127 + 141 - e) << 23);
						if (ch == 0)
							scale[r] = __uint_as_float((uint32_t)(127 - 141 + e) << 23);
#pragma unroll
						for (int j = 0; j < 4; j++) {
							const __half2 h = __floats2half2_rn(__uint_as_float(w[j] << 16) * f, __uint_as_float(w[j] & 0xffff0000u) * f);
							w[j] = *reinterpret_cast<const uint32_t *>(&h);
						}
					}
					if (change)
						sts128(at + T::place(r, ch), make_uint4(w[0], w[1], w[2], w[3]));
				}
			}
		}
		if constexpr (T::SCALED) {
			// keys: the factors as they are; values: relative to the tile's largest, which multiplies the tile's sums
			if (VALUES) {
				if (KIND == TIE_CUDA_KV_BF16)
					bar_sync<3, LOAD_THREADS>();
				float f[2] = {scale[t], scale[t + LOAD_THREADS]};
#pragma unroll
				for (int i = 0; i < 2; i++)  // (an infinite factor is as little a number as NaN, and NaN does not reach the largest)
					f[i] = fabsf(f[i]) <= FLT_MAX ? f[i] : __int_as_float(0x7fc00000);
				float top = fmaxf(fmaxf(fabsf(f[0]), fabsf(f[1])), 0.0f);
#pragma unroll
				for (int o = 16; o; o >>= 1)
					top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
				if (lane == 0)
					sh->load_max[slot][t >> 5] = top;
				bar_sync<3, LOAD_THREADS>();
				top = fmaxf(sh->load_max[slot][0], sh->load_max[slot][1]);
				top = top > 0.0f ? top : 1.0f;
				if (t == 0)
					sh->v_top[slot] = top;
				sh->v_scale[slot][t] = f[0] / top;
				sh->v_scale[slot][t + LOAD_THREADS] = f[1] / top;
			}
		}
		if (VALUES) {
			odd = __any_sync(0xffffffffu, odd);
			if (lane == 0)
				sh->odd[slot][t >> 5] = odd;
		} else {
			ptx::mbar_arrive(ptx::smem_u32(&sh->f_full[n & 3u]));
		}
		ptx::fence_proxy_async_smem();
		ptx::mbar_arrive(ptx::smem_u32(VALUES ? &sh->v_full[slot] : &sh->k_full[slot]));
	}

	__device__ __forceinline__ void run(Walk w, const AttnWork &work, const AttnArgs &a, const Waiter &wait)
	{
		uint64_t *free_bar = VALUES ? sh->v_free : sh->k_free;
		Walk wp = w;
		Piece p, q;  // of the tile to be finished next, and of the one to be requested next
		int pi = 0, qi = 0;
		uint32_t asked = 0, done = 0;
		bool more = advance_to_tile(w, q, work, a);
		advance_to_tile(wp, p, work, a);
		while (done < asked || more) {
			// the next request goes out as soon as its slot is free; until then what has come in is made ready
			bool can = more && asked - done < 2;
			if (can && asked >= 2) {
				if (done < asked)
					can = __all_sync(0xffffffffu, ptx::mbar_try_wait(ptx::smem_u32(&free_bar[asked & 1]), ((asked >> 1) & 1u) ^ 1u));
				else
					wait(free_bar[asked & 1], ((asked >> 1) & 1u) ^ 1u);
			}
			if (can) {
				__syncwarp();
				issue(q, q.unit0 + qi, asked);
				asked++;
				if (++qi == q.n_tiles) {
					qi = 0;
					more = advance_to_tile(w, q, work, a);
				}
				if (asked - done < 2 && more)
					continue;
			}
			if (asked - done == 2)
				ptx::cp_async_wait<1>();
			else
				ptx::cp_async_wait<0>();
			finish(p, p.unit0 + pi, done);
			done++;
			if (++pi == p.n_tiles) {
				pi = 0;
				advance_to_tile(wp, p, work, a);
			}
		}
	}
	__device__ __forceinline__ bool advance_to_tile(Walk &w, Piece &p, const AttnWork &work, const AttnArgs &a)
	{
		do {
			if (!next_piece(w, p, work, kv, st, a))
				return false;
		} while (p.n_tiles == 0);
		return true;
	}
};

template <int KIND, int D>
__global__ void __launch_bounds__(THREADS, 1) attn_tiles(const KvView kv, const StepView st, const AttnArgs a)
{
	using T = Tile<KIND, D>;
	constexpr int HALF = D / 2;
	extern __shared__ uint8_t smem_raw[];
	__shared__ Shared shared;
	__shared__ AttnWork work;
	Shared *sh = &shared;
	const uint32_t smem = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
	const uint32_t k_ring = smem, v_ring = smem + 2 * T::BYTES, hand = smem + 4 * T::BYTES;
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
	if (threadIdx.x == 0) {
		for (int i = 0; i < 2; i++) {
			ptx::mbar_init(ptx::smem_u32(&sh->k_full[i]), LOAD_THREADS);
			ptx::mbar_init(ptx::smem_u32(&sh->k_free[i]), 1);
			ptx::mbar_init(ptx::smem_u32(&sh->v_full[i]), LOAD_THREADS);
			ptx::mbar_init(ptx::smem_u32(&sh->v_free[i]), 1);
			ptx::mbar_init(ptx::smem_u32(&sh->s_full[i]), 1);
			ptx::mbar_init(ptx::smem_u32(&sh->p_full[i]), SOFT_THREADS / 2);
			ptx::mbar_init(ptx::smem_u32(&sh->o_full[i]), 1);
		}
		for (int i = 0; i < 4; i++)
			ptx::mbar_init(ptx::smem_u32(&sh->f_full[i]), LOAD_THREADS);
		ptx::mbar_init(ptx::smem_u32(&sh->o_free), SOFT_THREADS / 2);
		ptx::mbar_init(ptx::smem_u32(&sh->q_full), SOFT_THREADS);
		ptx::mbar_init(ptx::smem_u32(&sh->fin), 1);
		sh->abort = 0;
		ptx::fence_barrier_init();
		ptx::fence_proxy_async_smem();
	}
	if (warp == W_MMA) {
		ptx::tmem_alloc(ptx::smem_u32(&sh->tmem_base), 512);
		ptx::tmem_relinquish();
	}
	// whole items where each CTA has several, else their units shared out evenly
	Walk walk = {};
	attn_share_work<THREADS>(work, kv, st, [&](const SeqView &q) { return attn_items(kv, a, q, ROWS); });
	walk.total = work.start[st.n_seq];
	walk.n_cta = gridDim.x;
	walk.shared = walk.total < 3ll * gridDim.x;
	if (walk.shared) {
		__syncthreads();
		attn_share_work<THREADS>(work, kv, st, [&](const SeqView &q) { return attn_items(kv, a, q, ROWS) * attn_units(q); });
		walk.total = work.start[st.n_seq];
		walk.n_cta = (int)min((long long)gridDim.x, walk.total);
		if ((int)blockIdx.x < walk.n_cta) {
			walk.u = walk.total * blockIdx.x / walk.n_cta;
			walk.u_end = walk.total * (blockIdx.x + 1) / walk.n_cta;
		}
	}
	ptx::tc_fence_before();
	__syncthreads();
	ptx::tc_fence_after();
	const uint32_t tmem = sh->tmem_base;
	const Waiter wait = {&sh->abort, st.status};

	if (warp < W_KEYS) {
		// ================= softmax: a thread per row and warpgroup =================
		ptx::setmaxnreg_inc<SOFT_REGS>();
		const int wg = threadIdx.x >> 7, r = threadIdx.x & 127;
		const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);  // this warp's 32 lanes
		uint32_t tiles = 0;
		Piece p;
		while (next_piece(walk, p, work, kv, st, a)) {
			const int n_rows = p.seq.n_tok * a.group, row = p.row0 + r;
			const bool there = row < n_rows;
			const int tok = there ? row / a.group : p.seq.n_tok - 1;
			const int head = p.head * a.group + (there ? row - tok * a.group : 0);
			const long long q_row = ((long long)(p.seq.tok0 + tok) * a.n_head + head) * D;
			float row_scale = 0.0f;
			if (p.n_tiles > 0) {  // this thread's half of the row, hi and lo, into tensor memory
				float4 v[HALF / 4];
				float top = 0.0f;
#pragma unroll
				for (int i = 0; i < HALF / 4; i++) {
					v[i] = there ? *reinterpret_cast<const float4 *>(a.q + q_row + wg * HALF + 4 * i) : make_float4(0, 0, 0, 0);
					top = fmaxf(fmaxf(fmaxf(top, fabsf(v[i].x)), fmaxf(fabsf(v[i].y), fabsf(v[i].z))), fabsf(v[i].w));
				}
				sh->q_max[wg][r] = top;
				bar_sync<1, SOFT_THREADS>();
				top = fmaxf(sh->q_max[0][r], sh->q_max[1][r]);
				// the row is brought to 1 .. 2 by a power of two (any fp32 row then keeps its 22 bits); it also takes the scale's sign
				const int e = top > 0.0f ? min(max((int)(__float_as_uint(top) >> 23), 1), 253) : 127;
				const float down = copysignf(__uint_as_float((uint32_t)(254 - e) << 23), a.scale_log2e);
				row_scale = fabsf(a.scale_log2e) * __uint_as_float((uint32_t)e << 23);
#pragma unroll
				for (int c = 0; c < HALF / 32; c++) {
					uint32_t hi[16], lo[16];
#pragma unroll
					for (int i = 0; i < 8; i++) {
						const float4 x = v[8 * c + i];
						split2(x.x * down, x.y * down, hi[2 * i], lo[2 * i]);
						split2(x.z * down, x.w * down, hi[2 * i + 1], lo[2 * i + 1]);
					}
					ptx::tmem_st16(lanes + COL_Q + wg * (HALF / 2) + 16 * c, hi);
					ptx::tmem_st16(lanes + COL_Q + HALF + wg * (HALF / 2) + 16 * c, lo);
				}
				ptx::tmem_st_wait();
				ptx::tc_fence_before();
				ptx::mbar_arrive(ptx::smem_u32(&sh->q_full));
			}
			unsigned long long bits = 0;  // tree: the step's tokens that this row sees
			if (st.tree) {
				bits = st.tree[p.seq.tok0 + tok];
				if (p.seq.n_tok < 64)
					bits &= (1ull << p.seq.n_tok) - 1;
				else if (p.seq.n_tok > KV_MAX_TREE && r == 0)
					kv_report(st, ST_BAD_STEP);
			}
			const int sees_to = p.seq.kv_len + tok + 1;  // no tree
			float acc[D], m = -INFINITY, l = 0.0f;
#pragma unroll
			for (int i = 0; i < D; i++)
				acc[i] = 0.0f;
			for (int i = 0; i < p.n_tiles; i++, tiles++) {
				if ((int)(tiles & 1) != wg)
					continue;
				const int key0 = (p.unit0 + i) * TILE, slot = wg;  // (tile n has operand slot and warpgroup n & 1)
				const uint32_t ph = (tiles >> 1) & 1u, S = lanes + COL_S + wg * TILE;
				const uint32_t fslot = tiles & 3u;
				wait(sh->f_full[fslot], (tiles >> 2) & 1u);
				wait(sh->s_full[wg], ph);
				ptx::tc_fence_after();
				// the keys of each 32 that this row sees
				uint32_t vis[4] = {~0u, ~0u, ~0u, ~0u};
				const uint32_t bad = sh->bad[fslot];
				const bool masked = key0 + TILE > p.all_see || bad != 0;
				if (masked) {
#pragma unroll
					for (int c = 0; c < 4; c++) {
						if (st.tree) {
							const int j = key0 + 32 * c - p.seq.kv_len;
							if (j >= 0)
								vis[c] = j < 64 ? (uint32_t)(bits >> j) : 0u;
							else if (j > -32)
								vis[c] = ((1u << -j) - 1u) | (uint32_t)bits << -j;
						} else {
							const int n = sees_to - (key0 + 32 * c);
							vis[c] = n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u;
						}
						if (bad >> (2 * c) & 1)
							vis[c] &= 0xffff0000u;
						if (bad >> (2 * c + 1) & 1)
							vis[c] &= 0x0000ffffu;
					}
				}
				// scores of 32 keys, times their rows' factors; -infinity where the row does not see
				auto scores = [&](int c, float (&x)[32]) {
					uint32_t v[32];
					ptx::tmem_ld32(S + 32 * c, v);
					ptx::tmem_ld_wait();
#pragma unroll
					for (int k = 0; k < 32; k += 4) {
						float4 f = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
						if constexpr (T::SCALED)
							f = *reinterpret_cast<const float4 *>(&sh->k_scale[fslot][32 * c + k]);
						x[k] = __uint_as_float(v[k]) * f.x;
						x[k + 1] = __uint_as_float(v[k + 1]) * f.y;
						x[k + 2] = __uint_as_float(v[k + 2]) * f.z;
						x[k + 3] = __uint_as_float(v[k + 3]) * f.w;
					}
					if (masked) {
#pragma unroll
						for (int k = 0; k < 32; k++)
							x[k] = vis[c] >> k & 1 ? x[k] : -INFINITY;
					}
				};
				float top = -INFINITY;
#pragma unroll
				for (int c = 0; c < 4; c++) {
					float x[32];
					scores(c, x);
#pragma unroll
					for (int k = 0; k < 32; k++)
						top = fmaxf(top, x[k]);
				}
				top = fmaxf(m, top * row_scale);
				const float base = (top == -INFINITY ? 0.0f : top) - ATTN_P_SHIFT;
				const float alpha = m == -INFINITY ? 0.0f : exp2f(m - top);
				m = top;
				// the values' factors, and whether all of them are numbers; read before P is handed over: when its products are
				// made the slot is another tile's
				bool odd = false;
				float v_top = 1.0f;
				if (T::SCALED || masked) {
					wait(sh->v_full[slot], ph);
					odd = sh->odd[slot][0] | sh->odd[slot][1];
					if constexpr (T::SCALED)
						v_top = sh->v_top[slot];
				}
				float sum = 0.0f;
#pragma unroll
				for (int c = 0; c < 4; c++) {
					float x[32];
					scores(c, x);
					// the parts of 16 keys take the columns of their scores: hi 8, lo 8
					uint32_t out[2][16];
#pragma unroll
					for (int k = 0; k < 32; k += 2) {
						float p0 = exp2f(fmaf(x[k], row_scale, -base)), p1 = exp2f(fmaf(x[k + 1], row_scale, -base));
						sum += p0 + p1;
						if constexpr (T::SCALED) {
							const float2 f = *reinterpret_cast<const float2 *>(&sh->v_scale[slot][32 * c + k]);
							p0 = p0 == 0.0f ? 0.0f : p0 * f.x;
							p1 = p1 == 0.0f ? 0.0f : p1 * f.y;
						}
						split2(p0, p1, out[k >> 4][(k >> 1) & 7], out[k >> 4][8 + ((k >> 1) & 7)]);
					}
					ptx::tmem_st16(S + 32 * c, out[0]);
					ptx::tmem_st16(S + 32 * c + 16, out[1]);
				}
				ptx::tmem_st_wait();
				ptx::tc_fence_before();
				ptx::mbar_arrive(ptx::smem_u32(&sh->p_full[wg]));
				l = fmaf(l, alpha, sum);
				wait(sh->o_full[wg], ph);
				ptx::tc_fence_after();
#pragma unroll
				for (int c = 0; c < D / 32; c++) {
					uint32_t v[32];
					ptx::tmem_ld32(lanes + COL_O + 32 * c, v);
					ptx::tmem_ld_wait();
#pragma unroll
					for (int k = 0; k < 32; k++) {
						if constexpr (T::SCALED)
							acc[32 * c + k] = fmaf(__uint_as_float(v[k]), v_top, acc[32 * c + k] * alpha);
						else
							acc[32 * c + k] = fmaf(acc[32 * c + k], alpha, __uint_as_float(v[k]));
					}
				}
				ptx::tc_fence_before();
				ptx::mbar_arrive(ptx::smem_u32(&sh->o_free));
				if (KIND != TIE_CUDA_KV_Q8 && odd) {  // infinities and NaN among values that not every row sees: p > 0 times them is what they are
#pragma unroll 1
					for (int k = 0; k < TILE; k++) {
						if (key0 + k >= p.key_end)
							break;
						const uint32_t w = k < 32 ? vis[0] : k < 64 ? vis[1] : k < 96 ? vis[2] : vis[3];
						if (!(w >> (k & 31) & 1))
							continue;
						const int page = st.page_table[(long long)p.s * st.max_pages + ((key0 + k) >> kv.page_shift)];
						const long long at = (((long long)page * kv.n_head_kv + p.head) << kv.page_shift) + ((key0 + k) & ((1 << kv.page_shift) - 1));
						const uint32_t *src = reinterpret_cast<const uint32_t *>(kv.v + at * T::ROW);
						constexpr uint32_t EXPONENT = KIND == TIE_CUDA_KV_F16 ? 0x7c00u : 0x7f80u;
#pragma unroll
						for (int d = 0; d < D / 2; d++) {
							const uint32_t x = src[d];
							if (nonfinite16(x, EXPONENT)) {
								const float2 f = KIND == TIE_CUDA_KV_F16 ? __half22float2(*reinterpret_cast<const __half2 *>(&x))
													 : make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
								acc[2 * d] += (x & EXPONENT) == EXPONENT ? f.x : 0.0f;
								acc[2 * d + 1] += (x >> 16 & EXPONENT) == EXPONENT ? f.y : 0.0f;
							}
						}
					}
				}
			}

			// the two warpgroups' keys together: each finishes half of the dims
			sh->ml[wg][r] = make_float2(m, l);
			const uint32_t give = hand + (uint32_t)(wg ^ 1) * (ROWS * HALF * 4) + r * 16, take = hand + (uint32_t)wg * (ROWS * HALF * 4) + r * 16;
#pragma unroll
			for (int j = 0; j < HALF / 4; j++) {
				uint4 x;
				x.x = __float_as_uint(wg ? acc[4 * j] : acc[HALF + 4 * j]);
				x.y = __float_as_uint(wg ? acc[4 * j + 1] : acc[HALF + 4 * j + 1]);
				x.z = __float_as_uint(wg ? acc[4 * j + 2] : acc[HALF + 4 * j + 2]);
				x.w = __float_as_uint(wg ? acc[4 * j + 3] : acc[HALF + 4 * j + 3]);
				sts128(give + j * (ROWS * 16), x);
			}
			bar_sync<1, SOFT_THREADS>();
			const float2 other = sh->ml[wg ^ 1][r];
			const float top = fmaxf(m, other.x);
			const float f_own = m == -INFINITY ? 0.0f : exp2f(m - top), f_other = other.x == -INFINITY ? 0.0f : exp2f(other.x - top);
			const float sum = l * f_own + other.y * f_other;
			const bool whole = p.unit0 == 0 && p.unit1 == p.item_units;
			const float inv = !whole ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
			float *part = a.part + (2 * blockIdx.x + (p.unit0 == 0 ? 1 : 0)) * attn_part_floats(ROWS);
			float *dst = whole ? a.out + q_row + wg * HALF : part + r * D + wg * HALF;
			if (!whole || there) {
#pragma unroll
				for (int j = 0; j < HALF / 4; j++) {
					const uint4 x = lds128(take + j * (ROWS * 16));
					const uint32_t xo[4] = {x.x, x.y, x.z, x.w};
					float y[4];
#pragma unroll
					for (int k = 0; k < 4; k++) {
						const float mine = wg ? acc[HALF + 4 * j + k] : acc[4 * j + k];
						// (a warpgroup whose keys the row does not see has nothing to give)
						y[k] = ((f_own == 0.0f ? 0.0f : mine * f_own) + (f_other == 0.0f ? 0.0f : __uint_as_float(xo[k]) * f_other)) * inv;
					}
					*reinterpret_cast<float4 *>(dst + 4 * j) = make_float4(y[0], y[1], y[2], y[3]);
				}
			}
			if (!whole) {
				if (wg == 0) {
					part[ROWS * 128 + r] = top;
					part[ROWS * 128 + ROWS + r] = sum;
				}
				const long long i0 = walk.u - p.unit1, i1 = i0 + p.item_units - 1;  // (walk.u: behind this piece)
				const int c0 = attn_cta_of(i0, walk.total, walk.n_cta), c1 = attn_cta_of(i1, walk.total, walk.n_cta);
				__threadfence();
				bar_sync<1, SOFT_THREADS>();
				if (threadIdx.x == 0)
					work.last = atomicAdd(a.count + c0, 1u) == (unsigned)(c1 - c0);
				bar_sync<1, SOFT_THREADS>();
				if (work.last) {
					__threadfence();
					for (int i = warp; i < ROWS && p.row0 + i < n_rows; i += SOFT_THREADS / 32) {
						const int t = (p.row0 + i) / a.group;
						attn_join_row<D, ROWS>(a.part, c0, c1, i, lane,
								       a.out + ((long long)(p.seq.tok0 + t) * a.n_head + p.head * a.group + (p.row0 + i - t * a.group)) * D);
					}
					if (threadIdx.x == 0)
						a.count[c0] = 0;  // at rest again
				}
			}
		}
	} else if (warp < W_MMA) {
		ptx::setmaxnreg_dec<LOAD_REGS>();
		if (warp < W_VALUES) {
			Loader<KIND, D, false> loader = {kv, st, sh, k_ring, (int)threadIdx.x - W_KEYS * 32, lane};
			loader.run(walk, work, a, wait);
		} else {
			Loader<KIND, D, true> loader = {kv, st, sh, v_ring, (int)threadIdx.x - W_VALUES * 32, lane};
			loader.run(walk, work, a, wait);
		}
	} else {
		ptx::setmaxnreg_dec<MMA_REGS>();
		if (warp == W_MMA) {
			if (ptx::elect_one()) {
				constexpr uint32_t idesc_qk = ptx::umma_idesc_f16(ROWS, TILE);
				constexpr uint32_t idesc_pv = ptx::umma_idesc_f16(ROWS, D) | 1u << 16;	// V: dims contiguous
				uint32_t tiles = 0, pieces = 0;
				// P V of tile n
				auto products = [&](uint32_t n) {
					const uint32_t slot = n & 1u, ph = (n >> 1) & 1u;
					wait(sh->v_full[slot], ph);
					wait(sh->p_full[slot], ph);
					const bool ok = n == 0 || wait(sh->o_free, (n - 1) & 1u);
					ptx::tc_fence_after();
					if (ok && !*wait.abort) {
						// MN-major: 8 keys 1024 bytes apart, 64 dims a panel apart
						const uint32_t b = ptx::umma_desc_lo(v_ring + slot * T::BYTES) | (PANEL >> 4) << 16, P = tmem + COL_S + slot * TILE;
#pragma unroll
						for (int part = 1; part >= 0; part--)
#pragma unroll
							for (int k = 0; k < TILE / 16; k++)
								ptx::mma_f16_ts(tmem + COL_O, P + 16 * k + 8 * part, b + k * (2048 >> 4), idesc_pv, part == 0 || k > 0);
					}
					ptx::mma_commit(ptx::smem_u32(&sh->v_free[slot]));
					ptx::mma_commit(ptx::smem_u32(&sh->o_full[slot]));
				};
				Piece p;
				while (next_piece(walk, p, work, kv, st, a)) {
					if (p.n_tiles == 0)
						continue;
					wait(sh->q_full, pieces & 1u);
					for (int i = 0; i < p.n_tiles; i++, tiles++) {
						const uint32_t slot = tiles & 1u, ph = (tiles >> 1) & 1u;
						wait(sh->k_full[slot], ph);
						ptx::tc_fence_after();
						if (!*wait.abort) {
							const uint32_t b = ptx::umma_desc_lo(k_ring + slot * T::BYTES);
#pragma unroll
							for (int part = 1; part >= 0; part--)
#pragma unroll
								for (int k = 0; k < D / 16; k++)
									ptx::mma_f16_ts(tmem + COL_S + slot * TILE, tmem + COL_Q + part * HALF + 8 * k,
											b + (k >> 2) * (PANEL >> 4) + 2 * (k & 3), idesc_qk, part == 0 || k > 0);
						}
						ptx::mma_commit(ptx::smem_u32(&sh->k_free[slot]));
						ptx::mma_commit(ptx::smem_u32(&sh->s_full[slot]));
						if (i > 0)
							products(tiles - 1);
					}
					products(tiles - 1);
					pieces++;
				}
				ptx::mma_commit(ptx::smem_u32(&sh->fin));
			}
			__syncwarp();
			wait(sh->fin, 0);
		}
	}
	ptx::tc_fence_before();
	__syncthreads();
	if (warp == W_MMA) {
		ptx::tc_fence_after();
		ptx::tmem_dealloc(tmem, 512);
	}
}

template <int KIND, int D>
constexpr size_t smem_bytes()
{
	return 4 * (size_t)Tile<KIND, D>::BYTES + (size_t)ROWS * D * 4 + 1024;
}
template <int KIND, int D>
int go(tie_cuda_ctx *c, const KvView &kv, const StepView &st, const AttnArgs &a)
{
	attn_tiles<KIND, D><<<c->sm_count, THREADS, smem_bytes<KIND, D>(), c->stream>>>(kv, st, a);
	TIE_CUDA_LAUNCHED(c);
	return TIE_CUDA_OK;
}
template <int KIND>
int allow_smem(tie_cuda_ctx *c)
{
	TIE_CUDA_TRY(c, cudaFuncSetAttribute(attn_tiles<KIND, 128>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes<KIND, 128>()));
	TIE_CUDA_TRY(c, cudaFuncSetAttribute(attn_tiles<KIND, 64>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes<KIND, 64>()));
	return TIE_CUDA_OK;
}

}  // namespace

int attn_tc_setup(tie_cuda_ctx *c)
{
	int rc = allow_smem<TIE_CUDA_KV_F16>(c);
	rc = rc ? rc : allow_smem<TIE_CUDA_KV_BF16>(c);
	return rc ? rc : allow_smem<TIE_CUDA_KV_Q8>(c);
}

int launch_attn_tc(tie_cuda_ctx *c, const KvView &kv, const StepView &st, int kind, int head_dim, const AttnArgs &a)
{
#define TIE_GO(KIND) (head_dim == 128 ? go<KIND, 128>(c, kv, st, a) : go<KIND, 64>(c, kv, st, a))
	return kind == TIE_CUDA_KV_F16 ? TIE_GO(TIE_CUDA_KV_F16) : kind == TIE_CUDA_KV_BF16 ? TIE_GO(TIE_CUDA_KV_BF16) : TIE_GO(TIE_CUDA_KV_Q8);
#undef TIE_GO
}

}  // namespace tie
