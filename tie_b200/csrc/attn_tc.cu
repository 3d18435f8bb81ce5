// Attention over the paged cache for sequences with many query rows per key/value head (trees of drafted tokens, prompt
// pieces): tiles of 128 rows x 128 or 64 keys on tcgen05.
//
//   S = Q K^T, P = exp2(S - max), O = P V      rows (token, head of the group) on the 128 lanes of tensor memory
//
// fp32 results need more than one 16-bit operand per value.  F16 and Q8: Q and P are fp16 hi + lo (22 bits) against keys and
// values that are exact in fp16, the factors of Q8's rows applied in fp32; BF16: three bf16 parts (24 bits), tiles of 64
// keys, since tensor memory holds no more.  The products of a tile start from zero and are added to fp32 registers: the
// tensor cores cut every sum off, which over a long cache would add up.
//
// One CTA per SM, 640 threads:
//   * two warpgroups of softmax threads, a thread per row and half of a tile's keys; a third adds the tiles' products up, a
//     thread per row, with the row in registers (where the softmax threads did that too, they waited for half of the time
//     for products);
//   * a warp requests keys, another values, by TMA straight into the swizzled operand layout, a box per page (as one
//     cp.async per 16 bytes the address arithmetic alone took 5000 cycles a tile from two warps);
//   * two warps each make operands of what came in where it is not one yet: Q8's bytes become fp16 in place, values behind
//     the last key and values that are no numbers become zeros;
//   * one thread finds the CTA's pieces of work, one issues the MMAs (one for the scores and one for the products: 49.0 us
//     of the piece below became 53.1).  Q and P are operands in tensor memory (a step of shared memory then feeds only the keys or dims of the
//     other operand: half of what the memory delivers); P's parts of 16 keys take the columns of these keys' scores.
// What it takes (a piece of 512 tokens over 1500 keys, F16, 32 heads of 128 with 4 of keys: 47.3 us, 312 TFLOP/s, 620 of MMAs):
// a tile of 128 keys takes about 3400 cycles where its MMAs take 2050 and its exponentials 1024: the scores of a tile wait
// for the products of the last but one, and the issuing thread's four waits a tile cost 150 to 400 cycles each, complete or
// not; 16000 cycles pass before the first scores and 5000 behind the last products.
// Every wait is bounded, as in tensor.cu; after a time-out no wait waits any more and all roles run to their ends.
#include <float.h>

#include "attn.cuh"
#include "decode_common.cuh"
#include "kernels.cuh"
#include "tc_ptx.cuh"

namespace tie {
namespace {

constexpr int ROWS = ATTN_MAX_ROWS;
constexpr int THREADS = 640, SOFT_THREADS = 256, FOLD_THREADS = 128, MAKE_THREADS = 64;
constexpr int W_FOLD = 8, W_KEYS = 12, W_VALUES = 14, W_MMA = 16, W_PIECES = 17, W_ASK = 18;	// first warps of the roles behind the softmax warps
constexpr int SOFT_REGS = 104, FOLD_REGS = 176, MAKE_REGS = 56, REST_REGS = 40;
static_assert(2 * SOFT_REGS + FOLD_REGS + MAKE_REGS + REST_REGS <= 5 * 96, "a launch of 640 threads holds 96 registers a thread");
constexpr long long WAIT_CYCLES = 1ll << 30;
constexpr int OUT_BYTES = ROWS * 16 * 4;  // 16 dims of a tile's rows, on their way out

// A piece of work of a CTA: an item, or (few items: shared) some units of one.  No more of them: s < 0.
struct Piece {
	SeqView seq;
	int s, head, row0;
	int unit0, unit1;
	bool whole, first;  // the item, its first part
	int n_parts;	// first: parts of the item
	int n_tiles;	// from unit0 on: tiles that some row of the item sees keys of
	int key_end;	// first key that nobody sees
	int all_see;	// keys in front of this one are seen by every row
};
constexpr int PIECES = 4, MAX_STAGES = 4, MAX_SLOTS = 3, MAX_FACTS = 7, TILE_FACTS = 5;
struct Shared {
	uint64_t piece_full[PIECES], piece_free[PIECES];
	Piece piece[PIECES];	// made by a warp of its own: they cost several divisions each
	uint64_t k_raw[MAX_STAGES], k_full[MAX_STAGES], k_free[MAX_STAGES];  // keys have come in; are the operand; have been used
	uint64_t v_raw[MAX_STAGES], v_full[MAX_STAGES], v_free[MAX_STAGES];
	uint64_t s_full[MAX_SLOTS], p_full[MAX_SLOTS], o_full, o_free, q_come, q_full, l_full[PIECES], fin;
	// What the softmax threads need to know of a tile's keys outlives its operand slot, which is free once the scores are
	// made: tile n + FACTS is requested after the scores of tile n + SLOTS at the least, these after the products of n.
	uint64_t f_full[MAX_FACTS];
	uint32_t bad[MAX_FACTS], bad_values[MAX_STAGES];  // groups of 16 keys of a tile whose page does not exist
	alignas(16) float k_scale[640];	 // [FACTS][TK]
	alignas(16) float v_got[256], v_scale[256];  // [STAGES][TK]: factors as they came, and as shares of the tile's unit
	float v_unit[MAX_STAGES], make_max[MAX_STAGES][2];
	uint32_t odd[MAX_STAGES][2];  // a masked tile's values hold one that is no number (per warp)
	// of a row, per warpgroup: the largest query of a piece; in tiles of Q8 whose factors lie far apart, the largest share that the row
	// sees (by then q_full has come in from all who read the other)
	float row_max[2][ROWS];
	float half_top[2][2][ROWS];	 // per tile in turn and warpgroup: the largest score of a row
	// what the products of a tile have to be added up with: maximum of a row, unit (below 0: each row's own, by its exponent);
	// whether values are no numbers, bad pages
	float t_top[TILE_FACTS][ROWS], t_unit[TILE_FACTS];
	uint32_t t_odd[TILE_FACTS], t_bad[TILE_FACTS];
	// per piece in turn and warpgroup: sum of a row's p, relative to its maximum in the end.  (Of PIECES, since a piece without
	// tiles makes nobody wait for the warpgroup that takes them.)
	float l[PIECES][2][ROWS];
	uint32_t tmem_base, abort;
	uint8_t t_row_unit[TILE_FACTS][ROWS];
};

// How a launch's work is shared out.  WHOLE: items, several to a CTA.  EVEN: each CTA the same number of units, whatever items
// they belong to (a CTA then mostly has the end of one and the beginning of another).  PARTS: no more items than CTAs,
// each cut into as many equal parts as leave one part to a CTA.
enum Share : int { WHOLE, EVEN, PARTS };
// Where Q8's factors lie far apart in a tile that not every row sees in full (ATTN_WIDE), a row's p are raised by as much as the largest
// factor that it sees is below the tile's, so that their products with the shares fill the 16-bit parts again.  Shares are held
// times 2^WIDE_UP there and p are raised by that much less, or p of 1 would pass fp32's range for shares of 2^-114.
constexpr int WIDE_UP = 100;
// What a piece costs besides its tiles (set-up, first loads, joins), in units.
constexpr int PIECE_UNITS = 8;
struct Walk {
	Share share;
	long long total, u, u_end;
	int n_cta, round;
	int part_units;	 // PARTS: units of a part, at most
};

template <int TK>
__device__ __forceinline__ bool next_piece(Walk &w, Piece &p, const AttnWork &work, const KvView &kv, const StepView &st, const AttnArgs &a)
{
	long long i = w.u;  // unit, item or part
	if (w.share == WHOLE) {
		// a sequence's last rows (the ones that see most) first, there and back over the CTAs
		do {
			if ((long long)w.round * w.n_cta >= w.total)
				return false;
			i = (w.round & 1) ? (long long)(w.round + 1) * w.n_cta - 1 - blockIdx.x : (long long)w.round * w.n_cta + blockIdx.x;
			w.round++;
		} while (i >= w.total);
	} else if (w.u >= w.u_end) {
		return false;
	}
	p.s = attn_sequence_of(work, st.n_seq, i);
	p.seq = kv_sequence(st, kv.page_shift, p.s);
	const int tiles = (int)(((long long)p.seq.n_tok * a.group + ROWS - 1) / ROWS), units = attn_units(p.seq);
	const long long in_seq = i - work.start[p.s];
	const int parts = w.share == PARTS ? (units + w.part_units - 1) / w.part_units : 1;
	const long long item = attn_div(in_seq, w.share == EVEN ? units : parts);
	const int rest = (int)(in_seq - item * (w.share == EVEN ? units : parts));
	if (w.share == WHOLE) {
		const int back = (int)attn_div(item, kv.n_head_kv);
		p.row0 = (tiles - 1 - back) * ROWS;
		p.head = (int)(item - (long long)back * kv.n_head_kv);
	} else {
		p.head = (int)attn_div(item, tiles);
		p.row0 = (int)(item - (long long)p.head * tiles) * ROWS;
	}
	const int first_tok = p.row0 / a.group, last_tok = min((p.row0 + ROWS - 1) / a.group, p.seq.n_tok - 1);
	p.key_end = p.seq.kv_len + (st.tree ? p.seq.n_tok : last_tok + 1);
	p.all_see = p.seq.kv_len + (st.tree ? 0 : first_tok + 1);
	const int used = (p.key_end + ATTN_UNIT - 1) / ATTN_UNIT;  // units that some row sees keys of
	p.n_parts = 1;
	if (w.share == EVEN) {
		p.unit0 = rest;
		p.unit1 = (int)min((long long)units, rest + (w.u_end - w.u));
		p.whole = p.unit0 == 0 && p.unit1 == units;
		if (p.unit0 == 0 && !p.whole)  // the item goes on in the next CTAs
			p.n_parts = attn_cta_of(i + units - 1, w.total, w.n_cta) - (int)blockIdx.x + 1;
		w.u += p.unit1 - p.unit0;
	} else {
		p.unit0 = (int)attn_div((long long)used * rest, parts);
		p.unit1 = (int)attn_div((long long)used * (rest + 1), parts);
		p.whole = parts == 1;
		if (rest == 0)
			p.n_parts = parts;
		w.u++;
	}
	p.first = w.share == EVEN ? p.unit0 == 0 : rest == 0;
	p.n_tiles = max(0, (min(p.unit1 * ATTN_UNIT, p.key_end) - p.unit0 * ATTN_UNIT + TK - 1) / TK);
	return true;
}

template <int N>
__device__ __forceinline__ Walk start_walk(AttnWork &work, const KvView &kv, const StepView &st, const AttnArgs &a, int n_cta, int cta)
{
	Walk w = {};
	w.n_cta = n_cta;
	// Sums over the sequences, made by each warp for itself: a scan by all of them with its barriers for every size of part that
	// is tried took 13000 cycles with 8 sequences.
	auto total = [&](auto of) {
		if (st.n_seq == 1)
			return (long long)of(kv_sequence(st, kv.page_shift, 0));
		long long sum = 0;
		for (int s = threadIdx.x & 31; s < st.n_seq; s += 32)
			sum += of(kv_sequence(st, kv.page_shift, s));
#pragma unroll
		for (int o = 16; o; o >>= 1)
			sum += __shfl_xor_sync(0xffffffffu, sum, o);
		return sum;
	};
	auto items_of = [&](const SeqView &q) { return attn_items(kv, a, q, ROWS); };
	auto units_of = [&](const SeqView &q) { return attn_items(kv, a, q, ROWS) * attn_units(q); };
	const long long items = total(items_of);
	if (items == 0 || items >= 3ll * n_cta) {
		attn_share_work<N>(work, kv, st, items_of);
		w.share = WHOLE;
		w.total = items;
		return w;
	}
	const long long units = total(units_of);
	if (items <= n_cta) {
		// The smallest part size with which there are no more parts than CTAs; with several sequences tried in steps of an
		// eighth, and not kept where it costs more than a second piece in each CTA would.
		const int even = (int)min(attn_div(units + n_cta - 1, n_cta), 1ll << 30);
		auto parts_of = [&](const SeqView &q) { return attn_items(kv, a, q, ROWS) * ((attn_units(q) + w.part_units - 1) / w.part_units); };
		if (st.n_seq == 1) {
			const int each = (int)((unsigned)n_cta / (unsigned)items), of_item = attn_units(kv_sequence(st, kv.page_shift, 0));
			w.part_units = (of_item + each - 1) / each;
			w.total = total(parts_of);
		} else {
			for (w.part_units = even; w.part_units <= even + PIECE_UNITS; w.part_units += max(1, w.part_units >> 3)) {
				w.total = total(parts_of);
				if (w.total <= n_cta)
					break;
			}
		}
		if (w.total <= n_cta) {
			attn_share_work<N>(work, kv, st, parts_of);
			w.share = PARTS;
			w.u = cta;
			w.u_end = cta < w.total ? cta + 1 : cta;
			return w;
		}
	}
	attn_share_work<N>(work, kv, st, units_of);
	w.share = EVEN;
	w.total = units;
	w.n_cta = (int)min((long long)n_cta, units);
	if (cta < w.n_cta) {
		w.u = attn_div(w.total * cta, w.n_cta);
		w.u_end = attn_div(w.total * (cta + 1), w.n_cta);
	}
	return w;
}

template <int KIND, int D>
struct Tile {
	static constexpr bool SCALED = KIND == TIE_CUDA_KV_Q8;
	static constexpr int PARTS = KIND == TIE_CUDA_KV_BF16 ? 3 : 2;	 // of a value of Q and of P
	// Keys of a tile, and score tiles: as many as tensor memory holds beside Q and O.  Heads of 128, two parts: with two tiles of
	// 128 keys 8 trees of 64 tokens over 3500 keys (Q8) took 77.9 us and a piece of 512 over 1500 (F16) 53.4, with four of 64
	// keys 84.5 and 55.1, since each tile has its waits (71.6 and 47.3 now).  Three parts, heads of 64: a third tile of 64 keys
	// brought 4096 tokens from 290 to 266 us (257 now).
	static constexpr int TK = PARTS == 3 ? 64 : 128;
	static constexpr int SLOTS = D == 128 ? 2 : 3;
	static constexpr int STAGES = TK * D == 128 * 128 || (SCALED && D == 64) ? 2 : 4;
	static constexpr int FACTS = STAGES + SLOTS;
	static_assert(FACTS <= MAX_FACTS && (!SCALED || (FACTS * TK <= 640 && STAGES * TK <= 256)) && STAGES <= MAX_STAGES && SLOTS <= MAX_SLOTS && TILE_FACTS >= SLOTS + 2, "rings");
	// tensor memory: parts of Q, score tiles (and what P's parts need beyond their columns), O
	static constexpr int SLOT = PARTS == 3 ? TK + TK / 2 : TK, COL_Q = 0, COL_S = PARTS * D / 2, COL_O = COL_S + SLOTS * SLOT;
	static_assert(COL_O + D <= 512, "tensor memory");
	static constexpr uint32_t PANEL = TK * 128;  // 64 dims of a tile: rows of 128 bytes
	static constexpr uint32_t BYTES = TK * D * 2;
	static constexpr int ROW = SCALED ? D : 2 * D;	 // bytes of a head row of the cache
	static constexpr int BOX_BYTES = ROW < 128 ? ROW : 128, BOXES = ROW / BOX_BYTES;  // of a row, per TMA box
	static constexpr uint32_t RAW = SCALED && D == 64 ? TK * ROW : 0;  // rows of 64 bytes come in beside the operand
	static constexpr int Q_ROW = D * 4 + 16;  // bytes from row to row of the queries' tile in shared memory
	static constexpr size_t SMEM = 2 * (size_t)STAGES * (BYTES + RAW) + (size_t)ROWS * Q_ROW + OUT_BYTES + 1024;
	// where a 16-byte chunk of row r's 16-bit values lies in the operand tile
	__device__ static __forceinline__ uint32_t place(int r, int ch) { return (ch >> 3) * PANEL + r * 128 + (((ch & 7) ^ (r & 7)) << 4); }
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

// The same, and whether any thread brings a true one.
template <int ID, int N>
__device__ __forceinline__ bool bar_any(bool mine)
{
	uint32_t any;
	asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
		     : "=r"(any)
		     : "r"((uint32_t)mine), "n"(ID), "n"(N)
		     : "memory");
	return any != 0;
}

// Bounded; true once the barrier's phase is complete.
struct Waiter {
	volatile uint32_t *abort;
	unsigned *status;
	// always: also after another wait has given up (the pieces go on: whoever reads them does not wait for anything else then)
	__device__ __forceinline__ bool operator()(uint64_t &bar, uint32_t parity, bool always = false) const
	{
		const uint32_t b = ptx::smem_u32(&bar);
		if (ptx::mbar_try_wait(b, parity))
			return true;
		const long long t0 = clock64();
		while (!ptx::mbar_try_wait_suspend(b, parity, 20000u)) {
			if (!always && *abort)
				return false;
			if (clock64() - t0 > (always ? 4 * WAIT_CYCLES : WAIT_CYCLES)) {
				atomicOr(status, ST_WAIT_TIMEOUT);
				*abort = 1;
				return false;
			}
		}
		return true;
	}
};

// The n-th piece of work, for a warp (or the issuing thread): taken, and given back.
__device__ __forceinline__ Piece take_piece(Shared *sh, const Waiter &wait, uint32_t n)
{
	wait(sh->piece_full[n % PIECES], n / PIECES & 1u, true);
	return sh->piece[n % PIECES];
}
__device__ __forceinline__ void drop_piece(Shared *sh, uint32_t n, int lane)
{
	__syncwarp();
	if (lane == 0)
		ptx::mbar_arrive(ptx::smem_u32(&sh->piece_free[n % PIECES]));
}

// Two fp32 operations an instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
	float2 r;
	asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
	    : "=f"(r.x), "=f"(r.y)
	    : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
	return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
	float2 r;
	asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
	    : "=f"(r.x), "=f"(r.y)
	    : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
	return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
	float2 r;
	asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 w, {%6, %7};\n\tfma.rn.f32x2 z, x, y, w;\n\tmov.b64 {%0, %1}, z;\n\t}"
	    : "=f"(r.x), "=f"(r.y)
	    : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
	return r;
}
__device__ __forceinline__ float2 sub2(float2 a, float2 b)
{
	float2 r;
	asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tsub.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
	    : "=f"(r.x), "=f"(r.y)
	    : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
	return r;
}
// The 16-bit parts of a pair, the largest first: fp16 hi and lo, rounded (22 bits of 24), or three of bf16, cut off (8 bits
// each, and so all).
template <int KIND, int PARTS>
__device__ __forceinline__ void split2(float2 x, uint32_t (&part)[PARTS])
{
#pragma unroll
	for (int p = 0; p < PARTS; p++) {
		float2 f;
		if constexpr (KIND == TIE_CUDA_KV_BF16) {
			const uint32_t a = __float_as_uint(x.x), b = __float_as_uint(x.y);
			part[p] = __byte_perm(a, b, 0x7632);
			f = make_float2(__uint_as_float(a & 0xffff0000u), __uint_as_float(b & 0xffff0000u));
		} else {
			const __half2 h = __floats2half2_rn(x.x, x.y);
			part[p] = *reinterpret_cast<const uint32_t *>(&h);
			f = __half22float2(h);
		}
		if (p < PARTS - 1)
			x = sub2(x, f);
	}
}

// All ones over those of a pair that are numbers.
__device__ __forceinline__ uint32_t finite16(uint32_t w, uint32_t exponent)
{
	return ((w & exponent) == exponent ? 0u : 0xffffu) | ((w >> 16 & exponent) == exponent ? 0u : 0xffff0000u);
}

// Which keys a query row sees.
struct RowView {
	bool tree;
	int kv_len, sees_to;
	unsigned long long bits;  // tree: the step's tokens
	// of 32 keys from `key` on, without those of bad pages (a bit per 16)
	__device__ __forceinline__ uint32_t keys(int key, uint32_t bad) const
	{
		uint32_t vis = ~0u;
		if (tree) {
			const int j = key - kv_len;
			if (j >= 0)
				vis = j < 64 ? (uint32_t)(bits >> j) : 0u;
			else if (j > -32)
				vis = ((1u << -j) - 1u) | (uint32_t)bits << -j;
		} else {
			const int n = sees_to - key;
			vis = n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u;
		}
		return vis & ~((bad & 1 ? 0x0000ffffu : 0u) | (bad & 2 ? 0xffff0000u : 0u));
	}
};
__device__ __forceinline__ RowView row_view(const StepView &st, const Piece &p, int tok, bool report)
{
	RowView v = {st.tree != nullptr, p.seq.kv_len, p.seq.kv_len + tok + 1, 0};
	if (st.tree) {
		v.bits = st.tree[p.seq.tok0 + tok];
		if (p.seq.n_tok < 64)
			v.bits &= (1ull << p.seq.n_tok) - 1;
		else if (p.seq.n_tok > KV_MAX_TREE && report)
			kv_report(st, ST_BAD_STEP);
	}
	return v;
}

// Of a tile's keys from `first` on the largest share of a factor that a row sees, NaN where one is no number (out of line: the loops it is
// called from fill the instruction caches as they are).
__device__ __noinline__ float largest_share(const float *share, int first, int n, int key0, uint32_t bad, RowView view)
{
	float most = 0.0f;
#pragma unroll 1
	for (int k = first; k < first + n; k++)
		if (view.keys(key0 + k, bad >> (k >> 4) & 1u) & 1u)
			most = most == most && share[k] == share[k] ? fmaxf(most, fabsf(share[k])) : __int_as_float(0x7fc00000);
	return most;
}

// Requests the tiles of keys (VALUES false) or values: a warp, a lane per page of a tile.
template <int KIND, int D, bool VALUES>
__device__ __forceinline__ void ask(const KvView &kv, const StepView &st, Shared *sh, const CUtensorMap *map, uint32_t ring, uint32_t raw, const Waiter &wait,
				    int lane)
{
	using T = Tile<KIND, D>;
	const int run = min(1 << kv.page_shift, T::TK), n_runs = T::TK / run, page_mask = (1 << kv.page_shift) - 1;
	uint64_t *free_bar = VALUES ? sh->v_free : sh->k_free, *raw_bar = VALUES ? sh->v_raw : sh->k_raw;
	uint32_t n = 0;
	for (uint32_t pn = 0;; pn++) {
		const Piece p = take_piece(sh, wait, pn);
		drop_piece(sh, pn, lane);
		if (p.s < 0)
			break;
		const int *pages = st.page_table + (long long)p.s * st.max_pages;
		auto page_of = [&](int i) {  // of this lane's keys of the piece's tile i
			const int key = p.unit0 * ATTN_UNIT + i * T::TK + lane * run;
			return lane < n_runs && i < p.n_tiles && key < p.key_end ? pages[key >> kv.page_shift] : -1;
		};
		int next = page_of(0);
		for (int i = 0; i < p.n_tiles; i++, n++) {
			const int key0 = p.unit0 * ATTN_UNIT + i * T::TK, key = key0 + lane * run, page = next;
			const uint32_t slot = n % T::STAGES;
			next = page_of(i + 1);
			const bool wanted = lane < n_runs && key < p.key_end;
			long long row = wanted ? kv_page_row(kv, st, page, p.head) : -1;
			const bool in = row >= 0;
			const uint32_t got = __ballot_sync(0xffffffffu, in), lost = __ballot_sync(0xffffffffu, wanted && !in);
			row += key & page_mask;
			if (n >= T::STAGES)
				wait(free_bar[slot], (n / T::STAGES & 1u) ^ 1u);
			__syncwarp();
			if (lane == 0) {
				uint32_t bad = 0;
				if (lost)
					for (int g = 0; g < T::TK / 16; g++)
						bad |= (lost >> (g * 16 / run) & 1u) << g;
				(VALUES ? sh->bad_values[slot] : sh->bad[n % T::FACTS]) = bad;
				if (!VALUES && !T::SCALED)
					ptx::mbar_arrive(ptx::smem_u32(&sh->f_full[n % T::FACTS]));
				ptx::mbar_arrive_expect_tx(ptx::smem_u32(&raw_bar[slot]), __popc(got) * run * (T::ROW + (T::SCALED ? 4 : 0)));
			}
			__syncwarp();
			if (in) {
				const uint32_t bar = ptx::smem_u32(&raw_bar[slot]);
				const uint32_t dst = T::RAW ? raw + slot * T::RAW + lane * run * T::ROW
							    : ring + slot * T::BYTES + (T::SCALED ? T::PANEL : 0u) + lane * run * 128;
				if (run == T::TK || T::BOXES == 1) {
					ptx::tma_load_3d(dst, map, bar, 0, (int)row, 0);
				} else {
#pragma unroll
					for (int b = 0; b < T::BOXES; b++)  // (the halves of a page's rows lie a tile's panel apart)
						ptx::tma_load_3d(dst + b * T::PANEL, map, bar, 0, (int)row, b);
				}
				if constexpr (T::SCALED)
					bulk_g2s(ptx::smem_u32(VALUES ? sh->v_got + slot * T::TK : sh->k_scale + n % T::FACTS * T::TK) + 4 * lane * run, (VALUES ? kv.v_scale : kv.k_scale) + row,
						  run * 4, bar);
			}
		}
	}
	// (nothing that was requested is still on its way when the block ends, whoever has given up)
	for (uint32_t i = n < T::STAGES ? 0 : n - T::STAGES; i < n; i++)
		wait(raw_bar[i % T::STAGES], i / T::STAGES & 1u, true);
}

// Makes operands of what has come in: two warps for keys (Q8 only), two for values.
template <int KIND, int D, bool VALUES>
__device__ __forceinline__ void make(Shared *sh, uint32_t ring, uint32_t raw, const Waiter &wait, int t, int lane)
{
	using T = Tile<KIND, D>;
	uint32_t n = 0;
	for (uint32_t pn = 0;; pn++) {
		const Piece p = take_piece(sh, wait, pn);
		drop_piece(sh, pn, lane);
		if (p.s < 0)
			break;
		for (int i = 0; i < p.n_tiles; i++, n++) {
			const int key0 = p.unit0 * ATTN_UNIT + i * T::TK;
			const uint32_t slot = n % T::STAGES, at = ring + slot * T::BYTES;
			wait(VALUES ? sh->v_raw[slot] : sh->k_raw[slot], n / T::STAGES & 1u);
			const uint32_t bad = VALUES ? sh->bad_values[slot] : 0u;
			const bool masked = VALUES && (key0 + T::TK > p.all_see || bad != 0);
			bool odd = false;
			// the keys that are somebody's: the others' values are zeros, whatever has come in
			auto there = [&](int r) { return key0 + r < p.key_end && !(bad >> (r >> 4) & 1u); };
			if constexpr (T::SCALED) {
				constexpr int CHUNKS = T::ROW / 16, AT_ONCE = MAKE_THREADS / CHUNKS, PASSES = T::TK / AT_ONCE, B = 4;
				const int ch = t % CHUNKS, r0 = t / CHUNKS;
#pragma unroll 1
				for (int j0 = 0; j0 < PASSES; j0 += B) {
					uint4 v[B];
#pragma unroll
					for (int j = 0; j < B; j++) {
						const int r = r0 + (j0 + j) * AT_ONCE;
						v[j] = lds128(T::RAW ? raw + slot * T::RAW + r * T::ROW + ch * 16 : at + T::PANEL + r * 128 + ((ch ^ (r & 7)) << 4));
					}
					__syncwarp();  // a row's bytes are all in registers before its values overwrite them
#pragma unroll
					for (int j = 0; j < B; j++) {
						const int r = r0 + (j0 + j) * AT_ONCE;
						if (masked && !there(r))
							v[j] = make_uint4(0, 0, 0, 0);
						const uint32_t b[4] = {v[j].x ^ 0x80808080u, v[j].y ^ 0x80808080u, v[j].z ^ 0x80808080u, v[j].w ^ 0x80808080u};
						uint4 lo, hi;
						if constexpr (VALUES) {
							lo = make_uint4(int8_pair_low<0x4140>(b[0]), int8_pair_low<0x4342>(b[0]), int8_pair_low<0x4140>(b[1]), int8_pair_low<0x4342>(b[1]));
							hi = make_uint4(int8_pair_low<0x4140>(b[2]), int8_pair_low<0x4342>(b[2]), int8_pair_low<0x4140>(b[3]), int8_pair_low<0x4342>(b[3]));
						} else {
							lo = make_uint4(int8_pair<0x4140>(b[0]), int8_pair<0x4342>(b[0]), int8_pair<0x4140>(b[1]), int8_pair<0x4342>(b[1]));
							hi = make_uint4(int8_pair<0x4140>(b[2]), int8_pair<0x4342>(b[2]), int8_pair<0x4140>(b[3]), int8_pair<0x4342>(b[3]));
						}
						sts128(at + T::place(r, 2 * ch), lo);
						sts128(at + T::place(r, 2 * ch + 1), hi);
					}
				}
				if constexpr (VALUES) {	 // factors as shares of a unit, which multiplies the tile's sums
					constexpr int EACH = T::TK / MAKE_THREADS;
					float f[EACH];
					float top = 0.0f;
#pragma unroll
					for (int j = 0; j < EACH; j++) {
						f[j] = there(t + MAKE_THREADS * j) ? sh->v_got[slot * T::TK + t + MAKE_THREADS * j] : 0.0f;
						// (an infinite factor is as little a number as NaN, and NaN does not reach the largest)
						f[j] = fabsf(f[j]) <= FLT_MAX ? f[j] : __int_as_float(0x7fc00000);
						top = fmaxf(top, fabsf(f[j]));
					}
					top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));  // (as the number that its bits are)
					if (lane == 0)
						sh->make_max[slot][t >> 5] = top;
					bar_sync<2, MAKE_THREADS>();
					const float unit = attn_unit_of(fmaxf(sh->make_max[slot][0], sh->make_max[slot][1]));
					if (t == 0)
						sh->v_unit[slot] = unit;
#pragma unroll
					for (int j = 0; j < EACH; j++)
						sh->v_scale[slot * T::TK + t + MAKE_THREADS * j] = f[j] * attn_unit_inverse(unit);
				}
			} else if (masked) {
				constexpr uint32_t EXPONENT = KIND == TIE_CUDA_KV_F16 ? 0x7c00u : 0x7f80u;
				constexpr int CHUNKS = T::ROW / 16, AT_ONCE = MAKE_THREADS / CHUNKS, PASSES = T::TK / AT_ONCE;
				const int ch = t % CHUNKS, r0 = t / CHUNKS;
#pragma unroll 4
				for (int j = 0; j < PASSES; j++) {
					const int r = r0 + j * AT_ONCE;
					const uint32_t to = at + T::place(r, ch);
					const uint4 v = lds128(to);
					uint32_t w[4] = {v.x, v.y, v.z, v.w};
					bool change = false;
					if (!there(r)) {
						w[0] = w[1] = w[2] = w[3] = 0;
						change = true;
					} else {
#pragma unroll
						for (int k = 0; k < 4; k++)
							if (nonfinite16(w[k], EXPONENT)) {  // (its products are made by the rows that see it)
								w[k] &= finite16(w[k], EXPONENT);
								odd = change = true;
							}
					}
					if (change)
						sts128(to, make_uint4(w[0], w[1], w[2], w[3]));
				}
			}
			if (VALUES) {
				odd = __any_sync(0xffffffffu, odd);
				if (lane == 0)
					sh->odd[slot][t >> 5] = odd;
			} else {
				ptx::mbar_arrive(ptx::smem_u32(&sh->f_full[n % T::FACTS]));
			}
			ptx::fence_proxy_async_smem();
			ptx::mbar_arrive(ptx::smem_u32(VALUES ? &sh->v_full[slot] : &sh->k_full[slot]));
		}
	}
}

template <int KIND, int D>
__global__ void __launch_bounds__(THREADS, 1) attn_tiles(const KvView kv, const StepView st, const AttnArgs a, const __grid_constant__ CUtensorMap k_map,
						     const __grid_constant__ CUtensorMap v_map)
{
	using T = Tile<KIND, D>;
	constexpr int HALF = D / 2, D4 = D / 4, Q_ROW = T::Q_ROW;
	extern __shared__ uint8_t smem_raw[];
	__shared__ Shared shared;
	__shared__ AttnWork work;
	static_assert(T::SMEM + sizeof(Shared) + sizeof(AttnWork) <= 227 * 1024, "shared memory of a CTA");
	Shared *sh = &shared;
	const uint32_t smem = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
	constexpr int TK = T::TK;
	const uint32_t k_ring = smem, v_ring = k_ring + T::STAGES * T::BYTES, k_raw = v_ring + T::STAGES * T::BYTES, v_raw = k_raw + T::STAGES * T::RAW;
	const uint32_t hand = v_raw + T::STAGES * T::RAW, out_stage = hand + ROWS * Q_ROW;
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
	if (threadIdx.x == 0) {
		for (int i = 0; i < T::STAGES; i++) {
			ptx::mbar_init(ptx::smem_u32(&sh->k_raw[i]), 1);
			ptx::mbar_init(ptx::smem_u32(&sh->k_full[i]), MAKE_THREADS);
			ptx::mbar_init(ptx::smem_u32(&sh->k_free[i]), 1);
			ptx::mbar_init(ptx::smem_u32(&sh->v_raw[i]), 1);
			ptx::mbar_init(ptx::smem_u32(&sh->v_full[i]), MAKE_THREADS);
			ptx::mbar_init(ptx::smem_u32(&sh->v_free[i]), 1);
		}
		for (int i = 0; i < T::SLOTS; i++) {
			ptx::mbar_init(ptx::smem_u32(&sh->s_full[i]), 1);
			ptx::mbar_init(ptx::smem_u32(&sh->p_full[i]), SOFT_THREADS);
		}
		for (int i = 0; i < T::FACTS; i++)
			ptx::mbar_init(ptx::smem_u32(&sh->f_full[i]), T::SCALED ? MAKE_THREADS : 1);
		for (int i = 0; i < PIECES; i++) {
			ptx::mbar_init(ptx::smem_u32(&sh->piece_full[i]), 1);
			ptx::mbar_init(ptx::smem_u32(&sh->l_full[i]), SOFT_THREADS);
			ptx::mbar_init(ptx::smem_u32(&sh->piece_free[i]), SOFT_THREADS / 32 + FOLD_THREADS / 32 + 1 + 2 + (T::SCALED ? 4 : 2));  // softmax, fold, MMA, ask, make
		}
		ptx::mbar_init(ptx::smem_u32(&sh->o_full), 1);
		ptx::mbar_init(ptx::smem_u32(&sh->o_free), FOLD_THREADS);
		ptx::mbar_init(ptx::smem_u32(&sh->q_come), ROWS);
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
	const Walk walk = start_walk<THREADS>(work, kv, st, a, gridDim.x, blockIdx.x);
	ptx::tc_fence_before();
	__syncthreads();
	ptx::tc_fence_after();
	const uint32_t tmem = sh->tmem_base;
	const Waiter wait = {&sh->abort, st.status};

	if (warp < W_FOLD) {
		// ================= softmax: a thread per row and warpgroup =================
		ptx::setmaxnreg_inc<SOFT_REGS>();
		const int wg = threadIdx.x >> 7, r = threadIdx.x & 127;
		const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);  // this warp's 32 lanes
		uint32_t tiles = 0, loads = 0;
		Piece p;
		for (uint32_t n = 0;; n++) {
			p = take_piece(sh, wait, n);
			drop_piece(sh, n, lane);
			if (p.s < 0)
				break;
			const int n_rows = p.seq.n_tok * a.group, row = p.row0 + r;
			const bool there = row < n_rows;
			const int tok = there ? row / a.group : p.seq.n_tok - 1;
			// 4 dims of a row of the tile, in shared memory: rows a bank group apart, no conflicts
			auto spot = [&](int d4, int line) { return hand + (uint32_t)line * Q_ROW + d4 * 16; };
			float row_scale = 0.0f;
			bar_sync<1, SOFT_THREADS>();  // nobody reads rows or makes scores of the piece before any more
			if (p.n_tiles > 0) {
				// The rows as they lie, through shared memory (a thread's own row from global memory: 32 lines a load), a copy each (by
				// cp.async, 16 a thread, the addresses alone took 5000 cycles), and this thread's half of its row, in parts, into
				// tensor memory.
				if (lane < ROWS / 8) {
					const int line = warp * (ROWS / 8) + lane, q_row = p.row0 + line, t = q_row / a.group;
					const uint32_t bar = ptx::smem_u32(&sh->q_come);
					if (q_row < n_rows) {
						ptx::mbar_arrive_expect_tx(bar, D * 4);
						bulk_g2s(spot(0, line), a.q + ((long long)(p.seq.tok0 + t) * a.n_head + p.head * a.group + (q_row - t * a.group)) * D, D * 4, bar);
					} else {
						ptx::mbar_arrive(bar);
					}
				}
				wait(sh->q_come, loads++ & 1u, true);
				float top = 0.0f;
#pragma unroll 4
				for (int i = 0; i < HALF / 4; i++) {
					const uint4 x = there ? lds128(spot(wg * (HALF / 4) + i, r)) : make_uint4(0, 0, 0, 0);
					top = fmaxf(fmaxf(fmaxf(top, fabsf(__uint_as_float(x.x))), fmaxf(fabsf(__uint_as_float(x.y)), fabsf(__uint_as_float(x.z)))),
						    fabsf(__uint_as_float(x.w)));
				}
				sh->row_max[wg][r] = top;
				bar_sync<1, SOFT_THREADS>();
				top = fmaxf(sh->row_max[0][r], sh->row_max[1][r]);
				// the row is brought to 1 .. 2 by a power of two (any fp32 row then keeps its 22 bits); it also takes the scale's sign
				const int e = top > 0.0f ? min(max((int)(__float_as_uint(top) >> 23), 1), 253) : 127;
				float down = copysignf(__uint_as_float((uint32_t)(254 - e) << 23), a.scale_log2e);
				row_scale = fabsf(a.scale_log2e) * __uint_as_float((uint32_t)e << 23);
				if (row_scale == 0.0f) {  // the queries are zeros then, so that the -infinity of a key that is not seen stays one
					down = 0.0f;
					row_scale = 1.0f;
				}
#pragma unroll 1
				for (int c = 0; c < HALF / 16; c++) {
					uint32_t out[T::PARTS][8];
#pragma unroll
					for (int i = 0; i < 4; i++) {
						const uint4 x = there ? lds128(spot(wg * (HALF / 4) + 4 * c + i, r)) : make_uint4(0, 0, 0, 0);
						uint32_t part[2][T::PARTS];
						split2<KIND>(make_float2(__uint_as_float(x.x) * down, __uint_as_float(x.y) * down), part[0]);
						split2<KIND>(make_float2(__uint_as_float(x.z) * down, __uint_as_float(x.w) * down), part[1]);
#pragma unroll
						for (int k = 0; k < T::PARTS; k++) {
							out[k][2 * i] = part[0][k];
							out[k][2 * i + 1] = part[1][k];
						}
					}
#pragma unroll
					for (int k = 0; k < T::PARTS; k++)
						ptx::tmem_st8(lanes + T::COL_Q + k * HALF + wg * (HALF / 2) + 8 * c, out[k]);
				}
				ptx::tmem_st_wait();
				ptx::tc_fence_before();
				ptx::mbar_arrive(ptx::smem_u32(&sh->q_full));
			}
			const RowView view = row_view(st, p, tok, r == 0);
			float m = -INFINITY, l = 0.0f;
			for (int i = 0; i < p.n_tiles; i++, tiles++) {
				const int key0 = p.unit0 * ATTN_UNIT + i * TK;
				const uint32_t slot = tiles % T::STAGES, score = tiles % T::SLOTS, S = lanes + T::COL_S + score * T::SLOT;
				const uint32_t fslot = tiles % T::FACTS;
				wait(sh->f_full[fslot], tiles / T::FACTS & 1u);
				wait(sh->s_full[score], tiles / T::SLOTS & 1u);
				ptx::tc_fence_after();
				const uint32_t bad = sh->bad[fslot];
				const bool masked = key0 + TK > p.all_see || bad != 0;
				// scores of 32 keys, times their rows' factors; -infinity where the row does not see
				auto scores = [&](int c, float2 (&x)[16], bool scaled) {
					uint32_t v[32];
					ptx::tmem_ld32(S + 32 * c, v);
					ptx::tmem_ld_wait();
#pragma unroll
					for (int k = 0; k < 16; k++)
						x[k] = make_float2(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1]));
					if (T::SCALED && !scaled) {
#pragma unroll
						for (int k = 0; k < 16; k += 2) {
							const float4 f = *reinterpret_cast<const float4 *>(&sh->k_scale[fslot * TK + 32 * c + 2 * k]);
							x[k] = mul2(x[k], make_float2(f.x, f.y));
							x[k + 1] = mul2(x[k + 1], make_float2(f.z, f.w));
						}
					}
					if (masked && !(T::SCALED && scaled)) {
						const uint32_t vis = view.keys(key0 + 32 * c, bad >> (2 * c));
#pragma unroll
						for (int k = 0; k < 16; k++) {
							x[k].x = vis >> (2 * k) & 1 ? x[k].x : -INFINITY;
							x[k].y = vis >> (2 * k + 1) & 1 ? x[k].y : -INFINITY;
						}
					}
				};
				float top = -INFINITY;
				float2 x[16];  // where a warpgroup has no more than these of a tile, they are read once
				constexpr int CHUNKS = TK / 64;
#pragma unroll 1
				for (int c = wg * CHUNKS; c < wg * CHUNKS + CHUNKS; c++) {
					scores(c, x, false);
#pragma unroll
					for (int k = 0; k < 16; k++)
						top = fmaxf(top, fmaxf(x[k].x, x[k].y));
					if constexpr (T::SCALED && CHUNKS > 1) {
						// back with the factors in them: each read of those by all lanes costs the shared memory 512 cycles a tile
#pragma unroll
						for (int h = 0; h < 2; h++) {
							uint32_t v[16];
#pragma unroll
							for (int k = 0; k < 8; k++) {
								v[2 * k] = __float_as_uint(x[8 * h + k].x);
								v[2 * k + 1] = __float_as_uint(x[8 * h + k].y);
							}
							ptx::tmem_st16(S + 32 * c + 16 * h, v);
						}
					}
				}
				if constexpr (T::SCALED && CHUNKS > 1)
					ptx::tmem_st_wait();
				sh->half_top[i & 1][wg][r] = top;
				bar_sync<1, SOFT_THREADS>();
				top = fmaxf(m, fmaxf(top, sh->half_top[i & 1][wg ^ 1][r]) * row_scale);
				float base = ATTN_P_SHIFT<KIND> - (top == -INFINITY ? 0.0f : top);
				const float alpha = m == -INFINITY ? 0.0f : exp2_ftz(m - top);
				m = top;
				// the values' factors, and whether all of them are numbers; read before P is handed over: when its products are
				// made the slot is another tile's
				if (T::SCALED || masked)
					wait(sh->v_full[slot], tiles / T::STAGES & 1u);
				bool special = false, wide = false;
				int up = 0;  // p are larger by 2^up
				float lost = 0.0f;
				if (T::SCALED && masked) {
					const float share = fabsf(sh->v_scale[slot * TK + r]);
					const bool far = share * ATTN_WIDE < 1.0f && share != 0.0f;
					special = bar_any<1, SOFT_THREADS>(far || share != share);
					if (special)
						wide = bar_any<1, SOFT_THREADS>(far);
				}
				if (special) {
					// (in the products below 0 times what is no number is 0, for the rows that do not see it)
					const float most = largest_share(&sh->v_scale[slot * TK], wg * CHUNKS * 32, CHUNKS * 32, key0, bad, view);
					lost = most == most ? 0.0f : most;
					sh->row_max[wg][r] = most;
				}
				if (wide) {
					bar_sync<1, SOFT_THREADS>();
					if (wg == 0)
						sh->v_scale[slot * TK + r] *= __uint_as_float((127u + WIDE_UP) << 23);
					bar_sync<1, SOFT_THREADS>();
					const int e = __float_as_uint(sh->v_unit[slot]) >> 23;
					const int share = (int)(__float_as_uint(attn_unit_of(fmaxf(sh->row_max[0][r], sh->row_max[1][r]))) >> 23) - 127 + WIDE_UP;
					up = min(max(-share, -WIDE_UP), e - WIDE_UP - 1);
					base += (float)up;
					if (wg == 0)
						sh->t_row_unit[tiles % TILE_FACTS][r] = (uint8_t)(e - up - WIDE_UP);
				}
				if (wg == 0)
					sh->t_top[tiles % TILE_FACTS][r] = top;
				if (threadIdx.x == 0) {
					sh->t_odd[tiles % TILE_FACTS] = masked ? sh->odd[slot][0] | sh->odd[slot][1] : 0u;
					sh->t_bad[tiles % TILE_FACTS] = bad;
					sh->t_unit[tiles % TILE_FACTS] = !T::SCALED ? 1.0f : wide ? -1.0f : sh->v_unit[slot] * ATTN_Q8_DOWN;
				}
				float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll 1
				for (int c = wg * CHUNKS; c < wg * CHUNKS + CHUNKS; c++) {
					if constexpr (CHUNKS > 1)
						scores(c, x, true);
					// the first two parts of 16 keys take the columns of their scores, 8 each; a third comes behind all of them
#pragma unroll
					for (int h = 0; h < 2; h++) {
						uint32_t out[16], third[8];
						float4 vs;
#pragma unroll
						for (int k = 0; k < 8; k++) {
							const float2 e = fma2(x[8 * h + k], make_float2(row_scale, row_scale), make_float2(base, base));
							float2 pk = make_float2(exp2_ftz(e.x), exp2_ftz(e.y));
							sum = add2(sum, pk);
							if constexpr (T::SCALED) {
								if ((k & 1) == 0)
									vs = *reinterpret_cast<const float4 *>(&sh->v_scale[slot * TK + 32 * c + 16 * h + 2 * k]);
								const float2 z = mul2(pk, k & 1 ? make_float2(vs.z, vs.w) : make_float2(vs.x, vs.y));
								// (where a row does not see every key, a factor that is no number is nothing to it)
								pk = masked ? make_float2(pk.x == 0.0f ? 0.0f : z.x, pk.y == 0.0f ? 0.0f : z.y) : z;
							}
							uint32_t part[T::PARTS];
							split2<KIND>(pk, part);
							out[k] = part[0];
							out[8 + k] = part[1];
							if constexpr (T::PARTS == 3)
								third[k] = part[2];
						}
						ptx::tmem_st16(S + 32 * c + 16 * h, out);
						if constexpr (T::PARTS == 3)
							ptx::tmem_st8(S + TK + 16 * c + 8 * h, third);
					}
				}
				ptx::tmem_st_wait();
				ptx::tc_fence_before();
				ptx::mbar_arrive(ptx::smem_u32(&sh->p_full[score]));
				l = fmaf(l, alpha, T::SCALED ? (sum.x + sum.y) * __uint_as_float((uint32_t)(127 - up) << 23) + lost : sum.x + sum.y);
			}
			sh->l[n % PIECES][wg][r] = l;
			ptx::mbar_arrive(ptx::smem_u32(&sh->l_full[n % PIECES]));
		}
	} else if (warp < W_KEYS) {
		// ================= fold: a thread per row adds the tiles' products up =================
		ptx::setmaxnreg_inc<FOLD_REGS>();
		const int r = threadIdx.x & 127;
		const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
		uint32_t tiles = 0;
		for (uint32_t n = 0;; n++) {
			const Piece p = take_piece(sh, wait, n);
			drop_piece(sh, n, lane);
			if (p.s < 0)
				break;
			const int n_rows = p.seq.n_tok * a.group, row = p.row0 + r;
			const RowView view = row_view(st, p, row < n_rows ? row / a.group : p.seq.n_tok - 1, false);
			float2 acc[HALF];
			float top = -INFINITY;
#pragma unroll
			for (int i = 0; i < HALF; i++)
				acc[i] = make_float2(0.0f, 0.0f);
			for (int i = 0; i < p.n_tiles; i++, tiles++) {
				const uint32_t at = tiles % TILE_FACTS;
				wait(sh->o_full, tiles & 1u);
				ptx::tc_fence_after();
				// relative to the largest maximum so far (the tiles' are those of the two warpgroups)
				const float t_top = sh->t_top[at][r], next = fmaxf(top, t_top);
				float unit = sh->t_unit[at];
				if (T::SCALED && unit < 0.0f)
					unit = __uint_as_float((uint32_t)sh->t_row_unit[at][r] << 23) * ATTN_Q8_DOWN;
				const float f = t_top == -INFINITY ? 0.0f : exp2_ftz(t_top - next) * unit, g = top == -INFINITY ? 0.0f : exp2_ftz(top - next);
				const bool odd = KIND != TIE_CUDA_KV_Q8 && sh->t_odd[at];
				const uint32_t bad = sh->t_bad[at];
				top = next;
				const float2 f2 = make_float2(f, f), g2 = make_float2(g, g);
#pragma unroll
				for (int c = 0; c < D / 32; c++) {
					uint32_t v[32];
					ptx::tmem_ld32(lanes + T::COL_O + 32 * c, v);
					ptx::tmem_ld_wait();
#pragma unroll
					for (int k = 0; k < 16; k++)
						acc[16 * c + k] = fma2(make_float2(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1])), f2, mul2(acc[16 * c + k], g2));
				}
				ptx::tc_fence_before();
				if (i == p.n_tiles - 1)	 // (what the piece is finished with is read before the piece after the next can be)
					wait(sh->l_full[n % PIECES], n / PIECES & 1u);
				if (odd) {  // infinities and NaN among values that not every row sees: p > 0 times them is what they are
					const int key0 = p.unit0 * ATTN_UNIT + i * TK;
#pragma unroll 1
					for (int k = 0; k < TK && key0 + k < p.key_end; k++) {
						if (!(view.keys(key0 + (k & ~31), bad >> (k >> 4 & ~1)) >> (k & 31) & 1))
							continue;
						const int page = st.page_table[(long long)p.s * st.max_pages + ((key0 + k) >> kv.page_shift)];
						const long long src_row = (((long long)page * kv.n_head_kv + p.head) << kv.page_shift) + ((key0 + k) & ((1 << kv.page_shift) - 1));
						const uint32_t *src = reinterpret_cast<const uint32_t *>(kv.v + src_row * T::ROW);
						constexpr uint32_t EXPONENT = KIND == TIE_CUDA_KV_F16 ? 0x7c00u : 0x7f80u;
#pragma unroll
						for (int d = 0; d < HALF; d++) {
							const uint32_t x = src[d];
							if (nonfinite16(x, EXPONENT)) {
								const float2 y = KIND == TIE_CUDA_KV_F16 ? __half22float2(*reinterpret_cast<const __half2 *>(&x))
													 : make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
								acc[d].x += (x & EXPONENT) == EXPONENT ? y.x : 0.0f;
								acc[d].y += (x >> 16 & EXPONENT) == EXPONENT ? y.y : 0.0f;
							}
						}
					}
				}
				if (i < p.n_tiles - 1)
					ptx::mbar_arrive(ptx::smem_u32(&sh->o_free));
			}
			if (p.n_tiles == 0)
				wait(sh->l_full[n % PIECES], n / PIECES & 1u);
			const float sum = sh->l[n % PIECES][0][r] + sh->l[n % PIECES][1][r];  // (relative to the largest maximum, as the products)
			if (p.n_tiles > 0)
				ptx::mbar_arrive(ptx::smem_u32(&sh->o_free));
			if (!p.whole) {
				float *part = a.part + (2 * blockIdx.x + (p.first ? 1 : 0)) * attn_part_floats(ROWS);
				part[ROWS * 128 + r] = top;
				part[ROWS * 128 + ROWS + r] = sum;
#pragma unroll
				for (int j = 0; j < D4; j++)  // [4 dims][row]
					reinterpret_cast<float4 *>(part)[j * ROWS + r] = make_float4(acc[2 * j].x, acc[2 * j].y, acc[2 * j + 1].x, acc[2 * j + 1].y);
				continue;
			}
			// whole rows go out by 16 dims through shared memory, each warp its 32: 4 lanes then store 64 bytes of a row
			const float inv = sum == 0.0f ? 0.0f : (T::SCALED ? ATTN_Q8_UP : 1.0f) / sum;
			long long at[4];
#pragma unroll
			for (int i = 0; i < 4; i++) {
				const int line = p.row0 + (warp & 3) * 32 + i * 8 + lane / 4, t = line / a.group;
				at[i] = line < n_rows ? ((long long)(p.seq.tok0 + t) * a.n_head + p.head * a.group + (line - t * a.group)) * D + lane % 4 * 4 : -1;
			}
			const float2 i2 = make_float2(inv, inv);
#pragma unroll
			for (int c = 0; c < D / 16; c++) {
				__syncwarp();
#pragma unroll
				for (int j = 0; j < 4; j++) {
					const float2 y0 = mul2(acc[8 * c + 2 * j], i2), y1 = mul2(acc[8 * c + 2 * j + 1], i2);
					sts128(out_stage + (j * ROWS + (r ^ j)) * 16, make_uint4(__float_as_uint(y0.x), __float_as_uint(y0.y), __float_as_uint(y1.x), __float_as_uint(y1.y)));
				}
				__syncwarp();
#pragma unroll
				for (int i = 0; i < 4; i++) {
					const int line = (warp & 3) * 32 + i * 8 + lane / 4, j = lane % 4;
					const uint4 y = lds128(out_stage + (j * ROWS + (line ^ j)) * 16);
					if (at[i] >= 0)
						*reinterpret_cast<uint4 *>(a.out + at[i] + 16 * c) = y;
				}
			}
		}
	} else if (warp < W_MMA) {
		ptx::setmaxnreg_dec<MAKE_REGS>();
		if (warp >= W_VALUES)
			make<KIND, D, true>(sh, v_ring, v_raw, wait, (int)threadIdx.x - W_VALUES * 32, lane);
		else if (T::SCALED)
			make<KIND, D, false>(sh, k_ring, k_raw, wait, (int)threadIdx.x - W_KEYS * 32, lane);
	} else {
		ptx::setmaxnreg_dec<REST_REGS>();
		if (warp == W_MMA) {
			if (ptx::elect_one()) {
				constexpr uint32_t types = KIND == TIE_CUDA_KV_BF16 ? 1u << 7 | 1u << 10 : 0u;
				constexpr uint32_t idesc_qk = ptx::umma_idesc_f16(ROWS, TK) | types;
				constexpr uint32_t idesc_pv = ptx::umma_idesc_f16(ROWS, D) | types | 1u << 16;	// V: dims contiguous
				uint32_t tiles = 0, pieces = 0;
				auto products = [&](uint32_t n) {  // P V of tile n
					const uint32_t slot = n % T::STAGES;
					wait(sh->v_full[slot], n / T::STAGES & 1u);
					wait(sh->p_full[n % T::SLOTS], n / T::SLOTS & 1u);
					const bool ok = n == 0 || wait(sh->o_free, (n - 1) & 1u);
					ptx::tc_fence_after();
					if (ok && !*wait.abort) {
						// MN-major: 8 keys 1024 bytes apart, 64 dims a panel apart
						const uint32_t b = ptx::umma_desc_lo(v_ring + slot * T::BYTES) | (T::PANEL >> 4) << 16, P = tmem + T::COL_S + n % T::SLOTS * T::SLOT;
#pragma unroll
						for (int part = T::PARTS - 1; part >= 0; part--)
#pragma unroll
							for (int k = 0; k < TK / 16; k++)
								ptx::mma_f16_ts(tmem + T::COL_O, P + (part < 2 ? 16 * k + 8 * part : TK + 8 * k), b + k * (2048 >> 4), idesc_pv,
										part < T::PARTS - 1 || k > 0);
					}
					ptx::mma_commit(ptx::smem_u32(&sh->v_free[slot]));
					ptx::mma_commit(ptx::smem_u32(&sh->o_full));
				};
				Piece p;
				for (uint32_t n = 0;; n++) {
					p = take_piece(sh, wait, n);
					ptx::mbar_arrive(ptx::smem_u32(&sh->piece_free[n % PIECES]));
					if (p.s < 0)
						break;
					if (p.n_tiles == 0)
						continue;
					wait(sh->q_full, pieces & 1u);
					// scores as far ahead of the products as there are tiles for them
					for (int i = 0; i < p.n_tiles + T::SLOTS - 1; i++) {
						if (i < p.n_tiles) {
							const uint32_t n = tiles + i, slot = n % T::STAGES;
							wait(T::SCALED ? sh->k_full[slot] : sh->k_raw[slot], n / T::STAGES & 1u);
							ptx::tc_fence_after();
							if (!*wait.abort) {
								const uint32_t b = ptx::umma_desc_lo(k_ring + slot * T::BYTES);
#pragma unroll
								for (int part = T::PARTS - 1; part >= 0; part--)
#pragma unroll
									for (int k = 0; k < D / 16; k++)
										ptx::mma_f16_ts(tmem + T::COL_S + n % T::SLOTS * T::SLOT, tmem + T::COL_Q + part * HALF + 8 * k,
												b + (k >> 2) * (T::PANEL >> 4) + 2 * (k & 3), idesc_qk, part < T::PARTS - 1 || k > 0);
							}
							ptx::mma_commit(ptx::smem_u32(&sh->k_free[slot]));
							ptx::mma_commit(ptx::smem_u32(&sh->s_full[n % T::SLOTS]));
						}
						if (i >= T::SLOTS - 1)
							products(tiles + i - (T::SLOTS - 1));
					}
					tiles += p.n_tiles;
					pieces++;
				}
				ptx::mma_commit(ptx::smem_u32(&sh->fin));
			}
			__syncwarp();
			wait(sh->fin, 0, true);
		} else if (warp >= W_ASK) {
			if (warp == W_ASK)
				ask<KIND, D, false>(kv, st, sh, &k_map, k_ring, k_raw, wait, lane);
			else
				ask<KIND, D, true>(kv, st, sh, &v_map, v_ring, v_raw, wait, lane);
		} else if (lane == 0) {
			Piece p;
			Walk walk_on = walk;
			AttnJoin join = {0, 0, 0, 0, 0};
			for (uint32_t n = 0;; n++) {
				const bool any = next_piece<T::TK>(walk_on, p, work, kv, st, a);
				if (any) {
					join = {0, 0, 0, 0, 0};
					if (p.first && !p.whole)  // the CTA's last piece: its item goes on in others
						join = {p.n_parts, p.seq.tok0, p.head, p.row0, p.seq.n_tok * a.group};
				} else {
					a.join[blockIdx.x] = join;
					p.s = -1;
				}
				if (n >= PIECES)
					wait(sh->piece_free[n % PIECES], (n / PIECES & 1u) ^ 1u, true);
				sh->piece[n % PIECES] = p;
				ptx::mbar_arrive(ptx::smem_u32(&sh->piece_full[n % PIECES]));
				if (!any)
					break;
			}
		}
	}
	ptx::tc_fence_before();
	__syncthreads();
	pdl_trigger();	// attn_join may set itself up
	if (warp == W_MMA) {
		ptx::tc_fence_after();
		ptx::tmem_dealloc(tmem, 512);
	}
}

// The parts that CTAs left of the items they shared, joined: a CTA takes 32 rows x 32 dims of an item at a time, its warps the
// parts in turn, a lane a row; they are joined in their order.  A launch of its own: an item of a few tiles of keys a CTA has
// tens of parts of 66 KB, and one CTA, the last at the item, took 130 us to add them up (tree of 13 tokens over 9001 slots:
// 172 us).  Every CTA finds the shared items for itself, so that no more of them are launched than run at once (16 for each CTA
// of the launch before, most with nothing to do: 73.8 us instead of 71.8 for 8 trees of 64 tokens over 3500 keys).
constexpr int JOIN_THREADS = 256, JOIN_WARPS = JOIN_THREADS / 32, JOIN_CTAS = 4;  // CTAs per SM
template <int D, bool SCALED>
__device__ __forceinline__ void join_block(const AttnArgs &a, int c0, int block, float (&s_m)[JOIN_WARPS][32], float (&s_l)[JOIN_WARPS][32], float4 (&s_acc)[JOIN_WARPS][8][32],
					   int lane, int warp)
{
	const AttnJoin it = a.join[c0];
	const int n = it.n, first = (block & 3) * 32, r = first + lane, d40 = (block >> 2) * 8;
	if (it.row0 + first >= it.n_rows)
		return;
	constexpr size_t PART = attn_part_floats(ROWS);
	float top = -INFINITY, sum = 0.0f;
	float4 acc[8];
#pragma unroll
	for (int j = 0; j < 8; j++)
		acc[j] = make_float4(0, 0, 0, 0);
#pragma unroll 2
	for (int i = warp; i < n; i += JOIN_WARPS) {
		const float *part = a.part + (size_t)(2 * (c0 + i) + (i == 0 ? 1 : 0)) * PART;
		float4 v[8];
#pragma unroll
		for (int j = 0; j < 8; j++)
			v[j] = __ldcg(reinterpret_cast<const float4 *>(part) + (d40 + j) * ROWS + r);
		const float m = __ldcg(part + ROWS * 128 + r), l = __ldcg(part + ROWS * 128 + ROWS + r), next = fmaxf(top, m);
		const float f = m == -INFINITY ? 0.0f : exp2_ftz(m - next), g = top == -INFINITY ? 0.0f : exp2_ftz(top - next);
		top = next;
		sum = fmaf(l, f, sum * g);
#pragma unroll
		for (int j = 0; j < 8; j++)
			acc[j] = make_float4(fmaf(v[j].x, f, acc[j].x * g), fmaf(v[j].y, f, acc[j].y * g), fmaf(v[j].z, f, acc[j].z * g), fmaf(v[j].w, f, acc[j].w * g));
	}
	__syncthreads();  // (the block before has been read)
	s_m[warp][lane] = top;
	s_l[warp][lane] = sum;
#pragma unroll
	for (int j = 0; j < 8; j++)
		s_acc[warp][j][lane] = acc[j];
	__syncthreads();
	// a warp: 4 dims of the 32 rows
	top = -INFINITY;
#pragma unroll
	for (int i = 0; i < JOIN_WARPS; i++)
		top = fmaxf(top, s_m[i][lane]);
	sum = 0.0f;
	float4 y = make_float4(0, 0, 0, 0);
#pragma unroll
	for (int i = 0; i < JOIN_WARPS; i++) {
		const float f = s_m[i][lane] == -INFINITY ? 0.0f : exp2_ftz(s_m[i][lane] - top);
		const float4 v = s_acc[i][warp][lane];
		sum = fmaf(s_l[i][lane], f, sum);
		y = make_float4(fmaf(v.x, f, y.x), fmaf(v.y, f, y.y), fmaf(v.z, f, y.z), fmaf(v.w, f, y.w));
	}
	if (it.row0 + r >= it.n_rows)
		return;
	const float inv = sum == 0.0f ? 0.0f : (SCALED ? ATTN_Q8_UP : 1.0f) / sum;
	const int t = (it.row0 + r) / a.group;
	float *dst = a.out + ((long long)(it.tok0 + t) * a.n_head + it.head * a.group + (it.row0 + r - t * a.group)) * D;
	reinterpret_cast<float4 *>(dst)[d40 + warp] = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
}

template <int D, bool SCALED>
__global__ void __launch_bounds__(JOIN_THREADS, JOIN_CTAS) attn_join(const AttnArgs a, int n_cta)
{
	constexpr int BLOCKS = ROWS / 32 * (D / 32);
	__shared__ float s_m[JOIN_WARPS][32], s_l[JOIN_WARPS][32];
	__shared__ float4 s_acc[JOIN_WARPS][8][32];
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
	pdl_wait();
	int unit = blockIdx.x;	// of the shared items that follow; each has BLOCKS
	for (int base = 0; base < n_cta; base += 32) {
		// (all warps find the same)
		uint32_t shared = __ballot_sync(0xffffffffu, base + lane < n_cta && a.join[min(base + lane, n_cta - 1)].n_rows > 0);
		for (; shared; shared &= shared - 1) {
			for (; unit < BLOCKS; unit += gridDim.x)
				join_block<D, SCALED>(a, base + __ffs(shared) - 1, unit, s_m, s_l, s_acc, lane, warp);
			unit -= BLOCKS;
		}
	}
}

template <int KIND, int D>
int go(tie_cuda_ctx *c, const KvView &kv, const StepView &st, const AttnArgs &a)
{
	using T = Tile<KIND, D>;
	CUtensorMap map[2];
	const int rc = attn_maps(c, kv, T::SCALED ? 1 : 2, D, T::BOX_BYTES, T::TK, T::RAW ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, map);
	if (rc)
		return rc;
	attn_tiles<KIND, D><<<c->sm_count, THREADS, T::SMEM, c->stream>>>(kv, st, a, map[0], map[1]);
	TIE_CUDA_LAUNCHED(c);
	return launch_kernel(c, true, 1, attn_join<D, T::SCALED>, dim3(JOIN_CTAS * c->sm_count), JOIN_THREADS, 0, a, c->sm_count);
}
template <int KIND>
int allow_smem(tie_cuda_ctx *c)
{
	TIE_CUDA_TRY(c, cudaFuncSetAttribute(attn_tiles<KIND, 128>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Tile<KIND, 128>::SMEM));
	TIE_CUDA_TRY(c, cudaFuncSetAttribute(attn_tiles<KIND, 64>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Tile<KIND, 64>::SMEM));
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
