// The paged key/value cache and the tokens of a step as the kernels of kv_cache.cu and attn.cu see them.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace tie {

constexpr int KV_MAX_SEQ = 1024;      // sequences of a step
constexpr int KV_MAX_TREE = 64;	      // tokens of a sequence whose step has a tree: the bits of a mask
constexpr int KV_MIN_PAGE_SHIFT = 4;  // pages of 16 slots and more: a group of 16 keys lies in one page

struct KvView {
	uint8_t *k, *v;		 // [n_pages][n_head_kv][page_size] rows of head_dim values
	float *k_scale, *v_scale;  // Q8: one factor per row
	int n_head_kv, page_shift, n_pages;
};

struct StepView {
	const int *tok_start, *kv_len, *page_table;
	const unsigned long long *tree;	 // or null: a token sees the step's tokens up to itself
	const int *pos;			 // or null: the slot
	int n_seq, n_tokens, max_pages;
	unsigned *status;
};

__host__ __device__ __forceinline__ void kv_report(const StepView &st, unsigned bit)
{
#ifdef __CUDA_ARCH__
	atomicOr(st.status, bit);
#else
	*st.status |= bit;  // (the index functions below are tested on the host)
#endif
}

// One sequence of a step with everything that the kernels rely on made sure of: lengths are not negative, its tokens lie
// inside [0, n_tokens) and its slots inside its row of the page table.  Whatever else the arrays say is reported and cut off.
struct SeqView {
	int tok0, n_tok, kv_len;
};
__host__ __device__ __forceinline__ SeqView kv_sequence(const StepView &st, int page_shift, int s)
{
	SeqView q = {st.tok_start[s], st.tok_start[s + 1], st.kv_len[s]};
	const int end = q.n_tok;
	bool bad = q.tok0 < 0 || end < q.tok0 || end > st.n_tokens || q.kv_len < 0;
	q.n_tok = bad ? 0 : end - q.tok0;
	q.kv_len = bad ? 0 : q.kv_len;
	const long long room = (long long)st.max_pages << page_shift;
	if (q.kv_len > room) {
		bad = true;
		q.kv_len = 0;
		q.n_tok = 0;
	} else if (q.kv_len + (long long)q.n_tok > room) {  // the last tokens have no slots
		bad = true;
		q.n_tok = (int)(room - q.kv_len);
	}
	if (bad)
		kv_report(st, ST_BAD_STEP);
	return q;
}

// The sequence of row t, by a whole warp: -1 where no sequence has it.  One round of 32 starts, or two (KV_MAX_SEQ = 32 x 32).
__device__ __forceinline__ int kv_find_sequence(const StepView &st, int t, int lane)
{
	int stride = st.n_seq, s = 0;
	if (stride > 32) {
		stride = (st.n_seq + 31) >> 5;
		const int end = min((lane + 1) * stride, st.n_seq);
		s = __popc(__ballot_sync(0xffffffffu, t >= st.tok_start[end])) * stride;
	}
	const bool past = lane < stride && s + lane < st.n_seq && t >= st.tok_start[s + lane + 1];
	s += __popc(__ballot_sync(0xffffffffu, past));
	return s < st.n_seq && t >= st.tok_start[s] && t < st.tok_start[s + 1] ? s : -1;
}

// The same by one thread.
__host__ __device__ __forceinline__ int kv_find_sequence_alone(const StepView &st, int t)
{
	int lo = 0, hi = st.n_seq;  // the first sequence that ends behind t is in [lo, hi]
	while (lo < hi) {
		const int mid = (lo + hi) >> 1;
		if (t >= st.tok_start[mid + 1])
			lo = mid + 1;
		else
			hi = mid;
	}
	return lo < st.n_seq && t >= st.tok_start[lo] ? lo : -1;
}

// First row of (page, head), or -1 (reported) where the page is none of the cache's.
__host__ __device__ __forceinline__ long long kv_page_row(const KvView &kv, const StepView &st, int page, int head)
{
	if ((unsigned)page >= (unsigned)kv.n_pages) {
		kv_report(st, ST_BAD_PAGE);
		return -1;
	}
	return ((long long)page * kv.n_head_kv + head) << kv.page_shift;
}

}  // namespace tie
