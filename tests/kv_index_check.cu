// Host check of the index functions that every kernel of the paged cache reaches memory through (csrc/kv_cache.cuh):
// over steps that are right and steps whose arrays say anything at all, no row and no slot outside what they are for.
#include <stdio.h>
#include <stdlib.h>
#include <vector>

#include "../tie_b200/csrc/kv_cache.cuh"

using namespace tie;

static unsigned long long state = 1;
static int rnd(int lo, int hi)
{
	state = state * 6364136223846793005ull + 1442695040888963407ull;
	return lo + (int)((state >> 33) % (unsigned long long)(hi - lo + 1));
}

int main()
{
	int bad_reported = 0;
	for (int round = 0; round < 20000; round++) {
		const int shift = rnd(4, 7), n_seq = rnd(1, round % 50 == 0 ? 1024 : 40), max_pages = rnd(1, 6), n_tokens = rnd(0, 300);
		const int n_pages = rnd(1, 50), heads = rnd(1, 8), room = max_pages << shift;
		const bool wild = round % 2;
		std::vector<int> start(n_seq + 1), len(n_seq), table(n_seq * max_pages);
		int at = 0;
		for (int s = 0; s <= n_seq; s++) {
			start[s] = at;
			if (s < n_seq) {
				int n = rnd(0, 3) ? rnd(0, 5) : 0;
				n = at + n > n_tokens ? 0 : n;
				n = n > room ? room : n;
				at += n;
				len[s] = rnd(0, room - n);
			}
		}
		for (int &p : table)
			p = wild && !rnd(0, 3) ? (rnd(0, 1) ? rnd(-2147483647, -1) : rnd(n_pages, 2147483647)) : rnd(0, n_pages - 1);
		if (wild)
			for (int i = 0; i < 4; i++) {
				const int s = rnd(0, n_seq);
				switch (rnd(0, 3)) {
				case 0: start[s] = rnd(-5, n_tokens + 400); break;
				case 1: start[s] = rnd(0, 1) ? -2147483647 - 1 : 2147483647; break;
				case 2: if (s < n_seq) len[s] = rnd(-3, room + 30); break;
				default: if (s < n_seq) len[s] = rnd(0, 1) ? -2147483647 - 1 : 2147483647;
				}
			}
		unsigned status = 0;
		const StepView st = {start.data(), len.data(), table.data(), nullptr, nullptr, n_seq, n_tokens, max_pages, &status};
		const KvView kv = {nullptr, nullptr, nullptr, nullptr, heads, shift, n_pages};
		for (int s = 0; s < n_seq; s++) {
			const SeqView q = kv_sequence(st, shift, s);
			const bool ok = q.n_tok >= 0 && q.kv_len >= 0 && q.kv_len + (long long)q.n_tok <= room &&
					(q.n_tok == 0 || (q.tok0 >= 0 && q.tok0 + (long long)q.n_tok <= n_tokens));
			if (!ok || (!wild && (q.tok0 != start[s] || q.n_tok != start[s + 1] - start[s] || q.kv_len != len[s]))) {
				printf("round %d sequence %d: %d %d %d\n", round, s, q.tok0, q.n_tok, q.kv_len);
				return 1;
			}
		}
		if (!wild && status) {
			printf("round %d: a right step was reported\n", round);
			return 1;
		}
		bad_reported += wild && status;
		for (int t = 0; t < n_tokens; t++) {
			const int s = kv_find_sequence_alone(st, t);
			int want = -1;
			for (int i = 0; i < n_seq && !wild; i++)
				if (t >= start[i] && t < start[i + 1])
					want = i;
			if (s < -1 || s >= n_seq || (!wild && s != want) || (s >= 0 && !(t >= start[s] && t < start[s + 1]))) {
				printf("round %d row %d: sequence %d, not %d\n", round, t, s, want);
				return 1;
			}
		}
		for (int p : table) {
			const long long row = kv_page_row(kv, st, p, heads - 1);
			if (row < -1 || (row >= 0 && row + (1 << shift) > (long long)n_pages * heads << shift) || (row < 0) != (p < 0 || p >= n_pages)) {
				printf("round %d page %d: row %lld\n", round, p, row);
				return 1;
			}
		}
	}
	printf("ok, %d steps reported\n", bad_reported);
	return bad_reported > 1000 ? 0 : 1;
}
