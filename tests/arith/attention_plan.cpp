// The plan of attention calls and the keys of their workgroups, from the library's own header.  Each line of standard
// input is a call; the answer is the number of its rows that something goes wrong with.
//   total most_q most_kv window causal heads group head_dim type out_type lse table_width shift seqs
//       then seqs + 1 starts and seqs lengths
// or the word keys, the key that the kernels' places must stay below, and a call as above; the answer is 1 if some
// sequence has more keys than that.
#include <iostream>
#include <sstream>
#include <string>
#include <vector>

#include "attention_plan.h"

namespace {

struct Args {
    const int32_t *table, *starts, *kv_len;
    int64_t width;
    struct { int shift; } c;
    int total, most_q, most_kv, window, causal, splits, chunk;
};

// Rows of the sequence whose keys do not reach them exactly once, or whose sums the join would look for elsewhere.
int64_t wrong_rows(const Args& a, const iq4xs::AttentionPlan& p, int seq, int group) {
    int total_fresh;
    const iq4xs::Sequence s = iq4xs::sequence(a, seq, total_fresh);
    const int tile = p.tiles ? 16 * p.tiles : 128;
    int64_t wrong = 0;
    for (int row = 0; row < s.fresh * group; ++row) {
        const int token = row / group, row0 = row / tile * tile;
        if (row / tile >= p.row_tiles) {
            ++wrong;
            continue;
        }
        const int last = (s.fresh * group < row0 + tile ? s.fresh * group : row0 + tile) - 1;
        // what the row sees, from the definition
        const int64_t at = (int64_t)s.keys - total_fresh + token;
        int64_t lo = a.window > 0 && at + 1 - a.window > 0 ? at + 1 - a.window : 0, hi = a.causal ? at + 1 : s.keys;
        if (hi > s.keys) hi = s.keys;
        if (hi < 0) hi = 0;
        const bool some = hi > lo;
        const int l = iq4xs::least_key(a, s, total_fresh, token), h = iq4xs::end_key(a, s, total_fresh, token);
        bool ok = some ? l == lo && h == hi : h <= l;
        int first = 0, end = -1;
        const bool one = iq4xs::one_split(a, s, l, h);
        if (!one) iq4xs::splits_of(a, s, l, h, first, end);
        ok = ok && (one || !some || (first >= 0 && end < p.splits)) && (some || one || end < first);
        int64_t next = lo;  // the first key not yet taken
        int outs = 0;
        for (int split = 0; split < p.splits; ++split) {
            int k0, k1;
            const int any_lo = iq4xs::least_key(a, s, total_fresh, row0 / group);
            const int any_hi = iq4xs::end_key(a, s, total_fresh, last / group);
            const bool live = iq4xs::split_keys(a, s, any_lo, any_hi, split, k0, k1);
            const bool read = !one && split >= first && split <= end;
            if (!live) {
                ok = ok && !read;
                continue;
            }
            const iq4xs::RowEnd to = iq4xs::row_end(a, s, l, h, split);
            outs += to == iq4xs::ROW_OUT;
            const int64_t from = k0 > lo ? k0 : lo, up = k1 < hi ? k1 : hi;
            if (up > from) {
                ok = ok && from == next && (to == iq4xs::ROW_OUT || (to == iq4xs::ROW_PART && read));
                next = up;
            }
            ok = ok && (!read || to == iq4xs::ROW_PART);
        }
        ok = ok && (!some || next == hi) && outs == (one ? 1 : 0);
        wrong += !ok;
    }
    return wrong;
}

}  // namespace

int main() {
    std::string line;
    while (std::getline(std::cin, line)) {
        std::istringstream in(line);
        const bool ask_keys = line.compare(0, 5, "keys ") == 0;
        int64_t below = 0;
        std::string word;
        if (ask_keys) in >> word >> below;
        iq4xs_kv_cache cache = {};
        iq4xs_paged_attention_args g = {};
        int64_t heads, group, head_dim, type, out_type, lse, causal, shift;
        in >> g.total >> g.most_q >> g.most_kv >> g.window >> causal >> heads >> group >> head_dim >> type >> out_type >>
            lse >> g.table_width >> shift >> g.seqs;
        std::vector<int32_t> starts(g.seqs + 1), kv(g.seqs);
        for (auto& x : starts) in >> x;
        for (auto& x : kv) in >> x;
        if (!in) return 1;
        float some = 0;
        cache.heads = (int32_t)heads;
        cache.head_dim = (int32_t)head_dim;
        cache.type = (int32_t)type;
        g.cache = &cache;
        g.q_heads = (int32_t)(heads * group);
        g.out_type = (int32_t)out_type;
        g.causal = (int32_t)causal;
        g.lse = lse ? &some : nullptr;
        const iq4xs::AttentionPlan p = iq4xs::plan_of(g, 256);
        const Args a{nullptr, starts.data(), kv.data(), g.table_width, {(int)shift}, (int)g.total, (int)g.most_q,
                     iq4xs::most_kv_of(g), (int)iq4xs::window_of(g), g.causal, p.splits, p.chunk};
        if (ask_keys) {
            bool more = false;
            for (int seq = 0; seq < g.seqs; ++seq) {
                int total_fresh;
                more = more || iq4xs::sequence(a, seq, total_fresh).keys > below;
            }
            std::cout << more << "\n";
            continue;
        }
        int64_t wrong = p.splits < 1 || p.chunk < 1 || p.grid < 1;
        for (int seq = 0; seq < g.seqs && !wrong; ++seq) wrong += wrong_rows(a, p, seq, (int)group);
        std::cout << wrong << "\n";
    }
}
