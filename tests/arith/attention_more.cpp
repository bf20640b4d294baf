// Attention with first tokens beside a window, and with prefixes that sequences share: the keys of the workgroups and the
// parts that are joined, from the library's own header.  Each line of standard input is a call; the answer is the number
// of its rows that something goes wrong with.
//   sinks total most_q most_kv window causal heads group head_dim type lse shift sinks seqs, seqs + 1 starts, seqs lengths
//   shared total most_q most_kv causal heads group head_dim type lse shift groups given most_len most_rows seqs, seqs + 1
//          starts, seqs lengths, groups + 1 firsts (if given), groups lengths
#include <iostream>
#include <map>
#include <sstream>
#include <string>
#include <vector>

#include "attention_plan.h"

namespace {

struct Plain {
    const int32_t *table, *starts, *kv_len;
    int64_t width;
    struct { int shift; } c;
    int total, most_q, most_kv, window, causal, seqs, splits, chunk;
};
struct Args : Plain {
    static constexpr bool MORE = true;
    int pass, sinks;
    const int32_t *group_first, *shared_len;
    int groups, most_shared, all_seqs, prefix_splits, prefix_chunk, prefix_rows;
};

using Taken = std::map<int, int>;  // key -> times

// What a row takes in the workgroup of `split` of its tile, step by step; whether the kernel writes it there, and where.
template <int KEYS>
bool walk(const Args& a, const iq4xs::Sequence& s, int fresh, int tile, int row, int group, int split, Taken& taken,
          iq4xs::RowEnd& end, bool& ok) {
    const int row0 = row / tile * tile, rows = s.fresh * group;
    const int last = (rows < row0 + tile ? rows : row0 + tile) - 1;
    const int any_lo = iq4xs::least_key(a, s, fresh, row0 / group), any_hi = iq4xs::end_key(a, s, fresh, last / group);
    const int all_lo = iq4xs::least_key(a, s, fresh, last / group), all_hi = iq4xs::end_key(a, s, fresh, row0 / group);
    const int lo = iq4xs::least_key(a, s, fresh, row / group), hi = iq4xs::end_key(a, s, fresh, row / group);
    int k0, k1, extra;
    if (!iq4xs::split_keys_more(a, s, any_lo, any_hi, split, k0, k1, extra)) return false;
    end = iq4xs::row_end_more(a, s, lo, hi, split);
    const iq4xs::KeySteps<KEYS, true> span(k0, k1, extra);
    for (int base = span.start; base < k1; base += KEYS) {
        const bool all = span.all_see(base, all_lo, all_hi);
        for (int i = 0; i < KEYS; ++i) {
            const int key = span.place(base) + i;
            const bool in = key < span.stop(base) && key >= span.lo_in(base, lo) && key < span.hi_in(base, hi);
            const bool some = key < span.stop(base) && key >= span.lo_in(base, any_lo) && key < span.hi_in(base, any_hi);
            // 16 keys of which some are past the end are masked as a whole's parts, whatever `all` says
            ok = ok && (!all || in || key >= span.stop(base) / 16 * 16) && (!in || some);
            if (in) ++taken[key];
        }
        ok = ok && span.place(base) % 16 == 0;
    }
    return true;
}

bool walk(const Args& a, const iq4xs::AttentionPlan& p, const iq4xs::Sequence& s, int fresh, int row, int group, int split,
          Taken& taken, iq4xs::RowEnd& end, bool& ok) {
    return p.tiles ? walk<32>(a, s, fresh, 16 * p.tiles, row, group, split, taken, end, ok)
                   : walk<64>(a, s, fresh, 128, row, group, split, taken, end, ok);
}

// Rows of a sequence whose keys do not reach them exactly once, or whose parts are joined otherwise than written.
int64_t wrong_of_sinks(const Args& a, const iq4xs::AttentionPlan& p, int seq, int group) {
    int fresh;
    const iq4xs::Sequence s = iq4xs::sequence_more(a, seq, fresh);
    int64_t wrong = 0;
    for (int row = 0; row < s.fresh * group; ++row) {
        const int token = row / group;
        const int lo = iq4xs::least_key(a, s, fresh, token), hi = iq4xs::end_key(a, s, fresh, token);
        const bool one = iq4xs::one_split_more(a, s, lo, hi);
        std::vector<int> joined(p.splits, 0);
        bool ok = row / (p.tiles ? 16 * p.tiles : 128) < p.row_tiles;
        if (!one) {
            const iq4xs::RowParts parts = iq4xs::row_parts(a, s, lo, hi);
            for (int i = 0; i < parts.count(); ++i) {
                const int at = parts.at(i);
                if (at < 0 || at >= p.splits) ok = false; else ++joined[at];
            }
        }
        Taken all;
        int outs = 0;
        for (int split = 0; split < p.splits; ++split) {
            Taken mine;
            iq4xs::RowEnd end = iq4xs::ROW_NONE;
            const bool live = walk(a, p, s, fresh, row, group, split, mine, end, ok);
            outs += live && end == iq4xs::ROW_OUT;
            ok = ok && (joined[split] == 0 || (joined[split] == 1 && live && end == iq4xs::ROW_PART));
            if (!mine.empty()) ok = ok && (end == iq4xs::ROW_OUT || (end == iq4xs::ROW_PART && joined[split] == 1));
            for (auto& k : mine) all[k.first] += k.second;
        }
        ok = ok && outs == (one ? 1 : 0);
        const int64_t at = (int64_t)s.keys - fresh + token;
        int64_t seen = 0;
        for (int64_t j = 0; j < s.keys; ++j) {
            const bool sees = (!a.causal || j <= at) && (a.window == 0 || j > at - a.window || j < a.sinks);
            seen += sees;
            if (sees) ok = ok && all.count((int)j) && all[(int)j] == 1;
        }
        ok = ok && (int64_t)all.size() == seen;
        wrong += !ok;
    }
    return wrong;
}

int64_t wrong_of_shared(const Args& first, const Args& own, const iq4xs::SharedPlan& p, int group) {
    int64_t wrong = 0;
    for (int seq = 0; seq < own.all_seqs; ++seq) {
        int fresh;
        const iq4xs::Sequence s = iq4xs::sequence_more(own, seq, fresh);
        const int g = iq4xs::group_of(own, seq);
        for (int row = 0; row < s.fresh * group; ++row) {
            const int token = row / group, at = s.first + token;
            const int lo = iq4xs::least_key(own, s, fresh, token), hi = iq4xs::end_key(own, s, fresh, token);
            bool ok = !iq4xs::one_split_more(own, s, lo, hi) && at >= 0 && at < own.total;
            iq4xs::RowParts parts = iq4xs::row_parts(own, s, lo, hi);
            parts.before = iq4xs::prefix_parts(own, iq4xs::shared_keys(own, g));
            Taken all;
            std::vector<int> written(p.parts(), 0);
            for (int split = 0; split < p.own.splits; ++split) {
                Taken mine;
                iq4xs::RowEnd end = iq4xs::ROW_NONE;
                if (walk(own, p.own, s, fresh, row, group, split, mine, end, ok)) {
                    ok = ok && end == iq4xs::ROW_PART;
                    written[p.prefix.splits + split] = 1;
                    for (auto& k : mine) all[k.first] += k.second, written[p.prefix.splits + split] = 2;
                }
            }
            int64_t shared = 0;
            if (parts.before > 0) {
                const int from = own.group_first ? own.group_first[g] : 0;
                if (at - own.starts[from] >= own.prefix_rows) continue;  // not written
                int group_fresh;
                const iq4xs::Sequence f = iq4xs::sequence_more(first, g, group_fresh);
                const int group_row = (at - f.first) * group + row % group;
                ok = ok && at - f.first < f.fresh && f.pages == first.table + from * first.width;
                for (int split = 0; split < p.prefix.splits; ++split) {
                    Taken mine;
                    iq4xs::RowEnd end = iq4xs::ROW_NONE;
                    if (walk(first, p.prefix, f, group_fresh, group_row, group, split, mine, end, ok)) {
                        ok = ok && end == iq4xs::ROW_PART;
                        written[split] = 1;
                        for (auto& k : mine) all[k.first] += k.second, written[split] = 2;
                    }
                }
                shared = f.keys;
            }
            for (int i = 0; i < parts.count(); ++i) {
                const int part = parts.at(i);
                ok = ok && part >= 0 && part < p.parts() && written[part] != 0;
                if (part >= 0 && part < p.parts()) written[part] = 0;
            }
            for (int x : written) ok = ok && x != 2;  // every part with keys is joined
            const int64_t place = (int64_t)s.keys - fresh + token;
            int64_t seen = 0;
            for (int64_t j = 0; j < (s.keys > shared ? s.keys : shared); ++j) {
                const bool sees = j < shared || (j < s.keys && (!own.causal || j <= place));
                seen += sees;
                if (sees) ok = ok && all.count((int)j) && all[(int)j] == 1;
            }
            ok = ok && (int64_t)all.size() == seen;
            wrong += !ok;
        }
    }
    return wrong;
}

}  // namespace

int main() {
    std::string line, kind;
    while (std::getline(std::cin, line)) {
        std::istringstream in(line);
        iq4xs_kv_cache cache = {};
        iq4xs_paged_attention_args g = {};
        iq4xs_shared_prefix x = {};
        int64_t heads, group, head_dim, type, lse, causal, shift, sinks = 0, given = 0;
        in >> kind >> g.total >> g.most_q >> g.most_kv;
        if (kind == "sinks") in >> g.window;
        in >> causal >> heads >> group >> head_dim >> type >> lse >> shift;
        if (kind == "sinks") in >> sinks;
        else in >> x.groups >> given >> x.most_len >> x.most_rows;
        in >> g.seqs;
        std::vector<int32_t> starts(g.seqs + 1), kv(g.seqs), firsts(given ? x.groups + 1 : 0), lens(x.groups);
        for (auto& y : starts) in >> y;
        for (auto& y : kv) in >> y;
        for (auto& y : firsts) in >> y;
        for (auto& y : lens) in >> y;
        if (!in) return 1;
        float some = 0;
        cache.heads = (int32_t)heads;
        cache.head_dim = (int32_t)head_dim;
        cache.type = (int32_t)type;
        g.cache = &cache;
        g.q_heads = (int32_t)(heads * group);
        g.out_type = IQ4XS_TYPE_BF16;
        g.causal = (int32_t)causal;
        g.lse = lse ? &some : nullptr;
        x.path = IQ4XS_SHARED_ONCE;
        x.first = given ? firsts.data() : nullptr;
        x.len = lens.data();
        static const int32_t table[1] = {0};
        const int64_t width = 1 << 20;
        auto plain = [&](const iq4xs_paged_attention_args& c, const iq4xs::AttentionPlan& p) {
            return Plain{table, starts.data(), kv.data(), width, {(int)shift}, (int)c.total, (int)c.most_q,
                         iq4xs::most_kv_of(c), (int)iq4xs::window_of(c), c.causal, (int)c.seqs, p.splits, p.chunk};
        };
        int64_t wrong = 0;
        if (kind == "sinks") {
            iq4xs::AttentionPlan p;
            if (!iq4xs::plan_fits(g, 256, p)) return 1;
            const Args a{plain(g, p), iq4xs::PASS_SINKS, (int)sinks, nullptr, nullptr, 0, 0, (int)g.seqs, 0, 0, 0};
            for (int seq = 0; seq < g.seqs; ++seq) wrong += wrong_of_sinks(a, p, seq, (int)group);
        } else {
            iq4xs::SharedPlan p;
            if (!iq4xs::shared_plan_fits(g, x, 256, p)) return 1;
            const iq4xs_paged_attention_args pre = iq4xs::prefix_call(g, x);
            Args a{plain(pre, p.prefix), iq4xs::PASS_PREFIX, 0, x.first, x.len, (int)x.groups, (int)x.most_len, (int)g.seqs,
                   p.prefix.splits, p.prefix.chunk, (int)x.most_rows};
            Args b = a;
            static_cast<Plain&>(b) = plain(g, p.own);
            b.pass = iq4xs::PASS_OWN;
            wrong = wrong_of_shared(a, b, p, (int)group);
        }
        std::cout << wrong << "\n";
    }
}
