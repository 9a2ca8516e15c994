// What a pass over a paged cache hands to its kernels, and how its attention is cut into
// workgroups.  Host code alone.
//
// The rows of a pass are the new tokens of its sequences, one sequence after the other.  The
// query heads that share a kv head are rows too as far as attention goes: row r of a sequence's
// tile axis is token r / group, query head kv_head * group + r % group, so that one token of
// grouped heads and a chunk of tokens are the same thing to a kernel.
#pragma once

#include <algorithm>
#include <climits>
#include <cmath>
#include <unordered_map>
#include <vector>

namespace gh {

struct PassSeq {
    int len;    // positions after the pass
    int first;  // position of its first new row
    int row0;   // index of that row
    int table;  // where its page list begins
};

struct RowAt {
    int slot;  // page * page_tokens + place in the page
    int pos;
};

// One workgroup's work for one kv head: `rows` rows over the positions [k0, k1) of a page list.
struct AttendItem {
    int r0, rows;  // of a sequence's tile axis, or (map >= 0) as the map has them
    int k0, k1;
    int part;          // the place in memory that its result goes to, -1: it is whole and goes to the caller
    int join, joins;   // the joins that wait for it
    int first, row0, table;  // the sequence's; for a map, a position behind all others
    int map;           // rows of several sequences: where their (pass row * group + head of the group) are listed
    int pad;           // a multiple of 16 bytes
};

// A tile whose positions were dealt to several workgroups: the last of them to finish puts it together, first the parts of a
// prefix that it shares with other tiles (rows shared_row.. of those), then its own.
struct AttendJoin {
    int r0, rows, row0;
    int part, parts;
    int shared_part, shared_parts, shared_row;
};

struct AttendPlan {
    std::vector<AttendItem> items;
    std::vector<AttendJoin> joins;
    std::vector<int> maps;
    int parts = 0;  // places that parts need
};

// Sequences of a pass that begin with the same pages: `prefix` positions, all of them before every member's new rows.
struct SharedPrefix {
    int prefix;
    std::vector<int> members;
};

// Those among the sequences with `wanted` set, by their page lists: the ones with the same first page, and as many leading
// full pages as all of them have in common, where that is `least` positions or more.
inline std::vector<SharedPrefix> shared_prefixes(const std::vector<const std::vector<int>*>& pages, const std::vector<PassSeq>& seqs,
                                                 const std::vector<char>& wanted, int page_tokens, int least) {
    std::unordered_map<int, std::vector<int>> by_first;
    for (size_t i = 0; i < seqs.size(); i++)
        if (wanted[i] && seqs[i].first >= std::max(least, page_tokens)) by_first[(*pages[i])[0]].push_back(static_cast<int>(i));
    std::vector<SharedPrefix> found;
    for (auto& [page, members] : by_first) {
        if (members.size() < 2) continue;
        const std::vector<int>& lead = *pages[static_cast<size_t>(members[0])];
        int common = seqs[static_cast<size_t>(members[0])].first / page_tokens;
        for (int m : members) {
            const std::vector<int>& other = *pages[static_cast<size_t>(m)];
            common = std::min(common, seqs[static_cast<size_t>(m)].first / page_tokens);
            int n = 0;
            while (n < common && other[static_cast<size_t>(n)] == lead[static_cast<size_t>(n)]) n++;
            common = n;
        }
        if (common * page_tokens >= least) found.push_back({common * page_tokens, members});
    }
    std::sort(found.begin(), found.end(), [](const SharedPrefix& a, const SharedPrefix& b) { return a.members[0] < b.members[0]; });
    return found;
}

// Positions that rows [r0, r0 + rows) see any of.
inline void visible_span(const PassSeq& s, int r0, int rows, int group, bool causal, int window, int& k0, int& k1) {
    const int t0 = s.first + r0 / group, t1 = s.first + (r0 + rows - 1) / group;
    k1 = causal ? t1 + 1 : s.len;
    k0 = window > 0 ? std::max(0, t0 - window + 1) & ~15 : 0;
}

struct AttendCut {
    int group, kv_heads;
    int height;      // of a tile
    bool causal;
    int window;
    int workgroups;  // about as many, over all kv heads
    int least;       // positions of a part, at least
    int most;        // parts of a tile, at most
    int square = 0;    // ... and, if not 0, sqrt(positions / square): the last part to end joins them all, so n parts take
                       // positions / n + square n.  A tile of 1 / r-th the height has a join of 1 / r-th the time
    int resident = 0;  // if not 0: no more workgroups than this many where there are fewer tiles (one more is a round of its own)
};

// Tiles of `height` rows; a tile's positions are cut into parts of one length.  `shared`: prefixes whose members (of at
// most `height` rows each) meet them in common tiles; only without a window, where all their rows see all of it.
inline AttendPlan plan_attend(const std::vector<PassSeq>& seqs, const std::vector<int>& rows, const AttendCut& cut,
                              const std::vector<SharedPrefix>& shared = {}) {
    AttendPlan plan;
    const int height = cut.height;
    std::vector<int> prefix(seqs.size(), 0);  // that a sequence leaves to the common tiles
    std::vector<int> packed(shared.size(), 0);  // common tiles of a prefix: members whole, as many as fit
    for (size_t g = 0; g < shared.size(); g++) {
        int room = 0;
        for (int i : shared[g].members) {
            prefix[static_cast<size_t>(i)] = shared[g].prefix;
            const int n = rows[static_cast<size_t>(i)] * cut.group;
            if (n > room) {
                packed[g]++;
                room = height;
            }
            room -= n;
        }
    }
    const auto tile_span = [&](size_t i, int r0, int& n, int& k0, int& k1) {
        n = std::min(height, rows[i] * cut.group - r0);
        visible_span(seqs[i], r0, n, cut.group, cut.causal, cut.window, k0, k1);
        k0 = std::max(k0, prefix[i]);
    };
    long long total = 0;
    for (size_t i = 0; i < seqs.size(); i++)
        for (int r0 = 0; r0 < rows[i] * cut.group; r0 += height) {
            int n, k0, k1;
            tile_span(i, r0, n, k0, k1);
            total += k1 - k0;
        }
    for (size_t g = 0; g < shared.size(); g++) total += static_cast<long long>(shared[g].prefix) * packed[g];
    const long long each = (total * cut.kv_heads + cut.workgroups - 1) / std::max(cut.workgroups, 1);
    long long span = std::max<long long>(cut.least, (each + 127) / 128 * 128);
    // the length of the parts of [k0, k1), as even as whole runs of 32 positions allow, and their number
    const auto cut_up = [&](int n, int k0, int k1, int& run) {
        int most = cut.most;
        if (cut.square > 0) most = std::min(most, static_cast<int>(std::sqrt(static_cast<double>(k1 - k0) * height / n / cut.square) + 0.5));
        const int parts = std::max(1, static_cast<int>(std::min<long long>(most, (k1 - k0 + span - 1) / span)));
        run = (((k1 - k0 + parts - 1) / parts) + 31) / 32 * 32;
        return std::max(1, (k1 - k0 + run - 1) / run);
    };
    if (cut.resident > 0) {
        const auto count = [&](bool whole) {
            long long items = 0;
            for (size_t i = 0; i < seqs.size(); i++)
                for (int r0 = 0; r0 < rows[i] * cut.group; r0 += height) {
                    int n, k0, k1, run;
                    tile_span(i, r0, n, k0, k1);
                    items += whole ? 1 : cut_up(n, k0, k1, run);
                }
            return items * cut.kv_heads;
        };
        if (count(true) <= cut.resident)
            while (count(false) > cut.resident) span += std::max(32ll, span / 8 / 32 * 32);
    }
    const auto add_items = [&](AttendItem it, int k0, int k1, int parts, int run) {
        for (int j = 0; j < parts; j++) {
            it.k0 = k0 + j * run;
            it.k1 = std::min(k1, k0 + (j + 1) * run);
            plan.items.push_back(it);
            if (it.part >= 0) it.part++;
        }
    };
    const auto add_tile = [&](size_t i, int r0, AttendJoin join) {
        int n, k0, k1, run;
        tile_span(i, r0, n, k0, k1);
        const int parts = cut_up(n, k0, k1, run);
        const bool whole = parts == 1 && join.shared_parts == 0;
        AttendItem it{r0, n, 0, 0, whole ? -1 : plan.parts, static_cast<int>(plan.joins.size()), whole ? 0 : 1,
                      seqs[i].first, seqs[i].row0, seqs[i].table, -1, 0};
        add_items(it, k0, k1, parts, run);
        if (whole) return;
        join.r0 = r0;
        join.rows = n;
        join.row0 = seqs[i].row0;
        join.part = plan.parts;
        join.parts = parts;
        plan.joins.push_back(join);
        plan.parts += parts;
    };
    for (size_t g = 0; g < shared.size(); g++) {
        const std::vector<int>& members = shared[g].members;
        int run;
        const int parts = cut_up(height, 0, shared[g].prefix, run);
        for (size_t m = 0; m < members.size();) {
            AttendItem it{0, 0, 0, 0, plan.parts, static_cast<int>(plan.joins.size()), 0, INT_MAX - 1024, 0,
                          seqs[static_cast<size_t>(members[m])].table, static_cast<int>(plan.maps.size()), 0};
            plan.parts += parts;
            for (; m < members.size(); m++) {
                const size_t i = static_cast<size_t>(members[m]);
                const int n = rows[i] * cut.group;
                if (it.rows + n > height) break;
                for (int r = 0; r < n; r++) plan.maps.push_back((seqs[i].row0 + r / cut.group) * cut.group + r % cut.group);
                add_tile(i, 0, AttendJoin{0, 0, 0, 0, 0, it.part, parts, it.rows});
                it.rows += n;
                it.joins++;
            }
            add_items(it, 0, shared[g].prefix, parts, run);
        }
    }
    for (size_t i = 0; i < seqs.size(); i++)
        if (prefix[i] == 0)
            for (int r0 = 0; r0 < rows[i] * cut.group; r0 += height) add_tile(i, r0, AttendJoin{});
    // the longest go first: what is dealt last ends the launch
    std::stable_sort(plan.items.begin(), plan.items.end(), [](const AttendItem& a, const AttendItem& b) { return a.k1 - a.k0 > b.k1 - b.k0; });
    return plan;
}

}  // namespace gh
