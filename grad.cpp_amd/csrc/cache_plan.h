// What a pass over a paged cache hands to its kernels, and how its attention is cut into
// workgroups.  Host code alone.
//
// The rows of a pass are the new tokens of its sequences, one sequence after the other.  The
// query heads that share a kv head are rows too as far as attention goes: row r of a sequence's
// tile axis is token r / group, query head kv_head * group + r % group, so that one token of
// grouped heads and a chunk of tokens are the same thing to a kernel.
#pragma once

#include <algorithm>
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

// One workgroup's work for one kv head: rows [r0, r0 + rows) of a sequence's tile axis over the
// positions [k0, k1).  The parts of a tile meet through `tile`'s counter and the parts' places.
struct AttendItem {
    int seq, r0, rows, k0, k1;
    int part;   // place of the tile's first part among all that are left in memory, -1: the only part
    int index;  // which part this is
    int parts;
    int tile;
    int first, row0, table;  // the sequence's, so that a kernel has them with the rest
};

struct AttendPlan {
    std::vector<AttendItem> items;
    int parts = 0;  // places that split tiles need
    int tiles = 0;  // counters that they need
};

// Positions that rows [r0, r0 + rows) see any of.
inline void visible_span(const PassSeq& s, int r0, int rows, int group, bool causal, int window, int& k0, int& k1) {
    const int t0 = s.first + r0 / group, t1 = s.first + (r0 + rows - 1) / group;
    k1 = causal ? t1 + 1 : s.len;
    k0 = window > 0 ? std::max(0, t0 - window + 1) & ~15 : 0;
}

// Tiles of `height` rows; a tile's positions are cut into parts of one length so that the launch has about
// `workgroups` of them over all kv heads, none shorter than `least` positions and no tile in more than `most` parts.
inline AttendPlan plan_attend(const std::vector<PassSeq>& seqs, const std::vector<int>& rows, int group, int kv_heads, int height,
                              bool causal, int window, int workgroups, int least, int most) {
    AttendPlan plan;
    long long total = 0;
    for (size_t i = 0; i < seqs.size(); i++)
        for (int r0 = 0; r0 < rows[i] * group; r0 += height) {
            int k0, k1;
            visible_span(seqs[i], r0, std::min(height, rows[i] * group - r0), group, causal, window, k0, k1);
            total += k1 - k0;
        }
    const long long each = (total * kv_heads + workgroups - 1) / std::max(workgroups, 1);
    const int span = static_cast<int>(std::min<long long>(std::max<long long>(least, (each + 127) / 128 * 128), 1 << 30));
    for (size_t i = 0; i < seqs.size(); i++) {
        const int all = rows[i] * group;
        for (int r0 = 0; r0 < all; r0 += height) {
            const int n = std::min(height, all - r0);
            int k0, k1;
            visible_span(seqs[i], r0, n, group, causal, window, k0, k1);
            const int parts = std::max(1, std::min(most, (k1 - k0 + span - 1) / span));
            const int part = parts > 1 ? plan.parts : -1, tile = parts > 1 ? plan.tiles : 0;
            // as even as whole runs of 32 positions allow
            const int run = (((k1 - k0 + parts - 1) / parts) + 31) / 32 * 32;
            const int made = std::max(1, (k1 - k0 + run - 1) / run);
            for (int j = 0; j < made; j++)
                plan.items.push_back({static_cast<int>(i), r0, n, k0 + j * run, std::min(k1, k0 + (j + 1) * run), made > 1 ? part : -1, j, made, tile, seqs[i].first, seqs[i].row0, seqs[i].table});
            if (made > 1) {
                plan.parts += made;
                plan.tiles++;
            }
        }
    }
    // the longest go first: what is dealt last ends the launch
    std::stable_sort(plan.items.begin(), plan.items.end(), [](const AttendItem& a, const AttendItem& b) { return a.k1 - a.k0 > b.k1 - b.k0; });
    return plan;
}

}  // namespace gh
