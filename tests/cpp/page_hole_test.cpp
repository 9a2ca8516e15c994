// Streams that forget as they go: what a pass takes of their page lists, and where items find the pages of the places that their rows see.
// Exit status 0: all held.
#include "../../grad.cpp_amd/csrc/cache_plan.h"
#include "../../grad.cpp_amd/csrc/page_book.h"

#include <chrono>
#include <cstdio>
#include <random>

using namespace gh;

#define CHECK(x)                                                      \
    do {                                                              \
        if (!(x)) {                                                   \
            std::printf("%s:%d: %s\n", __FILE__, __LINE__, #x);       \
            return 1;                                                 \
        }                                                             \
    } while (0)

// As the kernels look a place's page up.
static int page_of(const AttendItem& it, const std::vector<int>& table, int lead, int page_tokens, int v) {
    const int position = lead > 0 && v >= lead ? v + it.gap : v;
    const int at = it.table + position / page_tokens - (lead > 0 && v >= lead ? it.hole() : 0);
    return at >= 0 && at < static_cast<int>(table.size()) ? table[static_cast<size_t>(at)] : -9;
}

static int passes(unsigned seed) {
    std::mt19937 rng(seed);
    const int T = 16 << (rng() % 3);
    PageBook book(4000, T);
    const int sinks = rng() % 3 ? static_cast<int>(rng() % 40) : 0, window = 1 + static_cast<int>(rng() % 300), lead = sinks_lead(sinks);
    std::vector<int> ids;
    for (int i = 0; i < 4; i++) ids.push_back(book.add());
    for (int step = 0; step < 60; step++) {
        std::vector<int> counts;
        for (int id : ids) {
            const int length = book.at(id).length;
            if (rng() % 4 == 0) {  // back to somewhere behind what is forgotten, or inside it
                const int least = rng() % 8 ? book.at(id).gone_to : book.at(id).gone_from;
                if (length > least) book.truncate(id, least + static_cast<int>(rng() % static_cast<unsigned>(length - least)));
            }
            // all that no row sees again, a part of it, or nothing
            const int now = book.at(id).length, end = now - window + 1 - static_cast<int>(rng() % 3 ? 0 : rng() % 50);
            const PageBook::Sequence& s = book.at(id);
            if (rng() % 5 && (s.gone_from == s.gone_to || end >= s.gone_from)) book.forget(id, sinks + (s.gone_from == s.gone_to && rng() % 4 == 0 ? 5 : 0), end);
            counts.push_back(rng() % 6 == 0 ? 0 : static_cast<int>(rng() % 3 ? rng() % 4 : rng() % 200));
        }
        std::vector<PassSeq> seqs;
        int row0 = 0, listed = 0;
        for (size_t i = 0; i < ids.size(); i++) {
            const PageBook::Sequence& s = book.at(ids[i]);
            const int hole = book.hole_of(s).pages();
            seqs.push_back({s.length + counts[i], s.length, row0, listed, hole});
            row0 += counts[i];
            listed += book.pages_for(s.length + counts[i]) - hole;
        }
        (void)book.extend(ids.data(), counts.data(), static_cast<int>(ids.size()));
        std::vector<int> table(static_cast<size_t>(listed), -7);
        int* to = table.data();
        for (size_t i = 0; i < ids.size(); i++) {
            CHECK(to == table.data() + seqs[i].table);
            to = book.write_list(book.at(ids[i]), to);
        }
        CHECK(to == table.data() + table.size());
        AttendCut cut{};
        cut.group = 1 + static_cast<int>(rng() % 4);
        cut.kv_heads = 2;
        cut.height = 16 << (rng() % 4);
        cut.causal = rng() % 3 != 0;
        cut.window = window;
        cut.sinks = sinks;
        cut.workgroups = 1 << (rng() % 9);
        cut.least = 128;
        cut.most = 64;
        const AttendPlan plan = plan_attend(seqs, counts, cut);
        for (const AttendItem& it : plan.items) {
            size_t i = 0;
            while (seqs[i].row0 != it.row0 || counts[i] == 0) i++;
            const PageBook::Sequence& s = book.at(ids[i]);
            // (a row that would see what is forgotten is refused: a stretch cut off and grown again may lie in the window)
            if (s.gone_from < s.gone_to && (s.gone_from < sinks || s.gone_to > std::max(0, seqs[i].first - window + 1))) continue;
            CHECK(it.map < 0);
            for (int v = it.k0; v < it.k1; v++) {
                const int position = lead > 0 && v >= lead ? v + it.gap : v, page = s.pages[static_cast<size_t>(position / T)];
                CHECK(page != PageBook::kNone && page_of(it, table, lead, T, v) == page);
            }
        }
    }
    return 0;
}

// A stream's pass takes what its rows see, however long it is, and forgetting visits what is new.
static int far(int positions) {
    const int T = 16, window = 1000, sinks = 4;
    PageBook book(1 << 15, T);
    const int id = book.add();
    const auto grow = [&](int n) { (void)book.extend(&id, &n, 1); };
    while (book.at(id).length < positions) {
        grow(400000);
        book.forget(id, sinks, book.at(id).length - window + 1);
        CHECK(book.pages() - book.pages_free() <= window / T + 3);
    }
    const auto start = std::chrono::steady_clock::now();
    std::vector<int> list(200, -7);
    for (int step = 0; step < 2000; step++) {
        book.forget(id, sinks, book.at(id).length - window + 1);
        grow(1);
        CHECK(book.write_list(book.at(id), list.data()) <= list.data() + window / T + 3);
    }
    // (visits to a hole of five million positions: 300 thousand pages a step, a second in all and more)
    CHECK(std::chrono::steady_clock::now() - start < std::chrono::milliseconds(200));
    return 0;
}

int main() {
    for (unsigned seed = 1; seed <= 200; seed++)
        if (passes(seed)) return 1;
    return far(5000000);
}
