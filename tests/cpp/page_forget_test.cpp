// Sequences that forget, against a model that keeps every position's value, and the cutting of a pass whose rows see sinks beside
// a window, against its definition.  Exit status 0: all held.
#include "../../grad.cpp_amd/csrc/cache_plan.h"
#include "../../grad.cpp_amd/csrc/page_book.h"

#include <cstdio>
#include <map>
#include <random>
#include <set>

using namespace gh;

#define CHECK(x)                                                      \
    do {                                                              \
        if (!(x)) {                                                   \
            std::printf("%s:%d: %s\n", __FILE__, __LINE__, #x);       \
            return 1;                                                 \
        }                                                             \
    } while (0)

constexpr int kGone = -2;

static int run_book(unsigned seed) {
    std::mt19937 rng(seed);
    const int T = 4, P = 24;
    PageBook book(P, T), other(12, T);
    std::vector<int> pool(P * T, -1);
    std::map<int, std::vector<int>> want;  // values, kGone for what is forgotten
    int next_value = 0;
    const auto pick = [&] { return std::next(want.begin(), static_cast<long>(rng() % want.size()))->first; };
    const auto apply = [&](const std::vector<PageCopy>& copies) {
        const std::vector<int> before = pool;
        for (const PageCopy& c : copies)
            for (int i = 0; i < c.tokens; i++) pool[c.to * T + i] = before[c.from * T + i];
    };
    for (int step = 0; step < 2000; step++) {
        const unsigned what = rng() % 14;
        if (want.empty() || what == 0) {
            const int s = book.add();
            CHECK(!want.count(s));
            want[s] = {};
        } else if (what == 1) {
            const int s = pick(), n = static_cast<int>(rng() % (want[s].size() + 1)), f = book.fork(s, n);
            want[f].assign(want[s].begin(), want[s].begin() + n);
        } else if (what == 2) {
            const int s = pick(), n = static_cast<int>(rng() % (want[s].size() + 1));
            book.truncate(s, n);
            want[s].resize(static_cast<size_t>(n));
        } else if (what == 3) {
            const int s = pick();
            book.drop(s);
            want.erase(s);
        } else if (what == 4) {
            const int used = book.pages() - book.pages_free();
            apply(book.compact());
            for (int p = 0; p < P; p++) CHECK((book.held(p) > 0) == (p < used));
        } else if (what == 5) {  // a copy in pages of its own
            const int s = pick(), free = book.pages_free();
            int id;
            try {
                id = book.add_like(book.at(s));
            } catch (const std::runtime_error&) {
                CHECK(book.pages_free() == free && book.sequences() == static_cast<int>(want.size()));
                continue;
            }
            want[id] = want[s];
            for (size_t i = 0; i < book.at(s).pages.size(); i++) {
                const int a = book.at(s).pages[i], b = book.at(id).pages[i];
                CHECK((a == PageBook::kNone) == (b == PageBook::kNone));
                if (a == PageBook::kNone) continue;
                CHECK(book.held(b) == 1);
                for (int k = 0; k < T; k++) pool[b * T + k] = pool[a * T + k];
            }
            const int room = other.pages_free();  // ... and in another book
            try {
                const int there = other.add_like(book.at(s));
                CHECK(other.at(there).length == book.at(s).length && other.at(there).gone_to == book.at(s).gone_to);
                other.drop(there);
            } catch (const std::runtime_error&) {
            }
            CHECK(other.pages_free() == room);
        } else if (what <= 8) {
            const int s = pick(), n = static_cast<int>(want[s].size());
            const int a = static_cast<int>(rng() % static_cast<unsigned>(n + 1)), b = static_cast<int>(rng() % static_cast<unsigned>(n + 3)) - 1;
            std::vector<int> after = want[s];
            for (int t = a; t < std::min(b, n); t++) after[static_cast<size_t>(t)] = kGone;
            int runs = 0;
            for (size_t t = 0; t < after.size(); t++) runs += after[t] == kGone && (t == 0 || after[t - 1] != kGone);
            const PageBook::Sequence was = book.at(s);
            try {
                book.forget(s, a, b);
                CHECK(a >= b || (b <= n && runs == 1));
                want[s] = after;
            } catch (const std::out_of_range&) {
                CHECK(a < b && b > n);
                CHECK(book.at(s).pages == was.pages && book.at(s).gone_from == was.gone_from && book.at(s).gone_to == was.gone_to);
            } catch (const std::invalid_argument&) {
                CHECK(a < b && b <= n && runs == 2);
                CHECK(book.at(s).pages == was.pages && book.at(s).gone_from == was.gone_from && book.at(s).gone_to == was.gone_to);
            }
        } else {
            std::vector<int> seqs, counts;
            for (const auto& [s, v] : want)
                if (rng() % 2) {
                    seqs.push_back(s);
                    counts.push_back(static_cast<int>(rng() % 7));
                }
            const int free = book.pages_free();
            std::vector<PageCopy> copies;
            try {
                copies = book.extend(seqs.data(), counts.data(), static_cast<int>(seqs.size()));
            } catch (const std::runtime_error&) {
                CHECK(book.pages_free() == free);
                continue;
            }
            apply(copies);
            for (size_t i = 0; i < seqs.size(); i++) {
                const PageBook::Sequence& s = book.at(seqs[i]);
                for (int t = s.length - counts[i]; t < s.length; t++) {
                    const int page = s.pages[static_cast<size_t>(t / T)];
                    CHECK(page != PageBook::kNone && book.held(page) == 1);
                    pool[page * T + t % T] = next_value;
                    want[seqs[i]].push_back(next_value++);
                }
            }
        }
        std::map<int, int> held;
        for (const auto& [s, v] : want) {
            const PageBook::Sequence& q = book.at(s);
            CHECK(q.length == static_cast<int>(v.size()) && static_cast<int>(q.pages.size()) == book.pages_for(q.length));
            for (int i = 0; i < static_cast<int>(q.pages.size()); i++) {
                const int p = q.pages[static_cast<size_t>(i)];
                bool all = true;  // a page is nobody's if and only if all it holds of the sequence is forgotten and it was full
                for (int t = i * T; t < std::min((i + 1) * T, q.length); t++) all = all && v[static_cast<size_t>(t)] == kGone;
                if (p == PageBook::kNone) CHECK(all);
                if (all && (i + 1) * T <= q.length) CHECK(p == PageBook::kNone);
                if (p != PageBook::kNone) held[p]++;
            }
            for (int t = 0; t < q.length; t++) {
                const int value = v[static_cast<size_t>(t)];
                CHECK(q.forgot(t, t + 1) == (value == kGone));
                if (value != kGone) CHECK(pool[q.pages[static_cast<size_t>(t / T)] * T + t % T] == value);
            }
        }
        int used = 0;
        for (int p = 0; p < P; p++) {
            CHECK(book.held(p) == (held.count(p) ? held[p] : 0));
            used += book.held(p) > 0;
        }
        CHECK(book.pages_free() == P - used);
    }
    return 0;
}

// Every row gets every position that it may see exactly once, from places inside the lists.
static int plans(unsigned seed) {
    std::mt19937 rng(seed);
    for (int round = 0; round < 30; round++) {
        AttendCut cut{};
        cut.group = 1 + static_cast<int>(rng() % 5);
        cut.kv_heads = 1 + static_cast<int>(rng() % 8);
        cut.height = 16 << (rng() % 4);
        cut.causal = rng() % 4 != 0;
        cut.window = 1 + static_cast<int>(rng() % 400);
        cut.sinks = rng() % 8 == 0 ? INT_MAX - 15 : 1 + static_cast<int>(rng() % (rng() % 2 ? 20 : 500));
        cut.workgroups = 1 << (rng() % 12);
        cut.least = 128;
        cut.most = 1 + static_cast<int>(rng() % 64);
        cut.square = rng() % 2 ? 1 << (rng() % 8) : 0;
        cut.resident = rng() % 2 ? 16 << (rng() % 6) : 0;
        std::vector<PassSeq> seqs;
        std::vector<int> news;
        int row0 = 0, table = 0;
        for (int i = static_cast<int>(rng() % 6); i >= 0; i--) {
            const int n = static_cast<int>(rng() % 3 ? rng() % 5 : rng() % 200), first = static_cast<int>(rng() % 3000);
            seqs.push_back({first + n, first, row0, table});
            news.push_back(n);
            row0 += n;
            table += (first + n + 15) / 16 + 1;
        }
        const AttendPlan plan = plan_attend(seqs, news, cut);
        const int lead = sinks_lead(cut.sinks);
        std::map<int, std::vector<int>> brought;
        for (const AttendItem& it : plan.items) {
            CHECK(it.rows >= 1 && it.rows <= cut.height && it.k0 < it.k1 && it.k0 >= 0 && it.k0 % 16 == 0 && it.gap % 16 == 0 && it.gap >= 0 && it.map < 0);
            const PassSeq* s = nullptr;
            for (const PassSeq& q : seqs)
                if (q.table == it.table) s = &q;
            CHECK(s && s->first == it.first);
            for (int r = 0; r < it.rows; r++)
                for (int v = it.k0; v < it.k1; v++) {
                    const int t = v >= lead ? v + it.gap : v;
                    CHECK(t < s->len);
                    brought[it.row0 * cut.group + it.r0 + r].push_back(t);
                }
        }
        for (size_t i = 0; i < seqs.size(); i++)
            for (int r = 0; r < news[i] * cut.group; r++) {
                const int pos = seqs[i].first + r / cut.group;
                std::vector<int>& got = brought[seqs[i].row0 * cut.group + r];
                std::sort(got.begin(), got.end());
                CHECK(std::adjacent_find(got.begin(), got.end()) == got.end());
                for (int t = 0; t < seqs[i].len; t++)
                    if ((!cut.causal || t <= pos) && (t > pos - cut.window || t < cut.sinks)) CHECK(std::binary_search(got.begin(), got.end(), t));
            }
    }
    return 0;
}

int main() {
    for (unsigned seed = 1; seed <= 20; seed++)
        if (run_book(seed) || plans(seed)) return 1;
    return 0;
}
