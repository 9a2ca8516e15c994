// The page bookkeeping of a paged cache against a model that keeps every position's value, and the cutting of a pass into
// workgroups against its definition.  Exit status 0: all held.
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

template <class E, class F>
static bool throws(F f) {
    try {
        f();
    } catch (const E&) {
        return true;
    } catch (...) {
    }
    return false;
}

static int run_book(unsigned seed) {
    std::mt19937 rng(seed);
    const int T = 4, P = 24;
    PageBook book(P, T);
    std::vector<int> pool(P * T, -1);  // what a page's places hold
    std::map<int, std::vector<int>> want;
    int next_value = 0;
    const auto pick = [&] { return std::next(want.begin(), static_cast<long>(rng() % want.size()))->first; };
    const auto apply = [&](const std::vector<PageCopy>& copies) {
        const std::vector<int> before = pool;  // all at once, as the device does it
        std::set<int> to;
        for (const PageCopy& c : copies) {
            if (!to.insert(c.to).second) return false;
            for (int i = 0; i < c.tokens; i++) pool[c.to * T + i] = before[c.from * T + i];
        }
        for (const PageCopy& c : copies)
            if (to.count(c.from)) return false;
        return true;
    };
    for (int step = 0; step < 3000; step++) {
        const unsigned what = rng() % 12;
        if (want.empty() || what == 0) {
            const int s = book.add();
            CHECK(!want.count(s));
            want[s] = {};
        } else if (what == 1) {
            const int s = pick(), n = static_cast<int>(rng() % (want[s].size() + 1));
            const int f = book.fork(s, n);
            CHECK(!want.count(f));
            want[f].assign(want[s].begin(), want[s].begin() + n);
        } else if (what == 2) {
            const int s = pick();
            const int n = static_cast<int>(rng() % (want[s].size() + 1));
            book.truncate(s, n);
            want[s].resize(static_cast<size_t>(n));
        } else if (what == 3) {
            const int s = pick();
            book.drop(s);
            want.erase(s);
        } else if (what == 4) {
            const int used = book.pages() - book.pages_free();
            CHECK(apply(book.compact()));
            for (int p = 0; p < P; p++) CHECK((book.held(p) > 0) == (p < used));
        } else {
            std::vector<int> seqs, counts;
            for (const auto& [s, v] : want)
                if (rng() % 2) {
                    seqs.push_back(s);
                    counts.push_back(static_cast<int>(rng() % 6));
                }
            for (size_t i = seqs.size(); i > 1; i--) {
                const size_t j = rng() % i;
                std::swap(seqs[i - 1], seqs[j]);
                std::swap(counts[i - 1], counts[j]);
            }
            const int free = book.pages_free();
            std::vector<PageCopy> copies;
            try {
                copies = book.extend(seqs.data(), counts.data(), static_cast<int>(seqs.size()));
            } catch (const std::runtime_error&) {
                CHECK(book.pages_free() == free);
                for (const auto& [s, v] : want) CHECK(book.at(s).length == static_cast<int>(v.size()));
                continue;
            }
            CHECK(apply(copies));
            for (size_t i = 0; i < seqs.size(); i++) {
                const PageBook::Sequence& s = book.at(seqs[i]);
                for (int t = s.length - counts[i]; t < s.length; t++) {
                    const int page = s.pages[static_cast<size_t>(t / T)];
                    CHECK(book.held(page) == 1);  // nobody else sees what is written
                    pool[page * T + t % T] = next_value;
                    want[seqs[i]].push_back(next_value++);
                }
            }
        }
        CHECK(book.sequences() == static_cast<int>(want.size()));
        std::map<int, int> held;
        for (const auto& [s, v] : want) {
            const PageBook::Sequence& q = book.at(s);
            CHECK(q.length == static_cast<int>(v.size()));
            CHECK(static_cast<int>(q.pages.size()) == book.pages_for(q.length));
            for (int p : q.pages) held[p]++;
            for (int t = 0; t < q.length; t++) CHECK(pool[q.pages[static_cast<size_t>(t / T)] * T + t % T] == v[static_cast<size_t>(t)]);
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

static int refusals() {
    PageBook book(4, 16);
    CHECK(throws<std::out_of_range>([&] { book.at(0); }));
    CHECK(throws<std::out_of_range>([&] { book.drop(-1); }));
    const int a = book.add(), b = book.add();
    const int twice[] = {a, a}, both[] = {a, b}, one[] = {1, 1}, much[] = {33, 17}, less[] = {-1, 0}, all[] = {16, 48}, huge[] = {INT_MAX, 1};
    CHECK(throws<std::invalid_argument>([&] { book.extend(twice, one, 2); }));
    CHECK(throws<std::invalid_argument>([&] { book.extend(both, less, 2); }));
    CHECK(throws<std::runtime_error>([&] { book.extend(both, much, 2); }));
    CHECK(throws<std::out_of_range>([&] { book.extend(both, huge, 2); }));
    CHECK(book.pages_free() == 4);
    CHECK(book.extend(both, all, 2).empty() && book.pages_free() == 0);
    CHECK(throws<std::out_of_range>([&] { book.fork(a, 17); }));
    CHECK(throws<std::out_of_range>([&] { book.fork(a, -1); }));
    CHECK(throws<std::out_of_range>([&] { book.truncate(b, 49); }));
    CHECK(throws<std::runtime_error>([&] { book.add_filled(1); }));
    CHECK(book.sequences() == 2);
    const int c = book.fork(b, 40);
    CHECK(throws<std::runtime_error>([&] { book.extend(&c, one, 1); }));  // the page it would write into is shared, none is free
    CHECK(book.at(c).length == 40);
    book.drop(a);
    const std::vector<PageCopy> copies = book.extend(&c, one, 1);
    CHECK(copies.size() == 1 && copies[0].tokens == 8 && copies[0].to == 0);
    return 0;
}

// Every (row, position it sees) is in exactly one item of its tile, spans lie inside the sequences, parts are counted.
static int plans(unsigned seed) {
    std::mt19937 rng(seed);
    for (int round = 0; round < 400; round++) {
        const int group = 1 + static_cast<int>(rng() % 5), height = 16 << (rng() % 3), kv = 1 + static_cast<int>(rng() % 8);
        const bool causal = rng() % 4 != 0;
        const int window = rng() % 3 ? 0 : 1 + static_cast<int>(rng() % 300);
        const int workgroups = 1 << (rng() % 12), least = 128, most = 1 + static_cast<int>(rng() % 64);
        std::vector<PassSeq> seqs;
        std::vector<int> news;
        for (int i = static_cast<int>(rng() % 5); i >= 0; i--) {
            const int n = static_cast<int>(rng() % 60), first = static_cast<int>(rng() % 2000);
            seqs.push_back({first + n, first, 0, 0});
            news.push_back(n);
        }
        const AttendPlan plan = plan_attend(seqs, news, group, kv, height, causal, window, workgroups, least, most);
        std::map<std::pair<int, int>, std::vector<AttendItem>> tiles;
        for (const AttendItem& it : plan.items) tiles[{it.seq, it.r0}].push_back(it);
        size_t n_tiles = 0;
        std::set<int> places, counters;
        for (size_t i = 0; i < seqs.size(); i++) {
            for (int r0 = 0; r0 < news[i] * group; r0 += height) {
                n_tiles++;
                const auto found = tiles.find({static_cast<int>(i), r0});
                CHECK(found != tiles.end());
                std::vector<AttendItem>& t = found->second;
                std::sort(t.begin(), t.end(), [](const AttendItem& a, const AttendItem& b) { return a.k0 < b.k0; });
                const int rows = std::min(height, news[i] * group - r0);
                int low = INT_MAX, high = 0;
                for (int r = r0; r < r0 + rows; r++) {
                    const int pos = seqs[i].first + r / group;
                    low = std::min(low, window ? std::max(0, pos - window + 1) : 0);
                    high = std::max(high, causal ? pos + 1 : seqs[i].len);
                }
                CHECK(static_cast<int>(t.size()) <= most);
                CHECK(t[0].k0 <= low && t[0].k0 % 16 == 0 && t.back().k1 == high);
                for (size_t j = 0; j < t.size(); j++) {
                    CHECK(t[j].rows == rows && t[j].parts == static_cast<int>(t.size()) && t[j].index == static_cast<int>(j));
                    CHECK(t[j].k0 < t[j].k1 && (j == 0 || t[j].k0 == t[j - 1].k1));
                    CHECK((t.size() > 1) == (t[j].part >= 0));
                    if (t.size() > 1) CHECK(places.insert(t[j].part + t[j].index).second && t[j].part + t[j].index < plan.parts && t[j].tile < plan.tiles);
                }
                if (t.size() > 1) CHECK(counters.insert(t[0].tile).second);
            }
        }
        CHECK(tiles.size() == n_tiles);
        CHECK(static_cast<int>(places.size()) <= plan.parts && static_cast<int>(counters.size()) == plan.tiles);
    }
    return 0;
}

int main() {
    for (unsigned seed = 1; seed <= 20; seed++)
        if (run_book(seed) || plans(seed)) return 1;
    return refusals();
}
