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

// Every row of a pass gets every position that it may see from exactly one item (of its own or of a shared prefix), spans lie
// inside the sequences, places of parts are used once, and every join knows whom it waits for.
static int plans(unsigned seed) {
    std::mt19937 rng(seed), more(seed + 1000);
    for (int round = 0; round < 300; round++) {
        AttendCut cut{};
        cut.group = 1 + static_cast<int>(rng() % 5);
        cut.kv_heads = 1 + static_cast<int>(rng() % 8);
        cut.height = 16 << (rng() % 3);
        cut.causal = rng() % 4 != 0;
        cut.window = rng() % 3 ? 0 : 1 + static_cast<int>(rng() % 300);
        cut.workgroups = 1 << (rng() % 12);
        cut.least = 128;
        cut.most = 1 + static_cast<int>(rng() % 64);
        cut.square = more() % 2 ? 1 << (more() % 8) : 0;
        cut.resident = more() % 2 ? 16 << (more() % 6) : 0;
        const int T = 16;
        std::vector<PassSeq> seqs;
        std::vector<int> news;
        std::vector<std::vector<int>> pages;
        const int families = 1 + static_cast<int>(rng() % 3);
        int row0 = 0, table = 0;
        for (int i = static_cast<int>(rng() % 9); i >= 0; i--) {
            const int n = static_cast<int>(rng() % 3 ? rng() % 5 : rng() % 60), first = static_cast<int>(rng() % 1500);
            seqs.push_back({first + n, first, row0, table});
            news.push_back(n);
            std::vector<int> p;
            const int family = static_cast<int>(rng() % static_cast<unsigned>(families)), common = static_cast<int>(rng() % 80);
            for (int k = 0; k < (first + n + T - 1) / T; k++) p.push_back(k < common ? family * 1000 + k : 100000 + 1000 * static_cast<int>(seqs.size()) + k);
            pages.push_back(p);
            row0 += n;
            table += static_cast<int>(p.size());
        }
        std::vector<const std::vector<int>*> lists;
        std::vector<char> few;
        for (size_t i = 0; i < seqs.size(); i++) {
            lists.push_back(&pages[i]);
            few.push_back(news[i] > 0 && news[i] * cut.group <= cut.height);
        }
        const std::vector<SharedPrefix> shared = shared_prefixes(lists, seqs, few, T, 128);
        for (const SharedPrefix& s : shared) {
            CHECK(s.members.size() >= 2 && s.prefix >= 128 && s.prefix % T == 0);
            for (int m : s.members) {
                CHECK(few[static_cast<size_t>(m)] && s.prefix <= seqs[static_cast<size_t>(m)].first);
                for (int k = 0; k < s.prefix / T; k++) CHECK(pages[static_cast<size_t>(m)][static_cast<size_t>(k)] == pages[static_cast<size_t>(s.members[0])][static_cast<size_t>(k)]);
            }
        }
        const AttendPlan plan = plan_attend(seqs, news, cut, cut.window == 0 ? shared : std::vector<SharedPrefix>{});
        if (cut.resident > 0 && (cut.window != 0 || shared.empty())) {
            size_t tiles = 0;
            for (int n : news) tiles += static_cast<size_t>((n * cut.group + cut.height - 1) / cut.height);
            const size_t kv = static_cast<size_t>(cut.kv_heads), most = static_cast<size_t>(cut.resident);
            CHECK(plan.items.size() >= tiles && (tiles * kv > most || plan.items.size() * kv <= most));
        }
        // position by position: who brings (pass row, head of the group) what
        std::map<int, std::vector<int>> brought;
        std::map<int, std::vector<std::pair<int, int>>> from;  // ... and from which place and row of it (-1: whole)
        for (int row = 0; row < row0 * cut.group; row++) brought[row];
        std::set<int> places;
        for (const AttendItem& it : plan.items) {
            CHECK(it.rows >= 1 && it.rows <= cut.height && it.k0 < it.k1 && it.k0 >= 0 && it.k0 % 16 == 0);
            CHECK(it.joins <= 16 || cut.height > 16);
            CHECK((it.part < 0) == (it.joins == 0));
            if (it.part >= 0) CHECK(it.part < plan.parts && places.insert(it.part).second);
            size_t owner = 0;
            while (seqs[owner].table != it.table || pages[owner].empty()) owner++;
            CHECK(it.k1 <= static_cast<int>(pages[owner].size()) * T);
            for (int r = 0; r < it.rows; r++) {
                const int row = it.map >= 0 ? plan.maps[static_cast<size_t>(it.map + r)] : it.row0 * cut.group + it.r0 + r;
                CHECK(brought.count(row));
                for (int t = it.k0; t < it.k1; t++) brought[row].push_back(t);
                from[row].push_back({it.part, r});
            }
        }
        std::map<int, std::vector<std::pair<int, int>>> wanted;  // what the joins read
        std::map<int, int> arrivals;
        for (const AttendItem& it : plan.items)
            for (int j = 0; j < it.joins; j++) arrivals[it.join + j]++;
        for (size_t j = 0; j < plan.joins.size(); j++) {
            const AttendJoin& join = plan.joins[j];
            CHECK(arrivals[static_cast<int>(j)] == join.parts + join.shared_parts && join.parts >= 1);
            for (int r = 0; r < join.rows; r++) {
                const int row = join.row0 * cut.group + join.r0 + r;
                for (int k = 0; k < join.shared_parts; k++) wanted[row].push_back({join.shared_part + k, join.shared_row + r});
                for (int k = 0; k < join.parts; k++) wanted[row].push_back({join.part + k, r});
            }
        }
        CHECK(arrivals.size() == plan.joins.size());
        for (size_t i = 0; i < seqs.size(); i++)
            for (int r = 0; r < news[i] * cut.group; r++) {
                const int row = seqs[i].row0 * cut.group + r, pos = seqs[i].first + r / cut.group;
                std::vector<int>& got = brought[row];
                std::sort(got.begin(), got.end());
                CHECK(std::adjacent_find(got.begin(), got.end()) == got.end());
                const int low = cut.window ? std::max(0, pos - cut.window + 1) : 0, high = cut.causal ? pos + 1 : seqs[i].len;
                CHECK(!got.empty() && got.front() <= low && got.back() >= high - 1 && got.back() < seqs[i].len);
                CHECK(static_cast<int>(got.size()) == got.back() - got.front() + 1);
                auto& given = from[row];
                if (given.size() == 1 && given[0].first < 0) {
                    CHECK(!wanted.count(row));
                } else {
                    std::sort(given.begin(), given.end());
                    std::sort(wanted[row].begin(), wanted[row].end());
                    CHECK(given == wanted[row]);
                }
            }
    }
    return 0;
}

int main() {
    for (unsigned seed = 1; seed <= 20; seed++)
        if (run_book(seed) || plans(seed)) return 1;
    return refusals();
}
