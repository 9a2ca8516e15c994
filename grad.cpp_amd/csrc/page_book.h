// Who holds which page of a paged cache: sequences as lists of pages, how often a page is held,
// which pages are free.  Host code alone, so that it can be tested without a GPU; the contents
// of pages are moved by whoever asks (every operation that wants contents moved says which).
//
// A page holds page_tokens positions of every layer, keys and values of all heads.  Sequences
// that were forked share pages; a page held more than once is never written: the position that
// would go into it goes into a copy (Copy, made by extend).  The lowest free page is handed out
// first, so that the pages in use stay near the front and the same calls give the same pages.
// A sequence can forget a stretch of its positions: the pages that lie wholly inside are nobody's
// any more (kNone in its list); the positions keep their numbers.
#pragma once

#include <algorithm>
#include <climits>
#include <functional>
#include <stdexcept>
#include <string>
#include <unordered_map>
#include <utility>
#include <vector>

namespace gh {

struct PageCopy {
    int from, to;  // pages
    int tokens;    // positions to copy, from the page's first on
};

class PageBook {
public:
    static constexpr int kNone = -1;

    struct Sequence {
        bool live = false;
        int length = 0;
        std::vector<int> pages;
        int gone_from = 0, gone_to = 0;  // positions that are forgotten
        bool forgot(int from, int to) const { return std::max(from, gone_from) < std::min(to, gone_to); }  // any of those
    };

    // The places of a sequence's list whose pages it has forgotten, but for the last one of a sequence cut off inside what was forgotten.
    struct Hole {
        int from, to;
        int pages() const { return to - from; }
    };
    Hole hole_of(const Sequence& s) const {
        const int from = pages_for(s.gone_from);
        return {from, std::max(from, s.gone_to / page_tokens_)};
    }
    // The list without its hole, which is as long as a stream is: what a pass takes along.  (A last page may be nobody's: it has no rows, nothing of it is read.)
    int* write_list(const Sequence& s, int* to) const {
        const Hole hole = hole_of(s);
        const int n = static_cast<int>(s.pages.size());
        for (int i = 0; i < hole.from && i < n; i++) *to++ = std::max(s.pages[static_cast<size_t>(i)], 0);
        for (int i = hole.to; i < n; i++) *to++ = std::max(s.pages[static_cast<size_t>(i)], 0);
        return to;
    }

    PageBook(int pages, int page_tokens) : page_tokens_(page_tokens), held_(static_cast<size_t>(pages), 0) {
        free_.reserve(held_.size());
        for (int p = 0; p < pages; p++) free_.push_back(p);  // ascending: a heap with the lowest on top
    }

    int pages() const { return static_cast<int>(held_.size()); }
    int pages_free() const { return static_cast<int>(free_.size()); }
    int sequences() const {
        return static_cast<int>(std::count_if(seqs_.begin(), seqs_.end(), [](const Sequence& s) { return s.live; }));
    }
    int held(int page) const { return held_[static_cast<size_t>(page)]; }

    const Sequence& at(int seq) const {
        if (seq < 0 || static_cast<size_t>(seq) >= seqs_.size() || !seqs_[static_cast<size_t>(seq)].live)
            throw std::out_of_range("cache: no sequence " + std::to_string(seq));
        return seqs_[static_cast<size_t>(seq)];
    }

    // A new, empty sequence: the lowest number that no sequence has.
    int add() {
        size_t i = lowest_;
        while (i < seqs_.size() && seqs_[i].live) i++;
        if (i == seqs_.size()) seqs_.emplace_back();
        lowest_ = i + 1;
        seqs_[i].live = true;
        seqs_[i].length = 0;
        seqs_[i].pages.clear();
        seqs_[i].gone_from = seqs_[i].gone_to = 0;
        return static_cast<int>(i);
    }

    // A sequence whose first `length` positions are seq's, in the same pages.
    int fork(int seq, int length) {
        const Sequence& from = at(seq);
        if (length < 0 || length > from.length)
            throw std::out_of_range("cache: a fork of " + std::to_string(length) + " positions of a sequence of "
                                    + std::to_string(from.length));
        std::vector<int> pages(from.pages.begin(), from.pages.begin() + pages_for(length));
        const int gone_from = from.gone_from, gone_to = from.gone_to;
        const int id = add();
        Sequence& s = seqs_[static_cast<size_t>(id)];
        s.pages = std::move(pages);
        s.length = length;
        s.gone_from = gone_from;
        s.gone_to = gone_to;
        cut_gone(s);
        for (int p : s.pages)
            if (p != kNone) held_[static_cast<size_t>(p)]++;
        return id;
    }

    void truncate(int seq, int length) {
        if (length < 0 || length > at(seq).length)
            throw std::out_of_range("cache: " + std::to_string(length) + " positions kept of a sequence of "
                                    + std::to_string(at(seq).length));
        Sequence& s = seqs_[static_cast<size_t>(seq)];
        while (static_cast<int>(s.pages.size()) > pages_for(length)) {
            if (s.pages.back() != kNone) release(s.pages.back());
            s.pages.pop_back();
        }
        s.length = length;
        cut_gone(s);
    }

    // Gives up positions [from, to); with those given up before they have to make one stretch.
    void forget(int seq, int from, int to) {
        (void)at(seq);
        Sequence& s = seqs_[static_cast<size_t>(seq)];
        if (from >= to) return;
        if (from < 0 || to > s.length)
            throw std::out_of_range("cache: positions " + std::to_string(from) + " to " + std::to_string(to) + " forgotten of a sequence of "
                                    + std::to_string(s.length));
        if (s.gone_from < s.gone_to && (from > s.gone_to || to < s.gone_from))
            throw std::invalid_argument("cache: sequence " + std::to_string(seq) + " has forgotten positions " + std::to_string(s.gone_from) + " to "
                                        + std::to_string(s.gone_to) + ": what else it forgets has to touch them");
        const bool any = s.gone_from < s.gone_to;
        const Hole before = hole_of(s);
        s.gone_from = any ? std::min(s.gone_from, from) : from;
        s.gone_to = any ? std::max(s.gone_to, to) : to;
        // (only pages with a position of this call can have become wholly forgotten, and those of the hole are: a stream's is as long as the stream)
        const int first = std::max(pages_for(s.gone_from), from / page_tokens_), end = std::min(s.gone_to / page_tokens_, pages_for(to));
        for (int i = first; i < end; i++) {
            if (i >= before.from && i < before.to) i = before.to;
            if (i >= end) break;
            int& p = s.pages[static_cast<size_t>(i)];
            if (p != kNone) release(p);
            p = kNone;
        }
    }

    void drop(int seq) {
        truncate(seq, 0);
        seqs_[static_cast<size_t>(seq)].live = false;
        lowest_ = std::min(lowest_, static_cast<size_t>(seq));
    }

    // counts[i] more positions for seqs[i]; the copies that have to be made before anything is
    // written.  Either all of it happens or, with an exception, nothing.
    std::vector<PageCopy> extend(const int* seqs, const int* counts, int n) {
        long long need = 0;
        std::unordered_map<int, int> leaving;  // holders of a shared last page that get one of their own
        std::vector<char> seen(seqs_.size(), 0);
        for (int i = 0; i < n; i++) {
            const Sequence& s = at(seqs[i]);
            if (seen[static_cast<size_t>(seqs[i])]++)
                throw std::invalid_argument("cache: sequence " + std::to_string(seqs[i]) + " is named twice in one pass");
            if (counts[i] < 0) throw std::invalid_argument("cache: negative number of positions");
            if (counts[i] == 0) continue;
            if (counts[i] > INT_MAX - page_tokens_ - s.length) throw std::out_of_range("cache: a sequence of more than 2^31 positions");
            need += pages_for(s.length + counts[i]) - pages_for(s.length);
            if (s.length % page_tokens_ != 0) {
                const int last = s.pages.back();
                if (last == kNone) {  // (cut off inside what was forgotten)
                    need++;
                } else if (held_[static_cast<size_t>(last)] - leaving[last] > 1) {
                    leaving[last]++;
                    need++;
                }
            }
        }
        check_free(need);
        std::vector<PageCopy> copies;
        copies.reserve(static_cast<size_t>(n));
        for (int i = 0; i < n; i++) {  // (memory for the page lists first: what follows does not throw)
            std::vector<int>& list = seqs_[static_cast<size_t>(seqs[i])].pages;
            const size_t want = static_cast<size_t>(pages_for(at(seqs[i]).length + counts[i]));
            if (want > list.capacity()) list.reserve(std::max(want, list.capacity() + list.capacity() / 2));
        }
        for (int i = 0; i < n; i++) {
            if (counts[i] == 0) continue;
            Sequence& s = seqs_[static_cast<size_t>(seqs[i])];
            const int used = s.length % page_tokens_;
            if (used != 0 && s.pages.back() == kNone) {
                s.pages.back() = take();
            } else if (used != 0 && held_[static_cast<size_t>(s.pages.back())] > 1) {
                const int from = s.pages.back();
                s.pages.back() = take();
                held_[static_cast<size_t>(from)]--;
                copies.push_back({from, s.pages.back(), used});
            }
            s.length += counts[i];
            while (static_cast<int>(s.pages.size()) < pages_for(s.length)) s.pages.push_back(take());
        }
        return copies;
    }

    // A sequence of `length` positions in pages of its own, contents to be written by the caller.
    int add_filled(int length) {
        const int id = add();
        try {
            (void)extend(&id, &length, 1);
        } catch (...) {
            drop(id);
            throw;
        }
        return id;
    }

    // A sequence like one of this or another book, in pages of its own, contents to be written by the caller.
    int add_like(const Sequence& other) {
        std::vector<int> pages = other.pages;
        const int length = other.length, gone_from = other.gone_from, gone_to = other.gone_to;
        check_free(static_cast<long long>(pages.size()) - std::count(pages.begin(), pages.end(), kNone));
        const int id = add();
        Sequence& s = seqs_[static_cast<size_t>(id)];
        for (int& p : pages)
            if (p != kNone) p = take();
        s.pages = std::move(pages);
        s.length = length;
        s.gone_from = gone_from;
        s.gone_to = gone_to;
        return id;
    }

    // Pages in use to the front of the pool, the last ones into the lowest free places.  No page
    // is both copied from and copied to.
    std::vector<PageCopy> compact() {
        const int used = pages() - pages_free();
        std::vector<int> to;
        for (int p = 0; p < used; p++)
            if (held_[static_cast<size_t>(p)] == 0) to.push_back(p);
        std::vector<PageCopy> moves;
        std::unordered_map<int, int> place;
        size_t next = 0;
        for (int p = used; p < pages(); p++)
            if (held_[static_cast<size_t>(p)] != 0) {
                moves.push_back({p, to[next], page_tokens_});
                place[p] = to[next++];
            }
        if (moves.empty()) return moves;
        for (PageCopy& m : moves) m.tokens = 0;
        std::vector<int> filled(held_.size(), 0);  // positions of a page that anybody holds
        for (const Sequence& s : seqs_)
            if (s.live)
                for (size_t i = 0; i < s.pages.size(); i++)
                    if (s.pages[i] != kNone) filled[static_cast<size_t>(s.pages[i])] =
                        std::max(filled[static_cast<size_t>(s.pages[i])], std::min(page_tokens_, s.length - static_cast<int>(i) * page_tokens_));
        for (PageCopy& m : moves) m.tokens = filled[static_cast<size_t>(m.from)];
        std::vector<int> rest;
        rest.reserve(held_.size());
        for (int p = used; p < pages(); p++) rest.push_back(p);
        // nothing throws from here on
        for (const PageCopy& m : moves) {
            held_[static_cast<size_t>(m.to)] = held_[static_cast<size_t>(m.from)];
            held_[static_cast<size_t>(m.from)] = 0;
        }
        for (Sequence& s : seqs_)
            for (int& p : s.pages)
                if (const auto it = place.find(p); it != place.end()) p = it->second;
        free_.swap(rest);
        return moves;
    }

    int pages_for(int length) const { return length / page_tokens_ + (length % page_tokens_ != 0); }
    int page_tokens() const { return page_tokens_; }

private:
    void check_free(long long need) const {
        if (need > pages_free())
            throw std::runtime_error("cache: out of pages (" + std::to_string(need) + " wanted, " + std::to_string(pages_free()) + " of "
                                     + std::to_string(pages()) + " free)");
    }
    static void cut_gone(Sequence& s) {
        s.gone_to = std::min(s.gone_to, s.length);
        if (s.gone_from >= s.gone_to) s.gone_from = s.gone_to = 0;
    }
    int take() {
        std::pop_heap(free_.begin(), free_.end(), std::greater<int>());
        const int p = free_.back();
        free_.pop_back();
        held_[static_cast<size_t>(p)] = 1;
        return p;
    }
    void release(int p) {
        if (--held_[static_cast<size_t>(p)] > 0) return;
        free_.push_back(p);  // (room was reserved: never more entries than pages)
        std::push_heap(free_.begin(), free_.end(), std::greater<int>());
    }

    int page_tokens_;
    std::vector<int> held_;  // by how many sequences
    std::vector<int> free_;  // a heap, the lowest on top
    std::vector<Sequence> seqs_;
    size_t lowest_ = 0;  // no sequence below this number is free
};

}  // namespace gh
