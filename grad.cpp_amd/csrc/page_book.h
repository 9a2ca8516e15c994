// Who holds which page of a paged cache: sequences as lists of pages, how often a page is held,
// which pages are free.  Host code alone, so that it can be tested without a GPU; the contents
// of pages are moved by whoever asks (every operation that wants contents moved says which).
//
// A page holds page_tokens positions of every layer, keys and values of all heads.  Sequences
// that were forked share pages; a page held more than once is never written: the position that
// would go into it goes into a copy (Copy, made by extend).  The lowest free page is handed out
// first, so that the pages in use stay near the front and the same calls give the same pages.
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
    struct Sequence {
        bool live = false;
        int length = 0;
        std::vector<int> pages;
    };

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
        return static_cast<int>(i);
    }

    // A sequence whose first `length` positions are seq's, in the same pages.
    int fork(int seq, int length) {
        const Sequence& from = at(seq);
        if (length < 0 || length > from.length)
            throw std::out_of_range("cache: a fork of " + std::to_string(length) + " positions of a sequence of "
                                    + std::to_string(from.length));
        std::vector<int> pages(from.pages.begin(), from.pages.begin() + pages_for(length));
        const int id = add();
        Sequence& s = seqs_[static_cast<size_t>(id)];
        s.pages = std::move(pages);
        s.length = length;
        for (int p : s.pages) held_[static_cast<size_t>(p)]++;
        return id;
    }

    void truncate(int seq, int length) {
        if (length < 0 || length > at(seq).length)
            throw std::out_of_range("cache: " + std::to_string(length) + " positions kept of a sequence of "
                                    + std::to_string(at(seq).length));
        Sequence& s = seqs_[static_cast<size_t>(seq)];
        while (static_cast<int>(s.pages.size()) > pages_for(length)) {
            release(s.pages.back());
            s.pages.pop_back();
        }
        s.length = length;
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
                if (held_[static_cast<size_t>(last)] - leaving[last] > 1) {
                    leaving[last]++;
                    need++;
                }
            }
        }
        if (need > pages_free())
            throw std::runtime_error("cache: out of pages (" + std::to_string(need) + " wanted, " + std::to_string(pages_free()) + " of "
                                     + std::to_string(pages()) + " free)");
        std::vector<PageCopy> copies;
        copies.reserve(static_cast<size_t>(n));
        for (int i = 0; i < n; i++) {  // (memory for the page lists first: what follows does not throw)
            const Sequence& s = at(seqs[i]);
            seqs_[static_cast<size_t>(seqs[i])].pages.reserve(static_cast<size_t>(pages_for(s.length + counts[i])));
        }
        for (int i = 0; i < n; i++) {
            if (counts[i] == 0) continue;
            Sequence& s = seqs_[static_cast<size_t>(seqs[i])];
            const int used = s.length % page_tokens_;
            if (used != 0 && held_[static_cast<size_t>(s.pages.back())] > 1) {
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
                    filled[static_cast<size_t>(s.pages[i])] =
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
