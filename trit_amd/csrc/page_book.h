// The host's side of a paged key/value cache: which sequence holds which
// pages, how many hold each, and what the device has to move when sequences
// are forked, reordered, copied or compacted. No device code: a call here
// only changes these books and says what to launch; a call that fails
// changes nothing.
#pragma once

#include <algorithm>
#include <functional>
#include <queue>
#include <stdexcept>
#include <string>
#include <unordered_map>
#include <utility>
#include <vector>

namespace trit {

class PageBook {
  public:
    static constexpr int BLOCK = 64;  // tokens of a block (a page holds a full one of every head and layer)

    // A sequence's open block and row of the page table, taken over by another: row `src` to row `dst`.
    struct RowCopy {
        int src, dst;
        int len;     // tokens of the sequence
        int blocks;  // entries of its page-table row
    };
    struct PageMove {
        int src, dst;
    };
    // An entry of the device's page table.
    struct Entry {
        int row, block, page;
    };

    PageBook(int layers, int pages, int sequences)
        : layers_(layers), refs_((size_t)pages, 0), seqs_((size_t)sequences) {
        for (int i = sequences - 1; i >= 0; --i) {
            free_ids_.push_back(i);
            free_rows_.push_back(i);
        }
        refill_free_pages();
    }

    int layers() const { return layers_; }
    int pages() const { return (int)refs_.size(); }
    int pages_in_use() const { return pages() - (int)free_pages_.size(); }
    int sequences() const { return (int)seqs_.size(); }
    int row(int id) const { return seq(id).row; }
    int length(int id, int layer) const {
        if (layer < 0 || layer >= layers_) refuse("layer " + std::to_string(layer) + " of " + std::to_string(layers_));
        return seq(id).len[(size_t)layer];
    }

    void open(int n, int* out) {
        need_ids(n);
        for (int i = 0; i < n; ++i) {
            const int id = take_id();
            seqs_[(size_t)id].len.assign((size_t)layers_, 0);
            out[i] = id;
        }
    }

    // New sequences with what `ids` hold: full blocks shared, the open ones copied.
    std::vector<RowCopy> fork(const int* ids, int n, int* out) {
        for (int i = 0; i < n; ++i) even(ids[i]);
        need_ids(n);
        // The ids come first: `out` may be the caller's array of ids.
        const std::vector<int> from(ids, ids + n);
        std::vector<RowCopy> copies;
        for (int i = 0; i < n; ++i) {
            const int id = take_id();
            Seq &to = seqs_[(size_t)id], &of = seqs_[(size_t)from[(size_t)i]];
            to.len = of.len;
            to.pages = of.pages;
            for (int p : to.pages) ++refs_[(size_t)p];
            copies.push_back({of.row, to.row, to.len[0], (int)to.pages.size()});
            out[i] = id;
        }
        return copies;
    }

    // Sequence ids[i] goes on with what parents[i] held before the call. A
    // parent's row goes to one of its children; only the others are copied.
    std::vector<RowCopy> reorder(const int* ids, const int* parents, int n) {
        if (n < 0) refuse("a negative number of sequences");
        std::vector<int> at((size_t)sequences(), -1);  // id -> its place in the call
        for (int i = 0; i < n; ++i) {
            even(ids[i]);
            even(parents[i]);
            if (at[(size_t)ids[i]] >= 0) refuse("sequence " + std::to_string(ids[i]) + " is named twice");
            at[(size_t)ids[i]] = i;
        }
        // heir[p]: the child that takes over the row of parent p (itself where it stays).
        std::vector<int> heir((size_t)sequences(), -1);
        for (int i = 0; i < n; ++i) {
            const int p = parents[i];
            if (at[(size_t)p] < 0) continue;  // a parent that is not reordered keeps its row
            if (heir[(size_t)p] < 0 || p == ids[i]) heir[(size_t)p] = ids[i];
        }
        std::vector<Seq> before;
        for (int i = 0; i < n; ++i) before.push_back(seqs_[(size_t)ids[i]]);
        std::vector<int> spare;  // rows of sequences that nobody goes on with
        for (int i = 0; i < n; ++i)
            if (heir[(size_t)ids[i]] < 0) spare.push_back(before[(size_t)i].row);
        std::vector<Seq> after;
        std::vector<RowCopy> copies;
        for (int i = 0; i < n; ++i) {
            const int p = parents[i];
            Seq s = seqs_[(size_t)p];
            if (at[(size_t)p] < 0 || heir[(size_t)p] != ids[i]) {
                const int src = s.row;
                s.row = spare.back();
                spare.pop_back();
                copies.push_back({src, s.row, s.len[0], (int)s.pages.size()});
            }
            for (int page : s.pages) ++refs_[(size_t)page];
            after.push_back(std::move(s));
        }
        for (const Seq& s : before) drop_pages(s.pages);
        for (int i = 0; i < n; ++i) seqs_[(size_t)ids[i]] = std::move(after[(size_t)i]);
        return copies;
    }

    // New sequences in `into` (which may be this book) that share no page with
    // the ones of `ids`; pages that several of `ids` share are copied once.
    void copy(const int* ids, int n, PageBook& into, int* out, std::vector<RowCopy>& rows,
              std::vector<PageMove>& pages, std::vector<Entry>& entries) {
        for (int i = 0; i < n; ++i) even(ids[i]);
        into.need_ids(n);
        // The copy of each page, and whether a sequence holds it yet (take_page counts the first).
        std::unordered_map<int, std::pair<int, bool>> to;
        std::vector<int> fresh;
        for (int i = 0; i < n; ++i)
            for (int p : seqs_[(size_t)ids[i]].pages)
                if (to.emplace(p, std::make_pair(-1, false)).second) fresh.push_back(p);
        into.need_pages((long long)fresh.size());
        const std::vector<int> from(ids, ids + n);
        for (int p : fresh) {
            to[p].first = into.take_page();
            pages.push_back({p, to[p].first});
        }
        for (int i = 0; i < n; ++i) {
            const int id = into.take_id();
            Seq& d = into.seqs_[(size_t)id];
            const Seq& s = seqs_[(size_t)from[(size_t)i]];
            d.len = s.len;
            for (size_t b = 0; b < s.pages.size(); ++b) {
                auto& [p, held] = to[s.pages[b]];
                if (held) ++into.refs_[(size_t)p];
                held = true;
                d.pages.push_back(p);
                entries.push_back({d.row, (int)b, p});
            }
            rows.push_back({s.row, d.row, d.len[0], 0});
            out[i] = id;
        }
    }

    void close(const int* ids, int n) {
        std::vector<char> named((size_t)sequences(), 0);
        for (int i = 0; i < n; ++i) {
            seq(ids[i]);
            if (named[(size_t)ids[i]]++) refuse("sequence " + std::to_string(ids[i]) + " is named twice");
        }
        for (int i = 0; i < n; ++i) {
            Seq& s = seqs_[(size_t)ids[i]];
            drop_pages(s.pages);
            free_rows_.push_back(s.row);
            free_ids_.push_back(ids[i]);
            s = Seq();
        }
    }

    // counts[i] more tokens of layer `layer` in sequence ids[i]: the table's new entries.
    std::vector<Entry> append(int layer, const int* ids, const int* counts, int n) {
        std::vector<char> named((size_t)sequences(), 0);
        long long fresh = 0;
        for (int i = 0; i < n; ++i) {
            const int len = length(ids[i], layer);
            if (named[(size_t)ids[i]]++) refuse("sequence " + std::to_string(ids[i]) + " is named twice");
            if (counts[i] < 0) refuse("a negative number of rows");
            if (counts[i] > MOST - len) refuse("a sequence holds at most " + std::to_string(MOST) + " tokens");
            fresh += std::max(0, (len + counts[i]) / BLOCK - (int)seqs_[(size_t)ids[i]].pages.size());
        }
        need_pages(fresh);
        std::vector<Entry> entries;
        for (int i = 0; i < n; ++i) {
            Seq& s = seqs_[(size_t)ids[i]];
            s.len[(size_t)layer] += counts[i];
            while ((int)s.pages.size() < s.len[(size_t)layer] / BLOCK) {
                s.pages.push_back(take_page());
                entries.push_back({s.row, (int)s.pages.size() - 1, s.pages.back()});
            }
        }
        return entries;
    }

    // Used pages to the front: what moves, and the table's entries that change.
    void compact(std::vector<PageMove>& moves, std::vector<Entry>& entries) {
        const int used = pages_in_use();
        std::vector<int> to((size_t)pages(), -1);
        int low = 0;
        for (int p = used; p < pages(); ++p) {
            if (!refs_[(size_t)p]) continue;
            while (refs_[(size_t)low]) ++low;
            to[(size_t)p] = low;
            moves.push_back({p, low});
            refs_[(size_t)low] = refs_[(size_t)p];
            refs_[(size_t)p] = 0;
        }
        if (moves.empty()) return;
        for (Seq& s : seqs_) {
            if (s.row < 0) continue;
            for (size_t b = 0; b < s.pages.size(); ++b) {
                const int p = to[(size_t)s.pages[b]];
                if (p < 0) continue;
                s.pages[b] = p;
                entries.push_back({s.row, (int)b, p});
            }
        }
        refill_free_pages();
    }

    // The pool's size, after compact().
    void resize(int pages) {
        refs_.resize((size_t)pages, 0);
        refill_free_pages();
    }

    // The entries of every sequence's row.
    std::vector<Entry> entries() const {
        std::vector<Entry> all;
        for (const Seq& s : seqs_)
            for (size_t b = 0; b < s.pages.size(); ++b) all.push_back({s.row, (int)b, s.pages[b]});
        return all;
    }

  private:
    static constexpr int MOST = 1 << 30;
    struct Seq {
        int row = -1;           // its open block and row of the page table; -1: no such sequence
        std::vector<int> len;   // tokens, layer by layer
        std::vector<int> pages;  // of its full blocks (as many as the layer with the most has)
    };

    [[noreturn]] static void refuse(const std::string& what) { throw std::runtime_error("paged cache: " + what); }

    const Seq& seq(int id) const {
        if (id < 0 || id >= sequences() || seqs_[(size_t)id].row < 0)
            refuse("there is no sequence " + std::to_string(id));
        return seqs_[(size_t)id];
    }
    // A sequence between steps: every layer holds the same tokens.
    void even(int id) const {
        const Seq& s = seq(id);
        for (int len : s.len)
            if (len != s.len[0])
                refuse("sequence " + std::to_string(id) + " holds different lengths in its layers");
    }
    void need_ids(int n) const {
        if (n < 0) refuse("a negative number of sequences");
        if (n > (int)free_ids_.size())
            refuse(std::to_string(n) + " more sequences where " + std::to_string(free_ids_.size()) + " of " +
                   std::to_string(sequences()) + " are free");
    }
    void need_pages(long long n) const {
        if (n > (long long)free_pages_.size())
            refuse(std::to_string(n) + " more pages where " + std::to_string(free_pages_.size()) + " of " +
                   std::to_string(pages()) + " are free");
    }
    int take_id() {
        const int id = free_ids_.back();
        free_ids_.pop_back();
        seqs_[(size_t)id].row = free_rows_.back();
        free_rows_.pop_back();
        return id;
    }
    int take_page() {
        const int p = free_pages_.top();
        free_pages_.pop();
        refs_[(size_t)p] = 1;
        return p;
    }
    void drop_pages(const std::vector<int>& pages) {
        for (int p : pages)
            if (!--refs_[(size_t)p]) free_pages_.push(p);
    }
    void refill_free_pages() {
        free_pages_ = {};
        for (int p = 0; p < pages(); ++p)
            if (!refs_[(size_t)p]) free_pages_.push(p);
    }

    int layers_;
    std::vector<int> refs_;  // sequences that hold each page
    std::vector<Seq> seqs_;  // by id
    std::vector<int> free_ids_, free_rows_;
    // The lowest free page first, so that a pool stays dense.
    std::priority_queue<int, std::vector<int>, std::greater<int>> free_pages_;
};

}  // namespace trit
