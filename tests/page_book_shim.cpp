// The page books behind a C interface, for tests/test_page_book.py. Calls
// return the count of device steps, or -1 with the reason in book_error().
#include <cstring>
#include <memory>

#include "../trit_amd/csrc/page_book.h"

using trit::PageBook;
static std::string error;
template <class F>
static int run(F&& f) {
    try {
        return f();
    } catch (const std::exception& e) {
        error = e.what();
        return -1;
    }
}
template <class T>
static int give(const std::vector<T>& v, int* out) {
    if (!v.empty()) std::memcpy(out, v.data(), v.size() * sizeof(T));
    return (int)v.size();
}

extern "C" {
const char* book_error() { return error.c_str(); }
PageBook* book_new(int layers, int pages, int sequences) { return new PageBook(layers, pages, sequences); }
void book_free(PageBook* b) { delete b; }
int book_used(PageBook* b) { return b->pages_in_use(); }
int book_row(PageBook* b, int id) { return run([&] { return b->row(id); }); }
int book_length(PageBook* b, int id, int layer) { return run([&] { return b->length(id, layer); }); }
int book_open(PageBook* b, int n, int* out) { return run([&] { b->open(n, out); return 0; }); }
int book_close(PageBook* b, const int* ids, int n) { return run([&] { b->close(ids, n); return 0; }); }
int book_fork(PageBook* b, const int* ids, int n, int* out, int* copies) {
    return run([&] { return give(b->fork(ids, n, out), copies); });
}
int book_reorder(PageBook* b, const int* ids, const int* parents, int n, int* copies) {
    return run([&] { return give(b->reorder(ids, parents, n), copies); });
}
int book_append(PageBook* b, int layer, const int* ids, const int* counts, int n, int* entries) {
    return run([&] { return give(b->append(layer, ids, counts, n), entries); });
}
// counts: row copies, page moves, entries.
int book_copy(PageBook* b, const int* ids, int n, PageBook* into, int* out, int* rows, int* moves, int* entries,
              int* counts) {
    return run([&] {
        std::vector<PageBook::RowCopy> r;
        std::vector<PageBook::PageMove> m;
        std::vector<PageBook::Entry> e;
        b->copy(ids, n, *into, out, r, m, e);
        counts[0] = give(r, rows);
        counts[1] = give(m, moves);
        counts[2] = give(e, entries);
        return 0;
    });
}
int book_compact(PageBook* b, int* moves, int* entries, int* counts) {
    return run([&] {
        std::vector<PageBook::PageMove> m;
        std::vector<PageBook::Entry> e;
        b->compact(m, e);
        counts[0] = give(m, moves);
        counts[1] = give(e, entries);
        return b->pages_in_use();
    });
}
int book_resize(PageBook* b, int pages) { return run([&] { b->resize(pages); return 0; }); }
}
