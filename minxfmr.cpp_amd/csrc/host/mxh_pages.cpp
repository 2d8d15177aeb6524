// mxh_pages.cpp — page bookkeeping (see mxh_pages.h).  Every operation that
// can fail does so before it changes anything: vectors have the room they may
// need from the start, so none but the constructor and the page lists allocate.
#include "mxh_pages.h"

#include <algorithm>

namespace mxh {

PageBook::PageBook(int n_pages, int page_rows, int max_seqs)
    : page_rows_(page_rows), refs_((size_t)n_pages, 0), seqs_((size_t)max_seqs) {
    free_.reserve((size_t)n_pages);
    for (int i = n_pages - 1; i >= 0; --i) free_.push_back(i);  // page 0 first
}

int PageBook::take() {
    const int page = free_.back();
    free_.pop_back();
    refs_[(size_t)page] = 1;
    return page;
}

void PageBook::give(int page) {
    if (--refs_[(size_t)page] == 0) free_.push_back(page);
}

void PageBook::cut(Seq& s, size_t pages) {
    while (s.pages.size() > pages) {
        give(s.pages.back());
        s.pages.pop_back();
    }
}

int PageBook::open() {
    for (size_t i = 0; i < seqs_.size(); ++i) {
        if (seqs_[i].open) continue;
        seqs_[i].open = true;
        return (int)i;
    }
    return -1;
}

int PageBook::fork(int seq) {
    const Seq& s = seqs_[(size_t)seq];
    const size_t held = ((size_t)s.length + (size_t)page_rows_ - 1) / (size_t)page_rows_;
    for (size_t i = 0; i < seqs_.size(); ++i) {
        Seq& c = seqs_[i];
        if (c.open) continue;
        std::vector<int> pages(s.pages.begin(), s.pages.begin() + (ptrdiff_t)held);  // (not what is only reserved)
        c.pages.swap(pages);
        c.open = true;
        c.length = c.reserved = s.length;
        for (int page : c.pages) ++refs_[(size_t)page];
        return (int)i;
    }
    return -1;
}

void PageBook::close(int seq) {
    Seq& s = seqs_[(size_t)seq];
    cut(s, 0);
    s = Seq{};
}

bool PageBook::extend(int seq, int rows, int* src, int* dst) {
    Seq& s = seqs_[(size_t)seq];
    const size_t pr = (size_t)page_rows_, held = s.pages.size(), end = (size_t)s.length + (size_t)rows;
    const size_t need = std::max(held, (end + pr - 1) / pr);
    // only the page of the row behind the last can be another sequence's too:
    // the pages behind it came from extend, and forks leave those out
    const size_t at = (size_t)s.length / pr;
    const bool copy = rows > 0 && at < held && (size_t)s.length % pr && refs_[(size_t)s.pages[at]] > 1;
    if (need - held + (copy ? 1 : 0) > free_.size()) return false;
    s.pages.reserve(need);
    *src = *dst = -1;
    if (copy) {
        *src = s.pages[at];
        *dst = take();
        give(*src);
        s.pages[at] = *dst;
    }
    while (s.pages.size() < need) s.pages.push_back(take());
    s.reserved = std::max(s.reserved, (int)end);
    return true;
}

int PageBook::common(const int* seqs, int n) const {
    if (n == 0) return 0;
    const std::vector<int>& a = pages(seqs[0]);
    size_t same = (size_t)length(seqs[0]) / (size_t)page_rows_;
    for (int i = 1; i < n; ++i) {
        const std::vector<int>& b = pages(seqs[i]);
        same = std::min(same, (size_t)length(seqs[i]) / (size_t)page_rows_);
        same = (size_t)(std::mismatch(a.begin(), a.begin() + (std::ptrdiff_t)same, b.begin()).first - a.begin());
    }
    return (int)same * page_rows_;
}

void PageBook::set_length(int seq, int rows) {
    Seq& s = seqs_[(size_t)seq];
    s.length = s.reserved = rows;
    cut(s, ((size_t)rows + (size_t)page_rows_ - 1) / (size_t)page_rows_);
}

}  // namespace mxh
