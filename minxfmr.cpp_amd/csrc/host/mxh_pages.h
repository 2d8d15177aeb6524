// mxh_pages.h — which pages of a K/V pool are whose: sequences as lists of
// pages with reference counts, forks that share them, copies on write.
// Host-only C++17.  The reference has one sequence per context, whose cache it
// resets (src/cache/kv_cache.cpp:77-83); there is nothing to share there.
#pragma once

#include <stddef.h>

#include <vector>

namespace mxh {

class PageBook {
public:
    PageBook(int n_pages, int page_rows, int max_seqs);

    bool valid(int seq) const { return seq >= 0 && seq < (int)seqs_.size() && seqs_[(size_t)seq].open; }
    int page_rows() const { return page_rows_; }
    int free_pages() const { return (int)free_.size(); }
    int length(int seq) const { return seqs_[(size_t)seq].length; }
    int reserved(int seq) const { return seqs_[(size_t)seq].reserved; }
    const std::vector<int>& pages(int seq) const { return seqs_[(size_t)seq].pages; }

    // a new sequence's id, -1 when all are open
    int open();
    // the id of a sequence with the same rows in the same pages, -1 as above
    int fork(int seq);
    void close(int seq);
    // false (and nothing changed) when there are too few free pages; *src = -1
    // without a copy
    bool extend(int seq, int rows, int* src, int* dst);
    // rows at most max(length, reserved)
    void set_length(int seq, int rows);

private:
    struct Seq {
        bool open = false;
        int length = 0, reserved = 0;
        std::vector<int> pages;
    };
    int take();
    void give(int page);
    void cut(Seq& s, size_t pages);

    int page_rows_;
    std::vector<int> refs_, free_;
    std::vector<Seq> seqs_;
};

}  // namespace mxh
