// page_book.hpp -- what the host knows of the cache pages of several sequences:
// who holds which.  The tables on the device are written by rdl_kv_plan_dev and
// rdl_kv_fork_dev, which hand out the pages of the free list from its front, in the order of
// the sequences and of the pairs; the book does the same, so nothing is read back
// to know a table row, and no number from the device is an index here.
#pragma once

#include <stddef.h>

#include <memory>
#include <vector>

namespace rdl {

struct PageBook {
    size_t n_pages = 0;
    int page = 1;              // positions
    std::vector<int> len;      // of each sequence
    std::vector<int> free;     // pages that none holds
    std::vector<int> holders;  // of each page: the sequences whose rows name it
    std::unique_ptr<int[]> rows;  // [sequence][n_pages]: the pages of its positions

    // Sequences without positions, all pages free.  May throw (std::bad_alloc).
    void begin(size_t n_seq, size_t pages, int page_positions) {
        std::unique_ptr<int[]> r(new int[n_seq * pages]);
        len.assign(n_seq, 0);
        holders.assign(pages, 0);
        free.resize(pages);
        for (size_t p = 0; p < pages; p++) free[p] = (int)p;
        rows = std::move(r);
        n_pages = pages;
        page = page_positions;
    }
    size_t pages_of(size_t positions) const { return (positions + (size_t)page - 1) / (size_t)page; }
    int* row(size_t seq) const { return rows.get() + seq * n_pages; }
    // Pages that counts[b] more positions of each sequence take.
    size_t step_pages(const int* counts) const {
        size_t n = 0;
        for (size_t b = 0; b < len.size(); b++) n += pages_of((size_t)len[b] + (size_t)counts[b]) - pages_of((size_t)len[b]);
        return n;
    }
    // They do (there are as many pages, and no sequence passes n_pages).
    void step(const int* counts) {
        size_t taken = 0;
        for (size_t b = 0; b < len.size(); b++) {
            const size_t had = pages_of((size_t)len[b]), now = pages_of((size_t)len[b] + (size_t)counts[b]);
            for (size_t p = had; p < now; p++) holders[row(b)[p] = free[taken++]] = 1;
            len[b] += counts[b];
        }
        take(taken);
    }
    // Pages that copies of these sequences take: one for each last page that is not full.
    size_t fork_pages(const int* parents, size_t n) const {
        size_t pages = 0;
        for (size_t i = 0; i < n; i++) pages += len[parents[i]] % page != 0;
        return pages;
    }
    // The empty sequences `children`, which differ and are no parents, become copies.
    void fork(const int* parents, const int* children, size_t n) {
        size_t taken = 0;
        for (size_t i = 0; i < n; i++) {
            const int positions = len[children[i]] = len[parents[i]];
            const int *from = row(parents[i]);
            int* to = row(children[i]);
            const size_t full = (size_t)(positions / page);
            for (size_t p = 0; p < full; p++) holders[to[p] = from[p]]++;
            if (positions % page) holders[to[full] = free[taken++]] = 1;
        }
        take(taken);
    }
    void drop(size_t seq) {
        for (size_t p = 0; p < pages_of((size_t)len[seq]); p++) {
            const int held = row(seq)[p];
            if (--holders[held] == 0) free.push_back(held);  // within the capacity it began with
        }
        len[seq] = 0;
    }

private:
    void take(size_t n) { free.erase(free.begin(), free.begin() + (ptrdiff_t)n); }
};

}  // namespace rdl
