// The page table of a paged cache (host only): tables of all sequences, owners per page, free pages handed out lowest number first.
// Everything is sized at construction; the calls allocate nothing and throw nothing.
#pragma once
#include <algorithm>
#include <cstdint>
#include <functional>
#include <vector>

#include "../../include/kata_paged.h"

struct kata_pages {
    int32_t n_pages = 0, page_size = 0, n_seqs = 0, max_slots = 0, width = 0;   // width: table entries per sequence
    std::vector<int32_t> table, count, owners, free_heap;                       // table [n_seqs][width]; free_heap: a min-heap

    kata_pages(int32_t pages, int32_t size, int32_t seqs, int32_t slots)
        : n_pages(pages), page_size(size), n_seqs(seqs), max_slots(slots), width((slots + size - 1) / size), table((size_t)seqs * width, 0), count(seqs, 0), owners(pages, 0), free_heap(pages) {
        for (int32_t i = 0; i < pages; i++) free_heap[i] = i;   // ascending order is a min-heap
    }
    int32_t pages_for(int32_t slots) const { return (int32_t)(((int64_t)slots + page_size - 1) / page_size); }
    int64_t capacity(int32_t seq) const { return std::min<int64_t>((int64_t)count[seq] * page_size, max_slots); }
    int32_t* row(int32_t seq) { return table.data() + (size_t)seq * width; }
    const int32_t* row(int32_t seq) const { return table.data() + (size_t)seq * width; }
    int32_t take() {
        std::pop_heap(free_heap.begin(), free_heap.end(), std::greater<int32_t>());
        const int32_t p = free_heap.back(); free_heap.pop_back(); owners[p] = 1; return p;
    }
    void drop(int32_t page) {
        if (--owners[page] == 0) { free_heap.push_back(page); std::push_heap(free_heap.begin(), free_heap.end(), std::greater<int32_t>()); }   // capacity n_pages since construction
    }
    int reserve(int32_t seq, int32_t n_slots) {
        if (seq < 0 || seq >= n_seqs || n_slots < 0 || n_slots > max_slots) return KATA_ERR_RANGE;
        const int32_t want = pages_for(n_slots);
        if (want > count[seq] && (size_t)(want - count[seq]) > free_heap.size()) return KATA_ERR_NOMEM;
        while (count[seq] < want) { row(seq)[count[seq]] = take(); count[seq]++; }
        return KATA_OK;
    }
    int trim(int32_t seq, int32_t n_slots) {
        if (seq < 0 || seq >= n_seqs || n_slots < 0) return KATA_ERR_RANGE;
        const int32_t want = pages_for(n_slots);
        while (count[seq] > want) { count[seq]--; drop(row(seq)[count[seq]]); }
        return KATA_OK;
    }
    int fork(int32_t src, int32_t dst, int32_t n_slots, int32_t& from, int32_t& to, int32_t& slots) {
        from = to = -1; slots = 0;
        if (src < 0 || src >= n_seqs || dst < 0 || dst >= n_seqs || src == dst || n_slots < 0 || n_slots > capacity(src)) return KATA_ERR_RANGE;
        if (count[dst]) return KATA_ERR_MODE;
        const int32_t whole = n_slots / page_size, rest = n_slots % page_size;
        if (rest && free_heap.empty()) return KATA_ERR_NOMEM;
        for (int32_t i = 0; i < whole; i++) { row(dst)[i] = row(src)[i]; owners[row(src)[i]]++; }
        count[dst] = whole;
        if (rest) { from = row(src)[whole]; to = take(); slots = rest; row(dst)[count[dst]++] = to; }
        return KATA_OK;
    }
    bool shared(int32_t seq, int32_t slot0, int32_t n_slots) const {   // whether any page of these slots has another owner
        for (int32_t i = slot0 / page_size; i < count[seq] && (int64_t)i * page_size < (int64_t)slot0 + n_slots; i++) if (owners[row(seq)[i]] > 1) return true;
        return false;
    }
};
