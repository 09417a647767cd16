// pages.hip -- which pages of a cache belong to which sequence (host code only).
//
// A page is counted once for every sequence that holds it. A fork shares all of
// its parent's pages; whoever is about to write to a shared page gets a fresh
// one in its place (mx4_pages_write). Free pages are handed out from a stack.
#include <algorithm>
#include <new>
#include <unordered_map>
#include <vector>

#include "mx4.h"

namespace mx4 {
mx4_status report(mx4_status st, const char* message);  // runtime.hip: sets mx4_last_error
}

struct mx4_pages {
    struct Sequence {
        std::vector<uint32_t> table;
        uint32_t tokens = 0;
    };
    uint32_t page_tokens = 0, next = 0;
    std::vector<uint32_t> holders;  // of each page
    std::vector<uint32_t> free;
    std::unordered_map<uint32_t, Sequence> sequences;
};

namespace {

using mx4::report;

// Nothing a C caller cannot see leaves an entry point: running out of host
// memory is a status.
template <class F>
mx4_status guarded(F&& f) {
    try {
        return f();
    } catch (const std::bad_alloc&) {
        return report(MX4_ERR_NO_MEMORY, "out of host memory");
    } catch (...) {
        return report(MX4_ERR_ARGUMENT, "unexpected failure of the page bookkeeping");
    }
}

mx4_pages::Sequence* find(const mx4_pages* p, uint32_t seq) {
    auto it = const_cast<mx4_pages*>(p)->sequences.find(seq);
    return it == const_cast<mx4_pages*>(p)->sequences.end() ? nullptr : &it->second;
}

// (`free` has room for every page, so this never allocates.)
void drop(mx4_pages* p, uint32_t page) {
    if (--p->holders[page] == 0) p->free.push_back(page);
}

}  // namespace

extern "C" {

mx4_status mx4_pages_create(uint32_t pages, uint32_t page_tokens, mx4_pages** out) {
    if (!out) return report(MX4_ERR_ARGUMENT, "null output pointer");
    *out = nullptr;
    if (pages == 0) return report(MX4_ERR_SHAPE, "a cache has at least one page");
    if (page_tokens < 16 || page_tokens > 4096 || (page_tokens & (page_tokens - 1)) != 0)
        return report(MX4_ERR_SHAPE, "page_tokens must be a power of two from 16 to 4096");
    return guarded([&] {
        mx4_pages* p = new mx4_pages;
        try {
            p->page_tokens = page_tokens;
            p->holders.assign(pages, 0);
            p->free.resize(pages);
        } catch (...) {
            delete p;
            throw;
        }
        for (uint32_t i = 0; i < pages; ++i) p->free[i] = pages - 1 - i;  // page 0 on top
        *out = p;
        return MX4_OK;
    });
}

void mx4_pages_destroy(mx4_pages* pages) { delete pages; }

mx4_status mx4_pages_free_count(const mx4_pages* p, uint32_t* out) {
    if (!p || !out) return report(MX4_ERR_ARGUMENT, "null argument");
    *out = (uint32_t)p->free.size();
    return MX4_OK;
}

mx4_status mx4_pages_open(mx4_pages* p, uint32_t* seq) {
    if (!p || !seq) return report(MX4_ERR_ARGUMENT, "null argument");
    return guarded([&] {
        while (p->sequences.count(p->next)) ++p->next;
        p->sequences.emplace(p->next, mx4_pages::Sequence());
        *seq = p->next++;
        return MX4_OK;
    });
}

mx4_status mx4_pages_fork(mx4_pages* p, uint32_t seq, uint32_t* child) {
    if (!p || !child) return report(MX4_ERR_ARGUMENT, "null argument");
    if (!find(p, seq)) return report(MX4_ERR_ARGUMENT, "no such sequence");
    return guarded([&] {
        mx4_pages::Sequence copy = *find(p, seq);
        while (p->sequences.count(p->next)) ++p->next;
        mx4_pages::Sequence& made = p->sequences[p->next];
        made = std::move(copy);
        for (uint32_t page : made.table) ++p->holders[page];
        *child = p->next++;
        return MX4_OK;
    });
}

mx4_status mx4_pages_write(mx4_pages* p, uint32_t seq, uint32_t from, uint32_t to, uint32_t pair[2], uint32_t* copies) {
    if (!p || !pair || !copies) return report(MX4_ERR_ARGUMENT, "null argument");
    *copies = 0;
    mx4_pages::Sequence* s = find(p, seq);
    if (!s) return report(MX4_ERR_ARGUMENT, "no such sequence");
    if (from > to || from > s->tokens) return report(MX4_ERR_ARGUMENT, "the positions do not follow the sequence's tokens");
    if (from == to) return mx4_pages_trim(p, seq, to);
    const uint32_t first = from / p->page_tokens, end = (to - 1) / p->page_tokens + 1, have = (uint32_t)s->table.size();
    uint64_t need = end > have ? end - have : 0;
    for (uint32_t i = first; i < std::min(end, have); ++i) need += p->holders[s->table[i]] > 1;
    // (the pages behind `end` go back only once the call is sure to succeed)
    if (need > p->free.size()) return report(MX4_ERR_NO_MEMORY, "too few free pages");
    return guarded([&] {
        s->table.reserve(std::max(end, have));  // nothing below allocates
        auto take = [&] {
            const uint32_t page = p->free.back();
            p->free.pop_back();
            p->holders[page] = 1;
            return page;
        };
        for (uint32_t i = first; i < end; ++i) {
            if (i >= s->table.size()) {
                s->table.push_back(take());
            } else if (p->holders[s->table[i]] > 1) {
                const uint32_t old = s->table[i];
                s->table[i] = take();
                drop(p, old);
                if (i * (uint64_t)p->page_tokens < from) {
                    pair[0] = old;
                    pair[1] = s->table[i];
                    *copies = 1;
                }
            }
        }
        while (s->table.size() > end) {
            drop(p, s->table.back());
            s->table.pop_back();
        }
        s->tokens = to;
        return MX4_OK;
    });
}

mx4_status mx4_pages_trim(mx4_pages* p, uint32_t seq, uint32_t tokens) {
    if (!p) return report(MX4_ERR_ARGUMENT, "null argument");
    mx4_pages::Sequence* s = find(p, seq);
    if (!s) return report(MX4_ERR_ARGUMENT, "no such sequence");
    if (tokens > s->tokens) return report(MX4_ERR_ARGUMENT, "the sequence has fewer tokens");
    const uint32_t keep = (uint32_t)(((uint64_t)tokens + p->page_tokens - 1) / p->page_tokens);
    while (s->table.size() > keep) {
        drop(p, s->table.back());
        s->table.pop_back();
    }
    s->tokens = tokens;
    return MX4_OK;
}

mx4_status mx4_pages_close(mx4_pages* p, uint32_t seq) {
    if (!p) return report(MX4_ERR_ARGUMENT, "null argument");
    mx4_pages::Sequence* s = find(p, seq);
    if (!s) return report(MX4_ERR_ARGUMENT, "no such sequence");
    for (uint32_t page : s->table) drop(p, page);
    p->sequences.erase(seq);
    return MX4_OK;
}

mx4_status mx4_pages_table(const mx4_pages* p, uint32_t seq, uint32_t* tokens, uint32_t* table, uint32_t capacity,
                           uint32_t* count) {
    if (!p || !count) return report(MX4_ERR_ARGUMENT, "null argument");
    const mx4_pages::Sequence* s = find(p, seq);
    if (!s) return report(MX4_ERR_ARGUMENT, "no such sequence");
    *count = (uint32_t)s->table.size();
    if (tokens) *tokens = s->tokens;
    if (!table) return MX4_OK;
    if (*count > capacity) return report(MX4_ERR_LENGTH, "the sequence has more pages than the table holds");
    std::copy(s->table.begin(), s->table.end(), table);
    return MX4_OK;
}

mx4_status mx4_pages_compact(mx4_pages* p, uint32_t* pairs, uint32_t capacity, uint32_t* count) {
    if (!p || !count || (!pairs && capacity)) return report(MX4_ERR_ARGUMENT, "null argument");
    return guarded([&] {
        const uint32_t pages = (uint32_t)p->holders.size(), live = pages - (uint32_t)p->free.size();
        std::vector<uint32_t> to(pages);
        std::vector<uint32_t> moved;
        uint32_t gap = 0;
        for (uint32_t i = 0; i < pages; ++i) {
            to[i] = i;
            if (i < live || !p->holders[i]) continue;
            while (p->holders[gap]) ++gap;  // there is one: live pages past `live` leave as many gaps before it
            to[i] = gap++;
            moved.push_back(i);
        }
        *count = (uint32_t)moved.size();
        if (moved.size() > capacity) return report(MX4_ERR_LENGTH, "more pages move than the list holds");
        for (uint32_t k = 0; k < moved.size(); ++k) {
            const uint32_t i = moved[k];
            pairs[2 * k] = i;
            pairs[2 * k + 1] = to[i];
            p->holders[to[i]] = p->holders[i];
            p->holders[i] = 0;
        }
        for (auto& s : p->sequences)
            for (uint32_t& page : s.second.table) page = to[page];
        for (uint32_t i = 0; i < p->free.size(); ++i) p->free[i] = pages - 1 - i;
        return MX4_OK;
    });
}

}  // extern "C"
