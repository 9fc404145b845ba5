// What a call reads and writes in memory, so that one whose results lie over anything else of it is refused: its blocks read at different
// times, some of them when others have written.
#pragma once
#include <stdint.h>

#include <initializer_list>

#include "common.cuh"

struct LlbRange {
    const char* name;
    const void* at;          // (null: nothing)
    long long bytes;
    bool over(const LlbRange& b) const {
        const uintptr_t x = (uintptr_t)at, y = (uintptr_t)b.at;
        return at && b.at && bytes > 0 && b.bytes > 0 && x < y + (uintptr_t)b.bytes && y < x + (uintptr_t)bytes;
    }
};

// 0, or a refusal that names the first of the `written` ranges that overlaps another one or one of the `read` ones.
inline int llb_refuse_overlap(const char* what, std::initializer_list<LlbRange> written, std::initializer_list<LlbRange> read) {
    for (const LlbRange* w = written.begin(); w != written.end(); ++w) {
        for (const LlbRange* o = w + 1; o != written.end(); ++o)
            if (w->over(*o)) return llb_fail("%s: %s must not lie over %s", what, w->name, o->name);
        for (const LlbRange& r : read)
            if (w->over(r)) return llb_fail("%s: %s must not lie over %s", what, w->name, r.name);
    }
    return 0;
}
