// What the C entry points check their arguments with.
#pragma once
#include <stddef.h>
#include <stdint.h>

namespace adder {

static bool overlaps(const void *a, size_t na, const void *b, size_t nb) {
    if (!a || !b) return false;
    const uintptr_t pa = reinterpret_cast<uintptr_t>(a), pb = reinterpret_cast<uintptr_t>(b);
    return pa < pb + nb && pb < pa + na;
}

struct Span { const void *p; size_t bytes; };

// no output may overlap an input or another output
template <int NO, int NI>
static bool any_alias(const Span (&outs)[NO], const Span (&ins)[NI]) {
    for (int o = 0; o < NO; ++o) {
        for (int i = 0; i < NI; ++i)
            if (overlaps(outs[o].p, outs[o].bytes, ins[i].p, ins[i].bytes)) return true;
        for (int q = o + 1; q < NO; ++q)
            if (overlaps(outs[o].p, outs[o].bytes, outs[q].p, outs[q].bytes)) return true;
    }
    return false;
}

}  // namespace adder
