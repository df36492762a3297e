// Where a call's tensors lie, so that one whose output lies over an input is refused before its launch.
#pragma once

#include <algorithm>
#include <initializer_list>

#include "common.h"

namespace ts {

// [rows][heads] pieces of `bytes`, a row `row` bytes from the next and a head `head`. NULL: nowhere.
struct Lies {
    const char *name;
    const void *at;
    uint64_t bytes, rows = 1, row = 0, heads = 1, head = 0;
};

// Pieces as repeats within repeats: the farther of rows and heads first.
struct Repeats {
    uint64_t count[2], step[2], span[3];  // span: of all, of one of the first repeats, of a piece

    explicit Repeats(const Lies &x) {
        const bool rows_first = x.heads <= 1 || (x.rows > 1 && x.row >= x.head);
        count[0] = rows_first ? x.rows : x.heads, step[0] = rows_first ? x.row : x.head;
        count[1] = rows_first ? x.heads : x.rows, step[1] = rows_first ? x.head : x.row;
        const bool some = x.at && x.bytes && x.rows && x.heads;
        span[2] = some ? x.bytes : 0;
        for (int i = 1; i >= 0; i--) span[i] = some ? span[i + 1] + (count[i] - 1) * step[i] : 0;
    }
};

// Whether a and b, whose first is `gap` bytes behind a's, have a byte in common. Repeats at one distance are compared one by
// one (parts of the same wider rows or heads), others as the whole that they span.
inline bool meet(const Repeats &a, const Repeats &b, int64_t gap, int of = 0) {
    const int64_t sa = (int64_t)a.span[of], sb = (int64_t)b.span[of];
    if (gap >= sa || -gap >= sb) return false;
    if (of == 2) return true;
    const int64_t na = (int64_t)a.count[of], nb = (int64_t)b.count[of], step = (int64_t)(na > 1 ? a.step[of] : b.step[of]);
    if (na <= 1 && nb <= 1) return meet(a, b, gap, of + 1);
    if (step <= 0 || (na > 1 && nb > 1 && a.step[of] != b.step[of])) return true;
    // Those of b's repeats that are `by` behind one of a's lie within its span only for some `by`.
    const int64_t least = std::max(1 - na, -((gap + (int64_t)b.span[of + 1]) / step) - 1);
    const int64_t most = std::min(nb - 1, ((int64_t)a.span[of + 1] - gap) / step + 1);
    if (most - least > 64) return true;
    for (int64_t by = least; by <= most; by++)
        if (meet(a, b, gap + by * step, of + 1)) return true;
    return false;
}
// No output lies over an input or over an output behind it in the list.
inline int outputs_apart(const char *rule, std::initializer_list<Lies> outputs, std::initializer_list<Lies> inputs) {
    for (const Lies *out = outputs.begin(); out != outputs.end(); out++) {
        if (!out->at) continue;
        const Repeats here(*out);
        auto over = [&](const Lies &other) {
            const int64_t gap = (int64_t)((uintptr_t)other.at - (uintptr_t)out->at);
            return other.at && gap < (int64_t)here.span[0] && meet(here, Repeats(other), gap);
        };
        for (const Lies &in : inputs)
            if (over(in)) return fail(TS_ERR_ARG, "%s: %s lies where %s does", rule, out->name, in.name);
        for (const Lies *other = out + 1; other != outputs.end(); other++)
            if (over(*other)) return fail(TS_ERR_ARG, "%s: %s lies where %s does", rule, out->name, other->name);
    }
    return TS_OK;
}

}  // namespace ts
