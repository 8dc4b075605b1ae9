// Do the rows that a kernel writes lie over rows that it reads?  Host only, exact, and without a loop where both lie apart or step alike.
#pragma once

#include <cstdint>

namespace hipq {

// rows of `bytes` bytes, `step` bytes apart
struct ByteRows {
    int64_t at, step, bytes;
    int count;
    int64_t first() const { return at; }
    int64_t end() const { return at + (count - 1) * step + bytes; }
    // does [lo, lo + n) share a byte with one of them?
    bool meets(int64_t lo, int64_t n) const
    {
        const int64_t behind = lo - (at + bytes); // the first row that ends behind lo
        const int64_t r = behind < 0 ? 0 : step > 0 ? behind / step + 1 : count;
        return r < count && at + r * step < lo + n;
    }
};

// steps above 0, or a single row
static inline bool overlap(const ByteRows &a, const ByteRows &b)
{
    if (a.end() <= b.first() || b.end() <= a.first())
        return false;
    if (a.step == b.step || a.count == 1 || b.count == 1) // how far apart two rows are depends on the difference of their numbers
        return a.meets(b.at, b.bytes) || b.meets(a.at, a.bytes);
    for (int i = 0; i < a.count; i++)
        if (b.meets(a.at + i * a.step, a.bytes))
            return true;
    return false;
}

} // namespace hipq
