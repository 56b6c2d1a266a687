// SPDX-License-Identifier: Apache-2.0
//
// Whether what one descriptor of a call writes is read or written by another one.

#ifndef FSTX_OVERLAP_H
#define FSTX_OVERLAP_H

#include <algorithm>
#include <stdint.h>
#include <stdlib.h>

namespace fstx_overlap {

// a block of bytes: `rows` segments of `width` bytes, `pitch` apart
struct Block {
    uint64_t at, width, pitch, rows;
    uint64_t end() const { return at + (rows - 1) * pitch + width; }
};

// [rows, cols] elements of `size` bytes with contiguous rows
inline Block block_of(const void *p, uint64_t rows, uint64_t cols, uint64_t pitch, uint64_t size) {
    return Block{(uint64_t)(uintptr_t)p, cols * size, (rows == 1 ? cols : pitch) * size, rows};
}

// ... with any strides: as rows or columns where these are contiguous, else the whole span
inline Block block_of(const void *p, uint64_t n0, uint64_t s0, uint64_t n1, uint64_t s1, uint64_t size) {
    if ((s1 == 1 || n1 == 1) && (n0 == 1 || s0 >= n1)) return block_of(p, n0, n1, s0, size);
    if ((s0 == 1 || n0 == 1) && (n1 == 1 || s1 >= n0)) return block_of(p, n1, n0, s1, size);
    const uint64_t span = ((n0 - 1) * s0 + (n1 - 1) * s1 + 1) * size;
    return Block{(uint64_t)(uintptr_t)p, span, span, 1};
}

inline bool overlap(const Block &a, const Block &b) {
    if (a.at >= b.end() || b.at >= a.end()) return false;
    // a single row has whatever pitch the other block has
    if (a.rows == 1 && b.rows > 1 && a.pitch != b.pitch && a.width <= b.pitch) return overlap(Block{a.at, a.width, b.pitch, 1}, b);
    if (b.rows == 1 && a.rows > 1 && a.pitch != b.pitch && b.width <= a.pitch) return overlap(a, Block{b.at, b.width, a.pitch, 1});
    if (a.pitch != b.pitch) return true; // spans that touch: not told apart further
    if (b.at < a.at) return overlap(b, a);
    // rows of one tensor: b starts `shift` rows and `col` bytes behind a
    const uint64_t shift = (b.at - a.at) / a.pitch, col = (b.at - a.at) % a.pitch;
    if (shift < a.rows && col < a.width) return true;
    return shift + 1 < a.rows && col + b.width > a.pitch; // b's rows run on into a's next rows
}

// What a descriptor touches.  A source may be its own descriptor's destination (the caller looks at how they lie).
enum Kind : uint32_t { kWritten, kSource, kRead };
struct Touched {
    Block block;
    uint32_t owner, kind;
};

inline bool conflict(const Touched &a, const Touched &b) {
    if (a.kind != kWritten && b.kind != kWritten) return false;
    if (a.owner == b.owner && (a.kind == kSource || b.kind == kSource)) return false;
    return overlap(a.block, b.block);
}

// Whether any two of `n` conflict.  Reorders `t`: sorted by address, one has to be held against those before it only
// that reach beyond its start, a few instead of all: a call may bring the weights of thousands of experts.
inline bool any_conflict(Touched *t, uint64_t n) {
    std::sort(t, t + n, [](const Touched &a, const Touched &b) { return a.block.at < b.block.at; });
    uint64_t reaching = 0; // t[0..reaching) may reach beyond the current start (compacted in place: reaching <= i)
    for (uint64_t i = 0; i < n; ++i) {
        const Touched now = t[i];
        uint64_t keep = 0;
        for (uint64_t k = 0; k < reaching; ++k) {
            if (t[k].block.end() <= now.block.at) continue;
            if (conflict(t[k], now)) return true;
            t[keep++] = t[k];
        }
        t[keep++] = now;
        reaching = keep;
    }
    return false;
}

// Room for `n` of them: on the stack for a few, else on the heap; null where there is no memory.
struct List {
    Touched few[64];
    Touched *at;
    uint64_t n = 0;
    explicit List(uint64_t room) : at(room <= 64 ? few : static_cast<Touched *>(malloc(room * sizeof(Touched)))) {}
    ~List() {
        if (at != few) free(at);
    }
    List(const List &) = delete;
    List &operator=(const List &) = delete;
    void add(const Block &b, uint32_t owner, Kind kind) { at[n++] = Touched{b, owner, kind}; }
};

} // namespace fstx_overlap

#endif // FSTX_OVERLAP_H
