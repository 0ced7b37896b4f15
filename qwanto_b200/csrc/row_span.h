// Where a call's rows lie in memory, to refuse outputs over inputs that are still read.
#pragma once

#include <cstdint>
#include <utility>

namespace qkv {

// rows in memory: where the first starts, and in bytes their distance and length
struct RowSpan {
    uintptr_t at;
    uint64_t stride, bytes, rows;
    uintptr_t end() const { return at + (rows - 1) * stride + bytes; }
};
// whether two sets of rows (one row at least, none longer than its stride) have a byte in common
inline bool rows_meet(RowSpan a, RowSpan b) {
    if (a.at > b.at) std::swap(a, b);
    if (b.at >= a.end()) return false;
    if (a.stride == b.stride) {  // side by side in one buffer, or not
        const uint64_t d = (b.at - a.at) % a.stride;
        return d < a.bytes || d + b.bytes > a.stride;
    }
    if (a.rows > b.rows) std::swap(a, b);
    for (uint64_t i = 0; i < a.rows; i++) {
        const uintptr_t x = a.at + i * a.stride;
        uint64_t next = 0;  // the first row of b that starts after x
        if (x >= b.at) {
            const uint64_t k = (x - b.at) / b.stride;
            if (k < b.rows && x - b.at - k * b.stride < b.bytes) return true;
            next = k + 1;
        }
        if (next < b.rows && b.at + next * b.stride < x + a.bytes) return true;
    }
    return false;
}

}  // namespace qkv
