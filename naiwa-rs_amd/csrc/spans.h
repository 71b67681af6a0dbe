// Whether two arguments of a call share memory, on the host.
#pragma once

#include <stdint.h>

namespace {

// `rows` rows of `bytes` bytes each, `step` bytes apart (rows = 0 or no address: nothing).
struct Span {
    uintptr_t at;
    int64_t rows, step, bytes;
};
static inline Span span_of(const void* p, int64_t rows, int64_t ld, int64_t n, int size) {
    return {(uintptr_t)p, p ? rows : 0, ld * size, n * size};
}
static inline Span span_of(const void* p, int64_t bytes) { return {(uintptr_t)p, p && bytes > 0 ? 1 : 0, bytes, bytes}; }

// Rows of one step share memory only if they do within a step: the halves of wider rows (a gate's and its up's, side
// by side) do not.  Of rows of different steps, all that lies between the first and the last counts.
static inline bool overlap(const Span& a, const Span& b) {
    if (a.rows <= 0 || b.rows <= 0) return false;
    const uintptr_t a_end = a.at + (uintptr_t)((a.rows - 1) * a.step + a.bytes);
    const uintptr_t b_end = b.at + (uintptr_t)((b.rows - 1) * b.step + b.bytes);
    if (a.at >= b_end || b.at >= a_end) return false;
    if (a.step != b.step) return true;
    const uintptr_t step = (uintptr_t)a.step, d = b.at >= a.at ? (b.at - a.at) % step : (step - (a.at - b.at) % step) % step;
    return d < (uintptr_t)a.bytes || step - d < (uintptr_t)b.bytes;
}

} // namespace
