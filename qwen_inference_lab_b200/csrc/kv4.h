// The layout of pages that hold keys and values in 4 bits, and what the kernels over them share.
//
// A row of a head is cut into groups of 32 neighbouring elements.  With lo and hi the smallest and the largest element
//   m = bfloat16(lo), s = bfloat16((hi - lo) / 15) (through float32 each), code = rint((y - m) / s) within 0 .. 15,
// and the value held is m + s code: 16 bytes of codes and 4 of (s, m) a group, 5 bits an element.  s = 0 has codes 0.  A group
// with an element that is not finite, or whose s or m overflows, has s = m = NaN: who attends to it gets NaN, as with any
// other cache.
//
// One layer's pages are bytes [page][2 (keys, values)][kv head][page_size / 8][160 G], G = head_dim / 32 groups: of a run of 8
// slots first the codes [G][8 slots][16], element i of a group in byte i / 2 (even ones in the low half), then the pairs
// (s low, m high) as 32-bit words [8 slots][G].  A run is what a tensor-core fragment takes at a time: the 8 slots' 16 bytes of
// one group are 128 neighbouring bytes, so 32 lanes read them in one access, from global or from shared memory.
#pragma once
#include "common.cuh"
#include <string.h>

#define KV4_GROUP 32
#define KV4_MAX_DIM 256

__host__ __device__ __forceinline__ int kv4_run_bytes(int groups) { return 160 * groups; }

// Byte offset of the run that holds `slot` of (page, plane, head).
__device__ __forceinline__ size_t kv4_run_at(int page, int plane, int head, int slot, int kv_heads, int page_size, int groups) {
    return ((((size_t)page * 2 + plane) * kv_heads + head) * (page_size >> 3) + (slot >> 3)) * (size_t)(160 * groups);
}
__device__ __forceinline__ int kv4_code_at(int group, int slot) { return group * 128 + (slot & 7) * 16; }
__device__ __forceinline__ int kv4_pair_at(int group, int slot, int groups) { return 128 * groups + (slot & 7) * 4 * groups + 4 * group; }

__device__ __forceinline__ float kv4_step(unsigned pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float kv4_base(unsigned pair) { return __uint_as_float(pair & 0xffff0000u); }

// Block tables [rows][width] of physical pages by position / page size.
struct Kv4Table {
    const int* pages;
    int rows, width, page_size, num_pages;
    // The page of a request's position, or -1 where the table has none: never one outside the pool, whatever row and position are.
    __device__ __forceinline__ int page(int row, int position) const {
        const int index = position / page_size;
        if (row < 0 || row >= rows || position < 0 || index >= width) return -1;
        const int found = pages[(size_t)row * width + index];
        return found < num_pages ? found : -1;
    }
};

// The share of a context that a span kernel's block takes.  The longest context of the step is cut into at most n_spans parts of
// equal length, a multiple of `tile`; a token's own keys [low, end) start at a tile's border.  Empty when the context is over before.
struct Kv4Span {
    int first, last;     // keys [first, last)
    int count;           // spans of this token that hold anything
};
__device__ __forceinline__ Kv4Span kv4_span(int span, int n_spans, int longest, int low, int end, int tile) {
    const int start = low / tile * tile;
    const int tiles = (longest + tile - 1) / tile;
    const int length = (tiles + n_spans - 1) / n_spans * tile;
    Kv4Span s;
    s.count = (end - start + length - 1) / length;
    if (s.count > n_spans) s.count = n_spans;
    const long long at = start + (long long)span * length;
    s.first = (int)(at < low ? low : at);
    // the last span takes what is left, should a description have understated its longest context
    s.last = (span == s.count - 1 || at + length > end) ? end : (int)(at + length);
    return s;
}

// The entries take one struct each, pointers first and 32-bit numbers behind them, which the caller packs: converting thirty
// arguments one by one takes the host 4.6 us a call, packing them 1.0.
template <typename Call> static inline Call kv4_call(const void* packed) {
    Call call;
    memcpy(&call, packed, sizeof(Call));
    return call;
}
