// Copies of byte ranges at any addresses.
#pragma once

#include "common.h"

namespace fie {

constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;                                      // 16-byte pieces of a thread on their way together
constexpr int kCopyChunk = kCopyThreads * kCopyUnroll * 16;         // bytes of a workgroup
constexpr int kMostBlocks = (1 << 24) - 1;                          // a launch holds fewer than 2^32 threads

// Memory of the device by an address of any make: without the address space the compiler has to
// take it for LDS as well, and waits for each access before the next.
#define FIE_GLOBAL __attribute__((address_space(1)))
template <class T> FIE_DEV T global_get(const void* p) { return *(const FIE_GLOBAL T*)(uintptr_t)p; }
template <class T> FIE_DEV void global_put(void* p, T v) { *(FIE_GLOBAL T*)(uintptr_t)p = v; }

typedef uint32_t vec4_t __attribute__((ext_vector_type(4)));
typedef uint32_t vec4_word_t __attribute__((ext_vector_type(4), aligned(4)));

// 16 bytes at p, whose low two bits are sh: the 16 from the word that holds the first, the word
// after them, and a shift.  Only words that hold some of the 16 bytes are touched.
struct Bytes16 {
    vec4_t r;
    uint32_t e;
    FIE_DEV void load(const uint8_t* p, uint32_t sh)
    {
        r = global_get<vec4_word_t>(p - sh);
        e = global_get<uint32_t>(p + (sh ? 16 - sh : 12));
    }
    FIE_DEV vec4_t get(uint32_t sh) const
    {
        return vec4_t{__builtin_amdgcn_alignbyte(r.y, r.x, sh), __builtin_amdgcn_alignbyte(r.z, r.y, sh),
                      __builtin_amdgcn_alignbyte(r.w, r.z, sh), __builtin_amdgcn_alignbyte(e, r.w, sh)};
    }
};

// Chunk `chunk` of the copy of a range of bytes: the kCopyChunk bytes from dst's 16-byte block on (and so
// many chunks further), as far as they are inside the range.  Whole blocks of dst go as one store
// each, the range's first and last bytes one by one.
FIE_DEV void copy_chunk(uint8_t* dst, const uint8_t* src, int64_t bytes, int chunk)
{
    const int tid = threadIdx.x;
    const int shift = (int)((uintptr_t)dst & 15);
    const int64_t left = shift + bytes - (int64_t)chunk * kCopyChunk;
    if (left <= 0) return;
    uint8_t* const d = dst - shift + (int64_t)chunk * kCopyChunk;               // aligned
    const uint8_t* const s = src - shift + (int64_t)chunk * kCopyChunk;
    const uint32_t sh = (uint32_t)(uintptr_t)s & 3u;
    const bool even = ((uintptr_t)s & 15) == 0;
    const int lo = chunk ? 0 : shift, hi = (int)(left < kCopyChunk ? left : kCopyChunk);
    const int first = (lo + 15) & ~15, last = hi & ~15;                         // whole blocks
    if (first == 0 && last == kCopyChunk && even) {
        vec4_t v[kCopyUnroll];
#pragma unroll
        for (int u = 0; u < kCopyUnroll; ++u) v[u] = global_get<vec4_t>(s + (u * kCopyThreads + tid) * 16);
#pragma unroll
        for (int u = 0; u < kCopyUnroll; ++u) global_put(d + (u * kCopyThreads + tid) * 16, v[u]);
        return;
    }
    if (first < last) {
        Bytes16 v[kCopyUnroll];
        // (a thread past the end loads the last block again)
#pragma unroll
        for (int u = 0; u < kCopyUnroll; ++u) {
            const uint8_t* p = s + min(first + (u * kCopyThreads + tid) * 16, last - 16);
            if (even) v[u].r = global_get<vec4_t>(p);
            else v[u].load(p, sh);
        }
#pragma unroll
        for (int u = 0; u < kCopyUnroll; ++u) {
            const int at = first + (u * kCopyThreads + tid) * 16;
            if (at < last) global_put(d + at, even ? v[u].r : v[u].get(sh));
        }
    }
    // the bytes in front of the blocks and behind them; without blocks [lo, hi) is at most two pieces
    const int front = min(first, hi), back = max(last, front);
    const int at = tid < 16 ? lo + tid : back + tid - 16;
    if (tid < 32 && at < (tid < 16 ? front : hi)) global_put(d + at, global_get<uint8_t>(s + at));
}

}  // namespace fie
