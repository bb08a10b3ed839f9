// Copies of byte ranges at any addresses.
#pragma once

#include "common.h"

namespace fie {

constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;                                      // 16-byte pieces of a thread on their way together
constexpr int kCopyChunk = kCopyThreads * kCopyUnroll * 16;         // bytes of a workgroup
constexpr int kMostBlocks = 1 << 24;                                // a launch holds fewer than 2^32 threads

// 16 bytes at p, whose low two bits are sh: the 16 from the word that holds the first, the word
// after them, and a shift.  Only words that hold some of the 16 bytes are touched.
struct Bytes16 {
    typedef uint32_t raw __attribute__((ext_vector_type(4), aligned(4)));
    raw r;
    uint32_t e;
    FIE_DEV void load(const uint8_t* p, uint32_t sh)
    {
        r = *(const raw*)(p - sh);
        e = sh ? *(const uint32_t*)(p - sh + 16) : 0;
    }
    FIE_DEV uint4 get(uint32_t sh) const
    {
        return make_uint4(__builtin_amdgcn_alignbyte(r.y, r.x, sh), __builtin_amdgcn_alignbyte(r.z, r.y, sh),
                          __builtin_amdgcn_alignbyte(r.w, r.z, sh), __builtin_amdgcn_alignbyte(e, r.w, sh));
    }
};

// The bytes [from, to) of dst, counted from dst's 16-byte block, that are inside [0, bytes) of
// the range: what a workgroup of kCopyThreads does of a copy of `bytes` bytes cut into chunks.  Whole
// blocks of dst go as one store each, its first and last bytes one by one.
FIE_DEV void copy_chunk(uint8_t* dst, const uint8_t* src, int64_t bytes, int chunk)
{
    const int tid = threadIdx.x;
    const int64_t shift = (int64_t)((uintptr_t)dst & 15);
    uint8_t* const d = dst - shift;                                 // aligned
    const uint8_t* const s = src - shift;
    const int64_t end = shift + bytes;
    const int64_t lo = (int64_t)chunk * kCopyChunk, hi = lo + kCopyChunk < end ? lo + kCopyChunk : end;
    if (lo >= end) return;
    const int64_t first = lo < shift ? 16 : lo, last = hi & ~INT64_C(15);       // whole blocks (shift < 16)
    if (chunk == 0 && shift && tid < 16) {
        const int64_t at = tid;
        if (at >= shift && at < end) d[at] = s[at];
    }
    if (hi == end && (end & 15) && (last >= first || shift == 0 || chunk > 0) && tid >= 64 && tid < 80) {
        const int64_t at = last + (tid - 64);
        if (at < end && at >= shift) d[at] = s[at];
    }
    const uint32_t sh = (uint32_t)(uintptr_t)s & 3u;
    if (((uintptr_t)s & 15) == 0) {
        uint4 v[kCopyUnroll];
#pragma unroll
        for (int u = 0; u < kCopyUnroll; ++u) {
            const int64_t at = first + ((int64_t)u * kCopyThreads + tid) * 16;
            if (at < last) v[u] = *(const uint4*)(s + at);
        }
#pragma unroll
        for (int u = 0; u < kCopyUnroll; ++u) {
            const int64_t at = first + ((int64_t)u * kCopyThreads + tid) * 16;
            if (at < last) *(uint4*)(d + at) = v[u];
        }
    } else {
        Bytes16 v[kCopyUnroll];
#pragma unroll
        for (int u = 0; u < kCopyUnroll; ++u) {
            const int64_t at = first + ((int64_t)u * kCopyThreads + tid) * 16;
            if (at < last) v[u].load(s + at, sh);
        }
#pragma unroll
        for (int u = 0; u < kCopyUnroll; ++u) {
            const int64_t at = first + ((int64_t)u * kCopyThreads + tid) * 16;
            if (at < last) *(uint4*)(d + at) = v[u].get(sh);
        }
    }
}

}  // namespace fie
