// The matrix product in 8-bit integers with scales for each token and channel
// (fie_int8_linear): y = x_scale w_scale sum_k x w + bias.
#pragma once

#include "launchers.h"
#include "fie_ops.h"

namespace fie {

typedef int32_t i32x4_t __attribute__((ext_vector_type(4)));

// D += A (16 x 64) B (64 x 16) in int32.  Lane l supplies 16 consecutive k of A's row l % 16
// and of B's column l % 16, k-group l / 16, and receives D rows 4 (l / 16) .. +3 of column
// l % 16.  Whatever order the instruction pairs k in, A and B take it alike.
FIE_DEV i32x4_t mfma_i8(i32x4_t a, i32x4_t b, i32x4_t c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }

template <int DT>
FIE_DEV uint16_t round16(float v)
{
    if constexpr (DT == FIE_BF16) return __builtin_bit_cast(uint16_t, (__bf16)v);
    else return __builtin_bit_cast(uint16_t, (_Float16)v);
}

// Four neighbouring channels of one token, scaled, from n on: one store where `wide` (rows of
// y aligned to four elements) and all four are inside.
template <int DT>
FIE_DEV void store_scaled(const fie_int8_args& a, int64_t m, int n, i32x4_t acc, float xs, bool wide)
{
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = min(n + i, a.n - 1);
        v[i] = (float)acc[i] * xs * a.w_scale[c];
        if (a.bias) v[i] += a.bias[c];
    }
    if constexpr (DT == FIE_F32) {
        float* p = (float*)a.y + m * a.y_stride + n;
        if (wide && n + 4 <= a.n) *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);
        else
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < a.n) p[i] = v[i];
    } else {
        uint16_t* p = (uint16_t*)a.y + m * a.y_stride + n;
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = round16<DT>(v[i]);
        if (wide && n + 4 <= a.n) *(uint2*)p = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
        else
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < a.n) p[i] = (uint16_t)h[i];
    }
}

constexpr int kI8K = 128;               // bytes of k a stage

// Chunk c (of 8) of operand row n sits at slot n * 8 + (c ^ (n & 7)): the eight lanes one LDS
// cycle serves read eight rows' chunk c from eight distinct bank groups.
FIE_DEV int i8_slot(int n, int c) { return n * 8 + (c ^ (n & 7)); }

// 16 bytes of a row from k0 on; those at or past K are 0.
FIE_DEV i32x4_t load_k(const int8_t* rowp, int k0, int K)
{
    typedef int32_t raw __attribute__((ext_vector_type(4), aligned(1)));
    if (k0 + 16 <= K) {
        const raw r = *(const raw*)(rowp + k0);
        return i32x4_t{r.x, r.y, r.z, r.w};
    }
    i32x4_t r{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (k0 + i < K) r[i / 4] |= (int32_t)((uint32_t)(uint8_t)rowp[k0 + i] << (8 * (i % 4)));
    return r;
}

// 64 WM tokens by 64 WN channels a workgroup of WM x WN waves, 64 x 64 each; k in stages of
// 128 through two LDS buffers, the next stage in registers meanwhile.  Grid: 8 * ceil(tiles /
// 8) * nrb, dealt to the XCDs so that a channel tile's token blocks follow one another on one.
template <int DT, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_int8_tile(const fie_int8_args a, int nrb, int wide)
{
    constexpr int BM = 64 * WM, BN = 64 * WN, TH = 64 * WM * WN;
    constexpr int NC = (BM + BN) * (kI8K / 16) / TH;            // 16-byte chunks per thread and stage
    __shared__ i32x4_t L[2][(BM + BN) * (kI8K / 16)];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int xcd = blockIdx.x & 7, kb = blockIdx.x >> 3;
    const int t0 = (8 * (kb / nrb) + xcd) * BN;
    const int64_t r0 = (int64_t)(kb % nrb) * BM;
    if (t0 >= a.n) return;
    const int8_t* src[NC];
    int dst[NC], off[NC];
#pragma unroll
    for (int j = 0; j < NC; ++j) {
        const int p = j * TH + tid, n = p >> 3, c = p & 7;
        src[j] = n < BM ? a.x + min(r0 + n, a.m - 1) * a.x_stride : a.w + (int64_t)min(t0 + n - BM, a.n - 1) * a.w_stride;
        off[j] = 16 * c;
        dst[j] = i8_slot(n, c);
    }
    const int ns = (a.k + kI8K - 1) / kI8K;
    i32x4_t r[NC];
    auto load = [&](int s) {
#pragma unroll
        for (int j = 0; j < NC; ++j) r[j] = load_k(src[j], s * kI8K + off[j], a.k);
    };
    const int wr = wave % WM, wn = wave / WM;
    i32x4_t acc[4][4];
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[m][q] = i32x4_t{0, 0, 0, 0};
    load(0);
    for (int s = 0; s < ns; ++s) {
        const int b = s & 1;
#pragma unroll
        for (int j = 0; j < NC; ++j) L[b][dst[j]] = r[j];
        __syncthreads();                        // the buffer's readers of two stages ago are behind it
        if (s + 1 < ns) load(s + 1);
#pragma unroll
        for (int kk = 0; kk < kI8K / 64; ++kk) {
            const int c = kk * 4 + (lane >> 4);
            i32x4_t fx[4], fw[4];
#pragma unroll
            for (int m = 0; m < 4; ++m) fx[m] = L[b][i8_slot(64 * wr + 16 * m + (lane & 15), c)];
#pragma unroll
            for (int q = 0; q < 4; ++q) fw[q] = L[b][i8_slot(BM + 64 * wn + 16 * q + (lane & 15), c)];
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[m][q] = mfma_i8(fw[q], fx[m], acc[m][q]);
        }
    }
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        const int64_t row = r0 + 64 * wr + 16 * m + (lane & 15);
        if (row >= a.m) continue;
        const float xs = a.x_scale[row];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int n = t0 + 64 * wn + 16 * q + 4 * (lane >> 4);
            if (n < a.n) store_scaled<DT>(a, row, n, acc[m][q], xs, wide);
        }
    }
}

}  // namespace fie
