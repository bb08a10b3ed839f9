// Low-rank adapters of many tokens (fie_adapter_linear): y = base + scale B (A x).
#pragma once

#include <type_traits>

#include "launchers.h"
#include "fie_decode.h"

namespace fie {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_word_t __attribute__((ext_vector_type(4), aligned(4)));

// 16 bytes of an operand a lane: consecutive elements of row l % 16, group l / 16.  One instruction
// of 8 two-byte elements a lane, four of one fp32 element; A and B take any order of the summed index
// alike.
template <int DT> struct Operand {
    static constexpr int SIZE = DT == FIE_F32 ? 4 : 2, EACH = 16 / SIZE, STEP = 4 * EACH;
    static FIE_DEV f32x4_t mul(u32x4_t a, u32x4_t b, f32x4_t c)
    {
        if constexpr (DT == FIE_BF16)
            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
        else if constexpr (DT == FIE_F16)
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
        else {
#pragma unroll
            for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
            return c;
        }
    }
    static FIE_DEV uint32_t bits(float v)
    {
        if constexpr (DT == FIE_BF16) return __builtin_bit_cast(uint16_t, (__bf16)v);
        else if constexpr (DT == FIE_F16) return __builtin_bit_cast(uint16_t, (_Float16)v);
        else return __float_as_uint(v);
    }
    static FIE_DEV float value(uint32_t b)
    {
        if constexpr (DT == FIE_BF16) return __uint_as_float(b << 16);
        else if constexpr (DT == FIE_F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)b);
        else return __uint_as_float(b);
    }
};

// The plan: [0] the number of tiles, then each tile's adapter (-1: none), first place and tokens,
// then the tokens in places.
constexpr int kPlanHead = 4, kPlanTile = 4;

FIE_DEV int plan_tiles_of(int tokens, int adapters, int tile) { return tokens / tile + min(tokens, adapters + 1); }

constexpr int kPlanThreads = 1024;

// One workgroup: counts, where each adapter's tokens begin, and the tokens' places.  (In which
// order an adapter's tokens stand changes no result: each is a column of its own.)
__global__ __launch_bounds__(kPlanThreads) void k_adapter_plan(const fie_adapter_plan_args a, int most)
{
    __shared__ int32_t count[FIE_MAX_ADAPTERS + 1], next[FIE_MAX_ADAPTERS + 1];
    __shared__ int32_t part[2][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, kinds = a.adapters + 1;
    int32_t* const tiles = a.plan + kPlanHead;
    int32_t* const order = tiles + (int64_t)most * kPlanTile;
    auto kind = [&](int t) {
        const int i = a.ids[t];
        return i >= 0 && i < a.adapters ? i + 1 : 0;
    };
    for (int i = tid; i < kinds; i += kPlanThreads) count[i] = 0;
    __syncthreads();
    for (int t = tid; t < a.tokens; t += kPlanThreads) atomicAdd(&count[kind(t)], 1);
    __syncthreads();
    const int each = (kinds + kPlanThreads - 1) / kPlanThreads, first = tid * each, last = min(first + each, kinds);
    int sum = 0, cut = 0;
    for (int i = first; i < last; ++i) {
        sum += count[i];
        cut += (count[i] + a.tile - 1) / a.tile;
    }
    const int s = (int)wave_incl_scan_u32((uint32_t)sum), c = (int)wave_incl_scan_u32((uint32_t)cut);
    if (lane == 63) {
        part[0][wave] = s;
        part[1][wave] = c;
    }
    __syncthreads();
    int at = s - sum, tile = c - cut;
    for (int w = 0; w < wave; ++w) {
        at += part[0][w];
        tile += part[1][w];
    }
    if (tid == kPlanThreads - 1) a.plan[0] = tile + cut;
    for (int i = first; i < last; ++i) {
        next[i] = at;
        for (int n = 0; n < count[i]; n += a.tile, ++tile) {
            tiles[tile * kPlanTile] = i - 1;
            tiles[tile * kPlanTile + 1] = at + n;
            tiles[tile * kPlanTile + 2] = min(a.tile, count[i] - n);
        }
        at += count[i];
    }
    __syncthreads();
    for (int t = tid; t < a.tokens; t += kPlanThreads) order[atomicAdd(&next[kind(t)], 1)] = t;
}

struct AdapterWork {
    float* h;                   // [splits][tokens in places][rank]
    int splits, most;           // of k; tiles of the plan
};

// What a lane holds of 16 bytes' worth of x: elements [at, at + EACH) of a row at any address, those at
// or past k as 0.
template <int DX, int DT, bool ALIGNED> struct TokenLoad {
    static constexpr int EACH = Operand<DT>::EACH;
    static constexpr int XS = DX == FIE_I8 ? 1 : Operand<DT>::SIZE;
    u32x4_t r;
    uint32_t e;
    FIE_DEV void load(const uint8_t* p)                 // inside the row
    {
        if constexpr (DX == FIE_I8) {
            if constexpr (ALIGNED) {
                if constexpr (EACH == 8) {
                    const uint2 v = *(const uint2*)p;
                    r.x = v.x;
                    r.y = v.y;
                } else r.x = *(const uint32_t*)p;
            } else {
                const uint32_t sh = (uint32_t)(uintptr_t)p & 3u;
                const uint32_t* w = (const uint32_t*)(p - sh);
                r.x = w[0];
                r.y = EACH == 8 || sh ? w[1] : 0;
                r.z = EACH == 8 && sh ? w[2] : 0;
                e = sh;
            }
        } else if constexpr (ALIGNED) r = *(const u32x4_t*)p;
        else if constexpr (DT == FIE_F32) r = *(const u32x4_word_t*)p;
        else {
            const uint32_t sh = (uint32_t)(uintptr_t)p & 2u;
            r = *(const u32x4_word_t*)(p - sh);
            e = *(const uint32_t*)(p + (sh ? 14 : 12));
        }
    }
    FIE_DEV u32x4_t get(const uint8_t* p) const
    {
        if constexpr (DX == FIE_I8) {
            uint32_t w[2] = {r.x, EACH == 8 ? r.y : 0};
            if constexpr (!ALIGNED) {
                w[0] = __builtin_amdgcn_alignbyte(r.y, r.x, e);
                w[1] = __builtin_amdgcn_alignbyte(r.z, r.y, e);
            }
            u32x4_t o;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                auto at = [&](int j) { return (float)(int8_t)(w[j / 4] >> (8 * (j % 4))); };
                if constexpr (EACH == 8) o[i] = Operand<DT>::bits(at(2 * i)) | (Operand<DT>::bits(at(2 * i + 1)) << 16);
                else o[i] = __float_as_uint(at(i));
            }
            return o;
        } else if constexpr (ALIGNED || DT == FIE_F32) return r;
        else {
            const uint32_t sh = (uint32_t)(uintptr_t)p & 2u;
            return u32x4_t{__builtin_amdgcn_alignbyte(r.y, r.x, sh), __builtin_amdgcn_alignbyte(r.z, r.y, sh),
                           __builtin_amdgcn_alignbyte(r.w, r.z, sh), __builtin_amdgcn_alignbyte(e, r.w, sh)};
        }
    }
    static FIE_DEV u32x4_t last(const uint8_t* row, int at, int k)
    {
        u32x4_t o{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            if (at + j >= k) continue;
            uint32_t b;
            if constexpr (DX == FIE_I8) b = Operand<DT>::bits((float)((const int8_t*)row)[at + j]);
            else if constexpr (DT == FIE_F32) b = ((const uint32_t*)row)[at + j];
            else b = ((const uint16_t*)row)[at + j];
            if constexpr (EACH == 8) o[j / 2] |= b << (16 * (j % 2));
            else o[j] = b;
        }
        return o;
    }
};

constexpr int kDownWaves = 4, kDownSteps = 4;           // steps of k of a wave at a time

// h = A x: grid (splits, tiles), 16 MT tokens by 16 RT ranks a workgroup, whose waves and the splits
// take k in turn.  Operands come straight from memory: a row of A is read once for its tile's
// tokens, x once.
template <int DX, int DT, int MT, int RT, bool ALIGNED>
__global__ __launch_bounds__(64 * kDownWaves) void k_adapter_down(const fie_adapter_args a, const AdapterWork w)
{
    using Op = Operand<DT>;
    using Tok = TokenLoad<DX, DT, ALIGNED>;
    constexpr int XS = Tok::XS;
    __shared__ f32x4_t red[kDownWaves][MT * RT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if ((int)blockIdx.y >= a.plan[0]) return;
    const int32_t* tile = a.plan + kPlanHead + blockIdx.y * kPlanTile;
    const int32_t* order = a.plan + kPlanHead + (int64_t)w.most * kPlanTile;
    const int id = tile[0], first = tile[1], count = tile[2];
    if (id < 0) return;
    const int rank = a.ranks[id];
    const uint8_t* row[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int t = order[first + min(16 * m + (lane & 15), count - 1)];
        row[m] = (const uint8_t*)a.x + (int64_t)t * a.x_stride * XS;
    }
    const int group = lane >> 4;
    const int full = a.k / Op::STEP, steps = (a.k + Op::STEP - 1) / Op::STEP;
    for (int r0 = 0; r0 < rank; r0 += 16 * RT) {
        const uint8_t* ar[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r)
            ar[r] = (const uint8_t*)a.a + ((int64_t)id * a.rank + min(r0 + 16 * r, a.rank - 16) + (lane & 15)) * a.k_pad * Op::SIZE + 16 * group;
        f32x4_t acc[MT][RT];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int r = 0; r < RT; ++r) acc[m][r] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        for (int c = (blockIdx.x * kDownWaves + wave) * kDownSteps; c < steps; c += gridDim.x * kDownWaves * kDownSteps) {
            if (c + kDownSteps <= full) {
                u32x4_t fa[kDownSteps][RT];
                Tok fx[kDownSteps][MT];
#pragma unroll
                for (int u = 0; u < kDownSteps; ++u) {
#pragma unroll
                    for (int r = 0; r < RT; ++r) fa[u][r] = *(const u32x4_t*)(ar[r] + (int64_t)(c + u) * 64);
#pragma unroll
                    for (int m = 0; m < MT; ++m) fx[u][m].load(row[m] + ((c + u) * Op::STEP + group * Op::EACH) * XS);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < kDownSteps; ++u)
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        const u32x4_t x = fx[u][m].get(row[m] + ((c + u) * Op::STEP + group * Op::EACH) * XS);
#pragma unroll
                        for (int r = 0; r < RT; ++r) acc[m][r] = Op::mul(fa[u][r], x, acc[m][r]);
                    }
            } else
#pragma unroll 1
                for (int u = c; u < min(c + kDownSteps, steps); ++u)
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        const u32x4_t x = Tok::last(row[m], u * Op::STEP + group * Op::EACH, a.k);
#pragma unroll
                        for (int r = 0; r < RT; ++r) acc[m][r] = Op::mul(*(const u32x4_t*)(ar[r] + (int64_t)u * 64), x, acc[m][r]);
                    }
        }
        __syncthreads();
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int r = 0; r < RT; ++r) red[wave][m * RT + r][lane] = acc[m][r];
        __syncthreads();
        for (int f = wave; f < MT * RT; f += kDownWaves) {
            f32x4_t t = red[0][f][lane];
#pragma unroll
            for (int i = 1; i < kDownWaves; ++i) t += red[i][f][lane];
            const int m = 16 * (f / RT) + (lane & 15), r = r0 + 16 * (f % RT) + 4 * group;
            if (m < count && r < a.rank) *(f32x4_t*)(w.h + ((int64_t)blockIdx.x * a.tokens + first + m) * a.rank + r) = t;
        }
    }
}

constexpr int kUpWaves = 4, kUpCols = 4;                // 16-channel blocks of a wave
constexpr int kUpChannels = 16 * kUpCols * kUpWaves;

template <int DT> FIE_DEV void load4(const void* p, int64_t at, bool wide, int left, float* v)
{
    using Op = Operand<DT>;
    if (wide && left >= 4) {
        if constexpr (DT == FIE_F32) {
            const float4 f = *(const float4*)((const float*)p + at);
            v[0] = f.x;
            v[1] = f.y;
            v[2] = f.z;
            v[3] = f.w;
        } else {
            const uint2 u = *(const uint2*)((const uint16_t*)p + at);
            v[0] = Op::value(u.x & 0xFFFFu);
            v[1] = Op::value(u.x >> 16);
            v[2] = Op::value(u.y & 0xFFFFu);
            v[3] = Op::value(u.y >> 16);
        }
    } else
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i >= left) continue;
            if constexpr (DT == FIE_F32) v[i] = ((const float*)p)[at + i];
            else v[i] = Op::value(((const uint16_t*)p)[at + i]);
        }
}

template <int DT> FIE_DEV void store4(void* p, int64_t at, bool wide, int left, const float* v)
{
    using Op = Operand<DT>;
    if (wide && left >= 4) {
        if constexpr (DT == FIE_F32) *(float4*)((float*)p + at) = make_float4(v[0], v[1], v[2], v[3]);
        else *(uint2*)((uint16_t*)p + at) = make_uint2(Op::bits(v[0]) | (Op::bits(v[1]) << 16), Op::bits(v[2]) | (Op::bits(v[3]) << 16));
    } else
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i >= left) continue;
            if constexpr (DT == FIE_F32) ((float*)p)[at + i] = v[i];
            else ((uint16_t*)p)[at + i] = (uint16_t)Op::bits(v[i]);
        }
}

// y = base + scale B h: grid (blocks of kUpChannels channels, tiles).  h goes into LDS summed over the
// splits, in fp32; with two-byte adapters each 16 ranks of it are taken as 16 leading and 16 trailing
// parts against the same 16 of B, one instruction.  fp16 tokens are brought to an exponent of their
// own first, so that no part overflows.  Bound by base and y.
template <int DT, int DY, int DB, int MT>
__global__ __launch_bounds__(64 * kUpWaves) void k_adapter_up(const fie_adapter_args a, const AdapterWork w, int wide)
{
    using Op = Operand<DT>;
    extern __shared__ float H[];                        // [16 MT][rank + 4]
    __shared__ float factor[16 * MT];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), group = lane >> 4;
    if ((int)blockIdx.y >= a.plan[0]) return;
    const int32_t* tile = a.plan + kPlanHead + blockIdx.y * kPlanTile;
    const int32_t* order = a.plan + kPlanHead + (int64_t)w.most * kPlanTile;
    const int id = tile[0], first = tile[1], count = tile[2];
    const int rank = id < 0 ? 0 : a.ranks[id], pitch = a.rank + 4;
    if (rank == 0 && a.base == a.y) return;
    const int ranks = (rank + 15) / 16 * 16;
    if (rank) {
        const float s = a.scale[id];
        for (int i = tid; i < 16 * MT * ranks; i += 64 * kUpWaves) {
            const int m = i / ranks, r = i - m * ranks;
            float v = 0.0f;
            if (m < count)
                for (int p = 0; p < w.splits; ++p) v += w.h[((int64_t)p * a.tokens + first + m) * a.rank + r];
            H[m * pitch + r] = v;
        }
        __syncthreads();
        if (tid < 16 * MT) {
            float f = s;
            if (a.x_scale && tid < count) f *= a.x_scale[order[first + tid]];
            if constexpr (DT == FIE_F16) {
                float most = 0.0f;
                for (int r = 0; r < ranks; ++r) most = __builtin_fmaxf(most, __builtin_fabsf(H[tid * pitch + r]));
                const int e = most > 0.0f && most <= 3.4e38f ? (int)((__float_as_uint(most) >> 23) & 255u) - 127 : 0;
                for (int r = 0; r < ranks; ++r) H[tid * pitch + r] = __builtin_ldexpf(H[tid * pitch + r], -e);
                f = __builtin_ldexpf(f, e);
            }
            factor[tid] = f;
        }
        __syncthreads();
    }
    const int n0 = (blockIdx.x * kUpWaves + wave) * (16 * kUpCols);
    if (n0 >= a.n) return;
    f32x4_t acc[MT][kUpCols];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int q = 0; q < kUpCols; ++q) acc[m][q] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    const uint8_t* br[kUpCols];
    const int inner = DT == FIE_F32 ? 16 * group : 16 * (group & 1);
#pragma unroll
    for (int q = 0; q < kUpCols; ++q)
        br[q] = (const uint8_t*)a.b + ((int64_t)max(id, 0) * a.n + min(n0 + 16 * q + (lane & 15), a.n - 1)) * a.rank * Op::SIZE + inner;
    for (int r0 = 0; r0 < ranks; r0 += 16) {
        u32x4_t fb[kUpCols];
#pragma unroll
        for (int q = 0; q < kUpCols; ++q) fb[q] = *(const u32x4_t*)(br[q] + r0 * Op::SIZE);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            if (16 * m >= count) continue;
            const float* h = H + (16 * m + (lane & 15)) * pitch + r0 + (DT == FIE_F32 ? 4 * group : 8 * (group & 1));
            u32x4_t fh;
            if constexpr (DT == FIE_F32) {
#pragma unroll
                for (int i = 0; i < 4; ++i) fh[i] = __float_as_uint(h[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t part[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float v = h[2 * i + j];
                        const uint32_t lead = Op::bits(v);
                        const float rest = v - Op::value(lead);
                        // (an infinity has no rest)
                        part[j] = group < 2 ? lead : Op::bits(__builtin_fabsf(Op::value(lead)) <= 3.4e38f ? rest : 0.0f);
                    }
                    fh[i] = part[0] | (part[1] << 16);
                }
            }
#pragma unroll
            for (int q = 0; q < kUpCols; ++q) acc[m][q] = Op::mul(fb[q], fh, acc[m][q]);
        }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int c = 16 * m + (lane & 15);
        if (c >= count) continue;
        const int64_t t = order[first + c];
        const float f = rank ? factor[c] : 0.0f;
#pragma unroll
        for (int q = 0; q < kUpCols; ++q) {
            const int n = n0 + 16 * q + 4 * group, left = a.n - n;
            if (left <= 0) continue;
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (a.base) load4<DB>(a.base, t * a.base_stride + n, wide & 1, left, v);
            if (rank)
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] += f * acc[m][q][i];
            store4<DY>(a.y, t * a.y_stride + n, wide & 2, left, v);
        }
    }
}

}  // namespace fie
