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

// The plan: [0] the number of tiles, then each tile's adapter (-1: none), first place and tokens (16 at
// most), then the tokens in places.
constexpr int kPlanHead = 4, kPlanTile = 4, kTileTokens = 16;

constexpr int kPlanThreads = 1024;

// One workgroup: counts, where each adapter's tokens begin, and the tokens' places.  (In which
// order an adapter's tokens stand changes no result: each is a column of its own.)  Once a batch: 1 and
// 250 tokens 2.6 us, 4001 8.5, 65536 113 (two passes of one workgroup, LDS atomics on few counters).
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
        cut += (count[i] + kTileTokens - 1) / kTileTokens;
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
        for (int n = 0; n < count[i]; n += kTileTokens, ++tile) {
            tiles[tile * kPlanTile] = i - 1;
            tiles[tile * kPlanTile + 1] = at + n;
            tiles[tile * kPlanTile + 2] = min(kTileTokens, count[i] - n);
        }
        at += count[i];
    }
    __syncthreads();
    for (int t = tid; t < a.tokens; t += kPlanThreads) order[atomicAdd(&next[kind(t)], 1)] = t;
}

struct AdapterWork {
    float* h;                   // [splits][places][rank], the first product by parts of k
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

constexpr int kDownWaves = 4;

// h = A x: grid (splits, tiles), 16 tokens of one adapter a workgroup.  The splits and their waves take k
// in turn, U steps each, straight from memory to the matrix instructions, 16 RT ranks at a time; a
// workgroup's sums meet in LDS, the splits' in the second product.  (One workgroup a tile, of 16 waves:
// 1 x 4096 6.8 us against 3.7, 250 tokens of 64 adapters 9.3 against 4.8: a CU alone is slow to
// bring in a whole A.)  Bound by A's way from memory for few tokens an adapter; for many by x's, and
// with more ranks by A's from the L2 (4001 x 4096: rank 16 11 us, rank 48 18, rank 64 22, rank 256 75; 4001
// x 4097 of rank 48 20).
template <int DX, int DT, int RT, int U, bool ALIGNED>
__global__ __launch_bounds__(64 * kDownWaves) void k_adapter_down(const fie_adapter_args a, const AdapterWork w)
{
    using Op = Operand<DT>;
    using Tok = TokenLoad<DX, DT, ALIGNED>;
    constexpr int XS = Tok::XS;
    __shared__ f32x4_t red[kDownWaves][RT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = lane >> 4;
    if ((int)blockIdx.y >= a.plan[0]) return;
    const int32_t* tile = a.plan + kPlanHead + blockIdx.y * kPlanTile;
    const int32_t* order = a.plan + kPlanHead + (int64_t)w.most * kPlanTile;
    const int id = tile[0], first = tile[1], count = tile[2];
    if (id < 0) return;
    const int rank = min(a.ranks[id], a.rank);
    const uint8_t* const row = (const uint8_t*)a.x + (int64_t)order[first + min(lane & 15, count - 1)] * a.x_stride * XS;
    const int full = a.k / Op::STEP, steps = (a.k + Op::STEP - 1) / Op::STEP;
    for (int r0 = 0; r0 < rank; r0 += 16 * RT) {
        const uint8_t* ar[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r)
            ar[r] = (const uint8_t*)a.a + ((int64_t)id * a.rank + min(r0 + 16 * r, a.rank - 16) + (lane & 15)) * a.k_pad * Op::SIZE + 16 * group;
        f32x4_t acc[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[r] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        for (int c = (blockIdx.x * kDownWaves + wave) * U; c < steps; c += gridDim.x * kDownWaves * U) {
            if (c + U <= full) {
                u32x4_t fa[U][RT];
                Tok fx[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
#pragma unroll
                    for (int r = 0; r < RT; ++r) fa[u][r] = *(const u32x4_t*)(ar[r] + (int64_t)(c + u) * 64);
                    fx[u].load(row + ((c + u) * Op::STEP + group * Op::EACH) * XS);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const u32x4_t x = fx[u].get(row + ((c + u) * Op::STEP + group * Op::EACH) * XS);
#pragma unroll
                    for (int r = 0; r < RT; ++r) acc[r] = Op::mul(fa[u][r], x, acc[r]);
                }
            } else
#pragma unroll 1
                for (int u = c; u < min(c + U, steps); ++u) {
                    const u32x4_t x = Tok::last(row, u * Op::STEP + group * Op::EACH, a.k);
#pragma unroll
                    for (int r = 0; r < RT; ++r) acc[r] = Op::mul(*(const u32x4_t*)(ar[r] + (int64_t)u * 64), x, acc[r]);
                }
        }
        if (r0) __syncthreads();                        // the sums before are read
#pragma unroll
        for (int r = 0; r < RT; ++r) red[wave][r][lane] = acc[r];
        __syncthreads();
        for (int f = wave; f < RT; f += kDownWaves) {
            f32x4_t t = red[0][f][lane];
#pragma unroll
            for (int i = 1; i < kDownWaves; ++i) t += red[i][f][lane];
            const int r = r0 + 16 * f + 4 * group;
#pragma unroll
            for (int i = 0; i < 4; ++i) t[i] = r + i < rank ? t[i] : 0.0f;      // (ranks of padding: an infinite x times 0)
            if ((lane & 15) < count && r < a.rank) *(f32x4_t*)(w.h + ((int64_t)blockIdx.x * a.tokens + first + (lane & 15)) * a.rank + r) = t;
        }
    }
}

// One and four elements as they are in memory (four: at an address aligned to four).
template <int DT> struct Raw {
    typedef typename std::conditional<DT == FIE_F32, float, uint16_t>::type one_t;
    typedef typename std::conditional<DT == FIE_F32, f32x4_t, uint2>::type four_t;
    static FIE_DEV float value(one_t r)
    {
        if constexpr (DT == FIE_F32) return r;
        else return Operand<DT>::value(r);
    }
    static FIE_DEV void open(const four_t& r, float* v)
    {
        if constexpr (DT == FIE_F32) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = r[i];
        } else {
            v[0] = value((uint16_t)r.x);
            v[1] = value((uint16_t)(r.x >> 16));
            v[2] = value((uint16_t)r.y);
            v[3] = value((uint16_t)(r.y >> 16));
        }
    }
    static FIE_DEV one_t close(float v)
    {
        if constexpr (DT == FIE_F32) return v;
        else return (uint16_t)Operand<DT>::bits(v);
    }
    static FIE_DEV four_t close(const float* v)
    {
        if constexpr (DT == FIE_F32) return f32x4_t{v[0], v[1], v[2], v[3]};
        else return make_uint2(close(v[0]) | ((uint32_t)close(v[1]) << 16), close(v[2]) | ((uint32_t)close(v[3]) << 16));
    }
};

constexpr int kUpWaves = 4, kUpCols = 4, kUpChannels = 16 * kUpCols;

// The second product's operand of 16 ranks, for 16 tokens: a lane's numbers of its token, summed
// over the splits.  With two-byte adapters lanes of groups 0 and 1 give the leading parts of 16 ranks
// and groups 2 and 3 the trailing parts, both against the same 16 of B.
template <int DT> struct UpOperand {
    static constexpr int N = DT == FIE_F32 ? 4 : 8;
    float v[N];
    FIE_DEV void load(const float* h, int64_t part, int splits)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = 0.0f;
        for (int p = 0; p < splits; p += 4) {           // four on their way together
            f32x4_t t[4][N / 4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < N / 4; ++i) t[u][i] = *(const f32x4_t*)(h + (int64_t)min(p + u, splits - 1) * part + 4 * i);
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] += p + u < splits ? t[u][i / 4][i % 4] : 0.0f;
        }
    }
    FIE_DEV float most(float m) const
    {
#pragma unroll
        for (int i = 0; i < N; ++i) m = __builtin_fmaxf(m, __builtin_fabsf(v[i]));
        return m;
    }
    FIE_DEV u32x4_t get(int e, bool trailing) const     // times 2^e
    {
        using Op = Operand<DT>;
        u32x4_t o;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == FIE_F32) o[i] = __float_as_uint(v[i]);
            else {
                uint32_t b[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float x = DT == FIE_F16 ? __builtin_ldexpf(v[2 * i + j], e) : v[2 * i + j];
                    const uint32_t lead = Op::bits(x);
                    const float back = Op::value(lead); // (an infinity has no rest)
                    b[j] = trailing ? Op::bits(__builtin_fabsf(back) <= 3.4e38f ? x - back : 0.0f) : lead;
                }
                o[i] = b[0] | (b[1] << 16);
            }
        }
        return o;
    }
};

// y = base + scale B h: a wave a tile of 16 tokens and `steps` times 64 channels next to each other, on
// its own; the four of a workgroup take four tiles, which mostly share their B.  h stays in registers as
// the matrix instructions take it (CH times 16 ranks; CH 0: any number, built anew for each step).  fp16
// tokens are brought to an exponent of their own first, so that no part overflows or loses bits.  Results cross LDS
// within the wave, so that base and y are read and written along their rows whatever these begin at.
// Bound by base and y for many tokens an adapter (4001 x 4096, rank 16: 17 us, 4.0 TB/s; rank 48 24 and
// rank 64 37, B's way from the L2; rank 48 at 4099 channels, a channel a lane, 33), by B for few (250 x
// 16384 of 64 adapters 16 us, 18 behind the 8-bit product with its fp32 base: 3.2 TB/s).  Ranks past 64 build
// their operand anew for each 64 channels (rank 128 139 us, rank 256 266).  Held to four waves a SIMD (rank
// 48 29 us with three, two tiles a wave that share B's registers 43 with two); that leaves CH 4 with an
// fp32 base 32 bytes a lane in memory, which costs nothing to be seen (250 x 16384 at k 512, both products 41.9
// us, with a bf16 base 41.4).  B's channels at every 128 bytes cost rank 64 52 us.
template <int DT, int DY, int DB, int CH>
__global__ __launch_bounds__(64 * kUpWaves, 4) void k_adapter_up(const fie_adapter_args a, const AdapterWork w, int wide, int steps)
{
    using Op = Operand<DT>;
    using Part = UpOperand<DT>;
    constexpr int kPitch = kUpChannels + 4, HELD = CH ? CH : 1;
    __shared__ float stage[kUpWaves][16 * kPitch];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = lane >> 4, col = lane & 15;
    const int t0 = blockIdx.y * kUpWaves + wave;
    if (t0 >= a.plan[0]) return;
    const int32_t* tile = a.plan + kPlanHead + (int64_t)t0 * kPlanTile;
    const int32_t* order = a.plan + kPlanHead + (int64_t)w.most * kPlanTile;
    const int id = tile[0], first = tile[1], count = tile[2];
    const int rank = id < 0 ? 0 : min(max(a.ranks[id], 0), a.rank);
    if (rank == 0 && a.base == a.y) return;
    const int chunks = (rank + 15) / 16;
    const int place = first + min(col, count - 1), mine = order[place];
    float factor = rank ? a.scale[id] : 0.0f;
    const bool trailing = group >= 2;
    const float* const h = w.h + (int64_t)place * a.rank + (DT == FIE_F32 ? 4 * group : 8 * (group & 1));
    const int64_t part = (int64_t)a.tokens * a.rank;
    int e = 0;
    u32x4_t fh[HELD];
    if (rank) {
        if (a.x_scale) factor *= a.x_scale[mine];
        Part p[HELD];
        float most = 0.0f;
        if constexpr (CH > 0) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                if (c < chunks) p[c].load(h + 16 * c, part, w.splits);
                if (c < chunks) most = p[c].most(most);
            }
        } else if constexpr (DT == FIE_F16)
            for (int c = 0; c < chunks; ++c) {
                p[0].load(h + 16 * c, part, w.splits);
                most = p[0].most(most);
            }
        if constexpr (DT == FIE_F16) {
            most = __builtin_fmaxf(most, __shfl_xor(most, 16, 64));
            // the largest to [2^14, 2^15), so that trailing parts of numbers far below it are normal, too (with
            // it at [1, 2) one 2^-11 of the largest was off by 2^-14 of itself).  Products of fp16 numbers are
            // multiples of 2^-48 and their sums below 2^49, so factor keeps its bits
            e = most > 0.0f && most <= 3.4e38f ? 127 + 14 - (int)((__float_as_uint(most) >> 23) & 255u) : 0;
            factor = __builtin_ldexpf(factor, -e);
        }
        if constexpr (CH > 0)
#pragma unroll
            for (int c = 0; c < CH; ++c) fh[c] = c < chunks ? p[c].get(e, trailing) : u32x4_t{0, 0, 0, 0};
    }
    float* const room = stage[wave];
    const uint8_t* const b0 = (const uint8_t*)a.b + (int64_t)max(id, 0) * a.n * a.b_pitch * Op::SIZE + 16 * (DT == FIE_F32 ? group : group & 1);
    for (int s = 0; s < steps; ++s) {
        const int n0 = (blockIdx.x * steps + s) * kUpChannels;
        if (n0 >= a.n) return;
        // base first, then B: both are on their way before anything is used.  Rows past the tile's tokens
        // repeat its last one's, channels past n the last
        const bool four = wide && n0 + kUpChannels <= a.n;
        const int nw = n0 + 4 * col, nl = min(n0 + lane, a.n - 1);
        typedef typename Raw<DB>::one_t base_t;
        typedef typename Raw<DB>::four_t base4_t;
        constexpr int W = sizeof(base4_t) / 4;          // words of four
        uint32_t raw[16];                               // of either kind, in the same registers
        if (a.base) {
            if (four) {                                 // 4 channels a lane of 4 tokens
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const base4_t v = *(const base4_t*)((const base_t*)a.base + (int64_t)__shfl(mine, 4 * i + group, 64) * a.base_stride + nw);
                    __builtin_memcpy(&raw[W * i], &v, sizeof v);
                }
            } else                                      // a channel a lane of 16
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const base_t v = ((const base_t*)a.base + (int64_t)__builtin_amdgcn_readlane(mine, r) * a.base_stride)[nl];
                    if constexpr (DB == FIE_F32) raw[r] = __float_as_uint(v);
                    else raw[r] = v;
                }
        }
        if (rank) {
            f32x4_t acc[kUpCols];
#pragma unroll
            for (int q = 0; q < kUpCols; ++q) acc[q] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
            const uint8_t* br[kUpCols];
#pragma unroll
            for (int q = 0; q < kUpCols; ++q) br[q] = b0 + (int64_t)min(n0 + 16 * q + col, a.n - 1) * a.b_pitch * Op::SIZE;
            if constexpr (CH > 0) {
                constexpr int Q = CH == 4 ? 2 : kUpCols;        // blocks at a time, as far as registers go
#pragma unroll
                for (int q0 = 0; q0 < kUpCols; q0 += Q) {
                    u32x4_t fb[CH][Q];
#pragma unroll
                    for (int c = 0; c < CH; ++c)
                        if (c == 0 || c < chunks)
#pragma unroll
                            for (int q = 0; q < Q; ++q) fb[c][q] = *(const u32x4_t*)(br[q0 + q] + c * 16 * Op::SIZE);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int c = 0; c < CH; ++c)
                        if (c == 0 || c < chunks)
#pragma unroll
                            for (int q = 0; q < Q; ++q) acc[q0 + q] = Op::mul(fb[c][q], fh[c], acc[q0 + q]);
                }
            } else
                for (int c = 0; c < chunks; ++c) {
                    Part p;
                    p.load(h + 16 * c, part, w.splits);
                    const u32x4_t f = p.get(e, trailing);
#pragma unroll
                    for (int q = 0; q < kUpCols; ++q) acc[q] = Op::mul(*(const u32x4_t*)(br[q] + c * 16 * Op::SIZE), f, acc[q]);
                }
#pragma unroll
            for (int q = 0; q < kUpCols; ++q) *(f32x4_t*)&room[col * kPitch + 16 * q + 4 * group] = acc[q] * factor;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        typename Raw<DY>::one_t* const y = (typename Raw<DY>::one_t*)a.y;
        if (four) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 4 * i + group;
                const int64_t t = __shfl(mine, r, 64);
                float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if (a.base) {
                    base4_t b;
                    __builtin_memcpy(&b, &raw[W * i], sizeof b);
                    Raw<DB>::open(b, v);
                }
                if (rank) {
                    const f32x4_t d = *(const f32x4_t*)&room[r * kPitch + 4 * col];
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] += d[j];
                }
                if (r < count) *(typename Raw<DY>::four_t*)(y + t * a.y_stride + nw) = Raw<DY>::close(v);
            }
        } else
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int64_t t = __builtin_amdgcn_readlane(mine, r);
                float v = a.base ? Operand<DB>::value(raw[r]) : 0.0f;
                if (rank) v += room[r * kPitch + lane];
                if (r < count && n0 + lane < a.n) y[t * a.y_stride + n0 + lane] = Raw<DY>::close(v);
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

}  // namespace fie
