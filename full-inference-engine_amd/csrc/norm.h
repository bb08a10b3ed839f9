// Block norms (fie_block_norm): the end of one block and the norm in front of the next.
//
// A row is held in registers, 8 neighbouring elements a vector, from its loads to its
// stores; each norm costs one reduction over the row's threads (a layer norm two, its
// squares taken about the mean: sum(x^2) - n mean^2 cancels where the mean is large).  Bound
// by HBM: x, residual and gate read once, residual and y written once.  bf16 8192 x 4096 with
// norms on both sides 54 us, 268 MB at 5.0 TB/s (a copy of 2 GiB runs at 4.8); few rows are
// bound by their chain of loads, barriers and stores: 1 x 4096 3.0 us, 333 x 2050 layer norms
// 7.7, 250 x 4096 to int8 4.2.
#pragma once

#include "launchers.h"
#include "fie_ops.h"

namespace fie {

// One 16-byte group of elements [e0, e0 + EPL) of a row, those at or past `width` 0.  Where the
// row ends inside it, the row's last 16 bytes are loaded and shifted down (element by element
// this one group cost a row of 2050 as much as all others: 9.0 us for 333 of them).
template <int DT>
FIE_DEV uint4 load_row16(const char* rowp, int e0, int width)
{
    constexpr int EPL = DTy<DT>::EPL, SZ = DTy<DT>::SZ;
    if (width < EPL) return load_group<DT>(rowp, e0, width);
    // the load itself on no branch, so that all of a thread's are on their way together
    uint4 r = load16<DT>(rowp + (int64_t)min(e0, width - EPL) * SZ);
    if (e0 + EPL > width) {
        const int past = min(e0 + EPL - width, EPL);
        const u128 v = ((u128)r.w << 96) | ((u128)r.z << 64) | ((u128)r.y << 32) | r.x;
        const u128 t = past < EPL ? v >> (8 * SZ * past) : 0;
        r = make_uint4((uint32_t)t, (uint32_t)(t >> 32), (uint32_t)(t >> 64), (uint32_t)(t >> 96));
    }
    return r;
}

// 8 elements from e0 on, as loaded; those at or past `width` are 0.
template <int DT> struct Vec8 { uint4 r[DT == FIE_F32 ? 2 : 1]; };

template <int DT>
FIE_DEV Vec8<DT> load8(const char* rowp, int e0, int width)
{
    Vec8<DT> v;
    v.r[0] = load_row16<DT>(rowp, e0, width);
    if constexpr (DT == FIE_F32) v.r[1] = load_row16<DT>(rowp, e0 + 4, width);
    return v;
}

template <int DT>
FIE_DEV float get8(const Vec8<DT>& v, int e)
{
    if constexpr (DT == FIE_F32) return lane_get<DT>(v.r[e >> 2], e & 3);
    else return lane_get<DT>(v.r[0], e);
}

// 8 elements of a parameter row, in DT or in fp32.
template <int DT>
FIE_DEV void load_param(float (&w)[8], const void* p, bool f32, int e0, int width)
{
    if (DT == FIE_F32 || f32) {
        const Vec8<FIE_F32> v = load8<FIE_F32>((const char*)p, e0, width);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = get8<FIE_F32>(v, e);
    } else {
        const Vec8<DT> v = load8<DT>((const char*)p, e0, width);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = get8<DT>(v, e);
    }
}

// fp32 to 16 bits, round to nearest even (NaN stays NaN).
template <int DT>
FIE_DEV uint32_t half_bits(float v)
{
    if constexpr (DT == FIE_BF16) {
        const __bf16 h = (__bf16)v;
        return __builtin_bit_cast(uint16_t, h);
    } else {
        const _Float16 h = (_Float16)v;
        return __builtin_bit_cast(uint16_t, h);
    }
}

template <int DT>
FIE_DEV void store8(char* rowp, int e0, int width, const float (&v)[8])
{
    typedef typename Raw16<DTy<DT>::SZ>::T raw;
    if constexpr (DT == FIE_F32) {
        float* p = (float*)rowp + e0;
        if (e0 + 8 <= width) {
            *(raw*)p = raw{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
            *(raw*)(p + 4) = raw{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])};
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e0 + e < width) p[e] = v[e];
        }
    } else {
        uint16_t* p = (uint16_t*)rowp + e0;
        uint32_t h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = half_bits<DT>(v[e]);
        if (e0 + 8 <= width) {
            *(raw*)p = raw{h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16)};
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e0 + e < width) p[e] = (uint16_t)h[e];
        }
    }
}

FIE_DEV void store8_i8(char* rowp, int e0, int width, const float (&v)[8])
{
    typedef uint32_t raw __attribute__((ext_vector_type(2), aligned(1)));
    uint32_t b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = (uint32_t)(int32_t)v[e] & 0xFFu;
    if (e0 + 8 <= width) {
        *(raw*)(rowp + e0) = raw{b[0] | (b[1] << 8) | (b[2] << 16) | (b[3] << 24), b[4] | (b[5] << 8) | (b[6] << 16) | (b[7] << 24)};
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e0 + e < width) rowp[e0 + e] = (char)b[e];
    }
}

FIE_DEV float dwave_sum_f32(float x)
{
    auto step = [](float v, auto mv) { return v + __uint_as_float(mv(__float_as_uint(v))); };
    x = step(x, [](uint32_t a) { return dpp_mov<kDppXor1>(a); });
    x = step(x, [](uint32_t a) { return dpp_mov<kDppXor2>(a); });
    x = step(x, [](uint32_t a) { return dpp_mov<kDppHalfMirror>(a); });
    x = step(x, [](uint32_t a) { return dpp_mov<kDppMirror>(a); });
    const uint32_t b = __float_as_uint(x);
    return (__uint_as_float(rl(b, 0)) + __uint_as_float(rl(b, 16))) + (__uint_as_float(rl(b, 32)) + __uint_as_float(rl(b, 48)));
}

// Over a row's threads: a wave's (ONE), or the workgroup's.  `slot` is a scratch area that
// no other reduction of the row uses, so one barrier is enough.
template <bool ONE>
FIE_DEV float row_sum(float x, float* slot)
{
    x = dwave_sum_f32(x);
    if (ONE) return x;
    const int waves = blockDim.x >> 6;
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = x;
    __syncthreads();
    float t = 0.0f;
    for (int w = 0; w < waves; ++w) t += slot[w];
    return t;
}

// The largest |v|, by bits: those of values >= 0 order them, and NaN's lie past infinity's, so that
// a row with a NaN gives NaN (a float maximum drops it).
FIE_DEV uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

template <bool ONE>
FIE_DEV float row_max(uint32_t x, float* slot)
{
    x = dwave_max_u32(x);
    if (ONE) return __uint_as_float(x);
    const int waves = blockDim.x >> 6;
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = __uint_as_float(x);
    __syncthreads();
    uint32_t t = 0;
    for (int w = 0; w < waves; ++w) t = max(t, __float_as_uint(slot[w]));
    return __uint_as_float(t);
}

// v / s in whole numbers, by IEEE quotients: what a plain x / (max|x| / 127) rounds to.
FIE_DEV void quantise8(float (&q)[8], const float (&v)[8], float s)
{
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float u = __builtin_rintf(v[e] / s);
        // 0 in rows without a scale (0) or with a NaN (its scale), and for inf / inf; past 127
        // where s is a few denormal units, rounded down
        q[e] = s > 0.0f && u == u ? __builtin_fminf(__builtin_fmaxf(u, -127.0f), 127.0f) : 0.0f;
    }
}

// DX: x and y; DR: residual.  A row's thread t holds vectors t, t + T, ..: VPT of them, 0 past
// the row's end (where parameters load as 0, and a weight's offset meets a 0).
// ONE: a wave a row, four rows a workgroup.
// EARLY: every load at once, parameters in DX (a wave's chain is the kernel's time for few tokens).
template <int DX, int DR, int VPT, bool ONE, bool EARLY>
__global__ __launch_bounds__(ONE ? 256 : (VPT > 2 ? 1024 : 512)) void k_norm(const fie_norm_args a)
{
    __shared__ float red[5][16];
    const int T = ONE ? 64 : blockDim.x;
    const int t = ONE ? threadIdx.x & 63 : threadIdx.x;
    const int64_t row = ONE ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : (int64_t)blockIdx.x;
    if (ONE && row >= a.tokens) return;
    const int H = a.width;
    const float inv = 1.0f / (float)H;
    constexpr int SX = DTy<DX>::SZ, SR = DTy<DR>::SZ;
    const char* xp = (const char*)a.x + row * a.x_stride * SX;
    const char* rp = (const char*)a.residual + row * a.residual_stride * SR;
    const char* gp = (const char*)a.gate + row * a.gate_stride * (a.gate_f32 ? 4 : SX);

    float v[VPT][8];
    Vec8<DR> res[VPT];
    Vec8<DX> xs[VPT];
    constexpr int PN = EARLY ? VPT : 1;
    Vec8<DX> pw[PN], pb[PN], gt[PN], nw[PN], nb[PN];
    const bool wf = a.weight_f32, gf = a.gate_f32, gate_row = a.gate && a.gate_step;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int e0 = (i * T + t) * 8;
        res[i] = load8<DR>(rp, e0, H);
        if (a.x) xs[i] = load8<DX>(xp, e0, H);
        if constexpr (EARLY) {
            if (a.post_weight) pw[i] = load8<DX>((const char*)a.post_weight, e0, H);
            if (a.post_bias) pb[i] = load8<DX>((const char*)a.post_bias, e0, H);
            if (gate_row) gt[i] = load8<DX>(gp, e0, H);
            if (a.weight) nw[i] = load8<DX>((const char*)a.weight, e0, H);
            if (a.bias) nb[i] = load8<DX>((const char*)a.bias, e0, H);
        }
    }
    float g1 = 1.0f;
    if (a.gate && !a.gate_step) g1 = DX == FIE_F32 || gf ? *(const float*)gp : load_elem<DX>(gp, 0);
    // (v - mean) / sqrt(mean((v - mean)^2) + eps) * weight + bias, in place
    auto param = [&](float (&w)[8], const void* p, bool f32, const Vec8<DX>& early, int e0) {
        if constexpr (EARLY) {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = get8<DX>(early, e);
        } else {
            load_param<DX>(w, p, f32, e0, H);
        }
    };
    auto norm = [&](const void* weight, const void* bias, const Vec8<DX> (&ew)[PN], const Vec8<DX> (&eb)[PN], int slot) {
        if (a.kind == FIE_NORM_LAYER) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < VPT; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) s += v[i][e];
            const float mean = row_sum<ONE>(s, red[slot]) * inv;
#pragma unroll
            for (int i = 0; i < VPT; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[i][e] = (i * T + t) * 8 + e < H ? v[i][e] - mean : 0.0f;
        }
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) s += v[i][e] * v[i][e];
        const float rstd = 1.0f / __builtin_sqrtf(row_sum<ONE>(s, red[slot + 1]) * inv + a.eps);
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int e0 = (i * T + t) * 8;
            float w[8], b[8];
            if (weight) param(w, weight, wf, ew[EARLY ? i : 0], e0);
            if (bias) param(b, bias, wf, eb[EARLY ? i : 0], e0);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[i][e] *= rstd;
                if (weight) v[i][e] *= w[e] + a.weight_offset;
                if (bias) v[i][e] += b[e];
            }
        }
    };
    if (a.x) {
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = get8<DX>(xs[i], e);
        if (a.post_norm) norm(a.post_weight, a.post_bias, pw, pb, 0);
        if (a.gate) {
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                float g[8];
                if (gate_row) param(g, gp, gf, gt[EARLY ? i : 0], (i * T + t) * 8);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] *= gate_row ? g[e] : g1;
            }
        }
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = get8<DR>(res[i], e) + a.scale * v[i][e];
    } else {
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = get8<DR>(res[i], e);
    }
    if (a.residual_out) {
        char* op = (char*)a.residual_out + row * a.residual_out_stride * SR;
#pragma unroll
        for (int i = 0; i < VPT; ++i) store8<DR>(op, (i * T + t) * 8, H, v[i]);
    }
    if (!a.y) return;
    if (a.kind != FIE_NORM_NONE) norm(a.weight, a.bias, nw, nb, 2);
    if (a.y_dtype != FIE_I8) {
        char* yp = (char*)a.y + row * a.y_stride * SX;
#pragma unroll
        for (int i = 0; i < VPT; ++i) store8<DX>(yp, (i * T + t) * 8, H, v[i]);
        return;
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max(m, abs_bits(v[i][e]));
    const float s = row_max<ONE>(m, red[4]) / 127.0f;
    if (t == 0) a.y_scale[row] = s;
    char* yp = (char*)a.y + row * a.y_stride;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        float q[8];
        quantise8(q, v[i], s);
        store8_i8(yp, (i * T + t) * 8, H, q);
    }
}

// A row wider than the registers of a workgroup, to int8 and nothing else: twice over it (the rows on
// their way at a time, 256 of 0.26 MB, are past the L2 but not past the cache behind it).  bf16
// 4096 x 131064 446 us, 1.6 GB read and written once at 3.6 TB/s; 250 x 131071 35 us, one row 25 (the chain of 32 loads a thread).
template <int DR>
__global__ __launch_bounds__(1024) void k_quantise_wide(const fie_norm_args a)
{
    __shared__ float red[16];
    const int64_t row = blockIdx.x;
    const int H = a.width;
    const char* rp = (const char*)a.residual + row * a.residual_stride * DTy<DR>::SZ;
    uint32_t m = 0;
    for (int e0 = threadIdx.x * 8; e0 < H; e0 += 8 * 1024) {
        const Vec8<DR> r = load8<DR>(rp, e0, H);
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max(m, abs_bits(get8<DR>(r, e)));
    }
    const float s = row_max<false>(m, red) / 127.0f;
    if (threadIdx.x == 0) a.y_scale[row] = s;
    char* yp = (char*)a.y + row * a.y_stride;
    for (int e0 = threadIdx.x * 8; e0 < H; e0 += 8 * 1024) {
        const Vec8<DR> r = load8<DR>(rp, e0, H);
        float v[8], q[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = get8<DR>(r, e);
        quantise8(q, v, s);
        store8_i8(yp, e0, H, q);
    }
}

}  // namespace fie
