// The norms around a transformer block, with the block's gate, residual scale and residual sum between
// them, in one launch, and their backward pass in one launch plus a small sum over workgroups:
//
//   z = N_post(y) * w_post + b_post      h = x + scale * gate * z      n = N_pre(h) * w_pre + b_pre
//
// N: over the channels of a column (b, t), (v - mean) * rstd (layer) or v * rstd (rms), rstd = 1 / sqrt(mean of
// squares + eps).  Tensors are [B, C, T] with dense time, so a norm runs across rows T apart: a workgroup owns a
// window of TW columns with all their channels and keeps every value it read in registers - one pass over
// memory, the statistics need no second one.  Lanes lie along time (one 16-byte access per lane and row), the
// channels are spread over the other lanes and the waves; column sums meet through LDS.
// Bound by memory: forward reads x, y, gate and writes h, n; backward reads dh, dn, h, y, gate, writes dx, dy, dgate.
// fp32, 32 x 256 x 2048: 75 us (4.5 TB/s), backward 136 us (3.9 TB/s).  bf16, 8 x 1024 x 4096, gate per item: 93 us (2.9 TB/s);
// 8 x up to 2047 x 1024 backward 130 us (1.6 TB/s): that many channels leave one workgroup per CU, whose loads and
// arithmetic alternate (and spill: 16 to 18 registers with eight rows per thread).
#include <hip/hip_runtime.h>
#include <atomic>
#include <stdint.h>
#include <stdio.h>
#include <string.h>
#include "../../include/vits_amd.h"
#include "api_internal.hpp"
#include "chunk_load.hpp"
#include "conv_mfma.hpp"      // vk_allow_lds

namespace {

typedef chunk_t u32x4;

struct NDev {
    vk_block_norm_args a;
    int windows;            // windows of an item
    float* part;            // backward: parameter gradient sums of every workgroup [workgroups][5][C]
    float* part_gate;       // backward, gate per item: [B][windows][C]
};

template <typename T> struct Pack { static constexpr int E = 16 / (int)sizeof(T); };

__device__ __forceinline__ void unpack(float (&v)[4], const u32x4& r)
{
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(r[e]);
}
__device__ __forceinline__ void unpack(float (&v)[8], const u32x4& r)      // bf16 is the upper half of an fp32
{
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[2 * e] = __uint_as_float(r[e] << 16);
        v[2 * e + 1] = __uint_as_float(r[e] & 0xffff0000u);
    }
}
// Keeps the compiler from holding the unpacked values of a row between two uses: twice the registers in bf16.
__device__ __forceinline__ void keep_packed(u32x4& r) { asm volatile("" : "+v"(r[0]), "+v"(r[1]), "+v"(r[2]), "+v"(r[3])); }

template <int CTRL>
__device__ __forceinline__ float dpp(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true)); }

// Sum over the lanes of a wave that sit LT apart (LT <= 8): rotations within 16 lanes, then across.
template <int LT>
__device__ __forceinline__ float sum_apart(float v)
{
    v += dpp<0x128>(v);                                     // rotate 16 lanes by 8
    if constexpr (LT <= 4) v += dpp<0x124>(v);
    if constexpr (LT <= 2) v += dpp<0x122>(v);
    if constexpr (LT <= 1) v += dpp<0x121>(v);
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}
// Sum over LT neighbouring lanes: within four, then a mirror of eight.
template <int LT>
__device__ __forceinline__ float sum_near(float v)
{
    if constexpr (LT >= 2) v += dpp<0xb1>(v);
    if constexpr (LT >= 4) v += dpp<0x4e>(v);
    if constexpr (LT >= 8) v += dpp<0x141>(v);
    return v;
}

// Sum over the channel groups of a workgroup, for every column.
template <int LT, int E, int NW>
__device__ __forceinline__ void column_sum(float (&v)[E], float* red)
{
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, lt = lane % LT;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = sum_apart<LT>(v[e]);
    __syncthreads();                                        // the previous sum has been read
    if (lane < LT)
#pragma unroll
        for (int e = 0; e < E; ++e) red[(wave * LT + lt) * E + e] = v[e];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.0f;
#pragma unroll 2                                            // all NW * E reads at once would take as many registers
    for (int w = 0; w < NW; ++w)
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] += red[(w * LT + lt) * E + e];
}

// Per column: mean (0 for rms) and 1 / sqrt(mean square about it + eps) of rows value(r, v), r < rows.  Two sweeps
// over the registers, so the variance is a sum of squares about the mean.
template <int LT, int E, int NW, int R, typename F>
__device__ __forceinline__ void column_stats(F value, int rows, int channels, float eps, bool layer, float* red,
                                             float (&mean)[E], float (&rstd)[E])
{
    const float inv = 1.0f / (float)channels;
    float sum[E];
#pragma unroll
    for (int e = 0; e < E; ++e) mean[e] = sum[e] = 0.0f;
    if (layer) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float v[E];
            value(r, v);
#pragma unroll
            for (int e = 0; e < E; ++e) mean[e] += r < rows ? v[e] : 0.0f;
        }
        column_sum<LT, E, NW>(mean, red);
#pragma unroll
        for (int e = 0; e < E; ++e) mean[e] *= inv;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float v[E];
        value(r, v);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float d = v[e] - mean[e];
            sum[e] = r < rows ? fmaf(d, d, sum[e]) : sum[e];
        }
    }
    column_sum<LT, E, NW>(sum, red);
#pragma unroll
    for (int e = 0; e < E; ++e) rstd[e] = 1.0f / sqrtf(fmaf(sum[e], inv, eps));
}

// Where a thread works: channels cg, cg + CG, .. (`rows` of them), columns t .. t + E - 1 of item b, of which those
// before `live` count.  LT lanes along time, the other lanes and the waves along the channels.  An address is the
// item's base (uniform) and a 32-bit offset, which the rows of a thread share but for a uniform part.
template <typename T, int LT, int NW>
struct Spot {
    static constexpr int E = Pack<T>::E, CG = 64 / LT * NW;
    int cg, rows, b, t, live, length, lt, channels, id;
    bool any, inside, tiny;         // a window at all; all of it live; rows shorter than a chunk
    int at, moved;                  // where this thread's chunks are read, and how far that is before t
    u32x4 keep;                     // the live columns as bits, where not all are
    __device__ __forceinline__ Spot(const NDev& p)
    {
        const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
        lt = lane % LT;
        cg = wave * (64 / LT) + lane / LT;
        // neighbouring windows share cache lines at their borders (and, narrower than a line, everywhere): they go to
        // one XCD, which takes every eighth workgroup
        const int n = p.a.batch * p.windows, per = (n + 7) >> 3;
        id = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
        any = ((int)blockIdx.x >> 3) < per && id < n;
        b = id / p.windows;
        const int t0 = (id - b * p.windows) * LT * E;
        t = t0 + lt * E;
        channels = p.a.channels;
        live = length = p.a.length;
        if (p.a.lengths && any) { const int64_t m = p.a.lengths[b]; live = __builtin_amdgcn_readfirstlane((int)(m < 0 ? 0 : m > length ? length : m)); }
        rows = cg < channels ? (channels - cg + CG - 1) / CG : 0;
        inside = t0 + LT * E <= live;
        tiny = length < E;
        at = min(t, max(length - E, 0));
        moved = min(t - at, E);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (E == 4) keep[j] = t + j < live ? 0xffffffffu : 0u;
            else keep[j] = (t + 2 * j < live ? 0xffffu : 0u) | (t + 2 * j + 1 < live ? 0xffff0000u : 0u);
        }
    }
    // Threads without a channel take their first (or channel 0) again and store nothing: no branches around the loads.
    __device__ __forceinline__ int channel(int r) const { return r < rows ? cg + r * CG : rows ? cg : 0; }
    // Byte offset of row r at column `col`.  Computed where it is used: held for all rows and tensors, the offsets
    // would take more registers than the data.
    __device__ __forceinline__ unsigned offset(int64_t cstride, int col, int r) const
    {
        unsigned o = ((unsigned)(rows ? cg : 0) * (unsigned)cstride + (unsigned)col) * (unsigned)sizeof(T);
        asm volatile("" : "+v"(o));
        return r < rows ? o + (unsigned)r * (unsigned)CG * (unsigned)cstride * (unsigned)sizeof(T) : o;
    }
    __device__ __forceinline__ u32x4 load_row(const void* base, int64_t bstride, int64_t cstride, int r) const
    {
        const char* row = (const char*)((const T*)base + (int64_t)b * bstride);
        const unsigned off = offset(cstride, at, r);
        u32x4 c;
        if (tiny) {
            unsigned long long v[2] = {0, 0};
#pragma unroll 1
            for (int e = 0; e < length; ++e) {
                const T x = *(const T*)(row + off + e * sizeof(T));
                unsigned bits = 0;
                __builtin_memcpy(&bits, &x, sizeof(T));
                const int pos = e * 8 * (int)sizeof(T);
                v[0] |= pos < 64 ? (unsigned long long)bits << pos : 0;
                v[1] |= pos >= 64 ? (unsigned long long)bits << (pos - 64) : 0;
            }
            c = u32x4{(unsigned)v[0], (unsigned)(v[0] >> 32), (unsigned)v[1], (unsigned)(v[1] >> 32)};
        } else {
            __builtin_memcpy(&c, row + off, 16);
        }
        if (!inside) c = chunk_shift<E>(c, moved) & keep;
        return c;
    }
    template <int R>
    __device__ __forceinline__ void load(u32x4 (&v)[R], const void* base, int64_t bstride, int64_t cstride) const
    {
#pragma unroll
        for (int r = 0; r < R; ++r) v[r] = load_row(base, bstride, cstride, r);
    }
    __device__ __forceinline__ void store_row(void* base, int64_t bstride, int64_t cstride, int r, const float (&v)[E]) const
    {
        if (r >= rows) return;
        char* row = (char*)((T*)base + (int64_t)b * bstride);
        const unsigned off = offset(cstride, t, r);
        T tmp[E];
#pragma unroll
        for (int e = 0; e < E; ++e) tmp[e] = (T)v[e];
        u32x4 c;
        __builtin_memcpy(&c, tmp, 16);
        if (!inside) c &= keep;
        if (inside || t + E <= length) {
            __builtin_memcpy(row + off, &c, 16);
        } else {
            unsigned long long q[2] = {c[0] | (unsigned long long)c[1] << 32, c[2] | (unsigned long long)c[3] << 32};
#pragma unroll 1
            for (int e = 0; e < length - t; ++e) {
                const int pos = e * 8 * (int)sizeof(T);
                const unsigned bits = (unsigned)(pos < 64 ? q[0] >> pos : q[1] >> (pos - 64));
                __builtin_memcpy(row + off + e * sizeof(T), &bits, sizeof(T));
            }
        }
    }
};

// The per-channel numbers of a pass in LDS: ones and zeros where something is not given.  An item without live columns has
// no part in any sum, so its gate does not either: a NaN there (a mean over no columns) times its zeros would.
enum { P_SCALE, P_GATE, P_WPOST, P_BPOST, P_WPRE, P_BPRE, P_COUNT };
template <typename T>
__device__ __forceinline__ void stage_params(float* par, const vk_block_norm_args& a, int b, int live)
{
    const bool item = a.gate && a.gate_per_item && live > 0;
    const float* src[P_COUNT] = {a.scale, nullptr, a.w_post, a.b_post, a.w_pre, a.b_pre};
    for (int c = (int)threadIdx.x; c < a.channels; c += (int)blockDim.x) {
#pragma unroll
        for (int i = 0; i < P_COUNT; ++i)
            if (i != P_GATE) par[i * a.channels + c] = src[i] ? src[i][c] : (i == P_BPOST || i == P_BPRE) ? 0.0f : 1.0f;
        par[P_GATE * a.channels + c] = item ? (float)((const T*)a.gate)[(int64_t)b * a.gate_bstride + (int64_t)c * a.gate_cstride] : 1.0f;
    }
}

template <typename T, int LT, int NW, int R>
__global__ __launch_bounds__(64 * NW)
void block_norm_kernel(NDev p)
{
    using S = Spot<T, LT, NW>;
    constexpr int E = S::E;
    extern __shared__ __align__(16) float lds[];
    float* red = lds;
    float* par = lds + NW * LT * E;
    const vk_block_norm_args& a = p.a;
    const S at(p);
    if (!at.any) return;
    const int C = a.channels;
    const bool layer = a.norm == VK_NORM_LAYER, full_gate = a.gate && !a.gate_per_item;
    u32x4 xr[R], yr[R];
    if (a.y) at.load(yr, a.y, a.y_bstride, a.y_cstride);
    at.load(xr, a.x, a.x_bstride, a.x_cstride);
    stage_params<T>(par, a, at.b, at.live);
    __syncthreads();
    float h[R][E];
    if (a.y) {
        float mean[E], rstd[E];
        if (a.w_post) column_stats<LT, E, NW, R>([&](int r, float (&v)[E]) { unpack(v, yr[r]); keep_packed(yr[r]); }, at.rows, C, a.eps, layer, red, mean, rstd);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float* q = par + at.channel(r);
            const float s = q[P_SCALE * C] * q[P_GATE * C], w = q[P_WPOST * C], bias = q[P_BPOST * C];
            float g[E], z[E];
            if (full_gate) unpack(g, at.load_row(a.gate, a.gate_bstride, a.gate_cstride, r));
            unpack(z, yr[r]);
            unpack(h[r], xr[r]);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (a.w_post) z[e] = fmaf((z[e] - mean[e]) * rstd[e], w, bias);
                h[r][e] = fmaf(full_gate ? g[e] * s : s, z[e], h[r][e]);
            }
        }
    } else {
#pragma unroll
        for (int r = 0; r < R; ++r) unpack(h[r], xr[r]);
    }
    if (a.h)
#pragma unroll
        for (int r = 0; r < R; ++r) at.store_row(a.h, a.h_bstride, a.h_cstride, r, h[r]);
    if (!a.n) return;
    float mean[E], rstd[E];
    column_stats<LT, E, NW, R>([&](int r, float (&v)[E]) {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = h[r][e]; }, at.rows, C, a.eps, layer, red, mean, rstd);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float* q = par + at.channel(r);
        const float w = q[P_WPRE * C], bias = q[P_BPRE * C];
        float o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf((h[r][e] - mean[e]) * rstd[e], w, bias);
        at.store_row(a.n, a.n_bstride, a.n_cstride, r, o);
    }
}

// Gradient through a norm: g -> (g - mean(g) - vhat * mean(g * vhat)) * rstd (layer; without mean(g) for rms).
//
// The gradient of h stays in registers in fp32 from the norm before the next block to the norm after this one.
// Parameter gradients are sums over the columns of a row: over the lanes of a column group, then one number per
// row and workgroup goes to memory, and a second kernel adds the workgroups in a fixed order.
template <typename T, int LT, int NW, int R>
__global__ __launch_bounds__(64 * NW)
void block_norm_backward_kernel(NDev p)
{
    using S = Spot<T, LT, NW>;
    constexpr int E = S::E;
    extern __shared__ __align__(16) float lds[];
    float* red = lds;
    float* par = lds + NW * LT * E;
    const vk_block_norm_args& a = p.a;
    const S at(p);
    if (!at.any) return;
    const int C = a.channels;
    const bool layer = a.norm == VK_NORM_LAYER, full_gate = a.gate && !a.gate_per_item, item_gate = a.dgate && a.gate_per_item;
    const float inv = 1.0f / (float)C;
    float* part = p.part + (int64_t)at.id * 5 * C;
    auto over_columns = [&](const float (&x)[E]) {
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) s += x[e];
        return sum_near<LT>(s);
    };

    float g[R][E];              // gradient of h, then of z
    if (a.dn) {
        u32x4 hr[R], dr[R];
        at.load(hr, a.h, a.h_bstride, a.h_cstride);
        at.load(dr, a.dn, a.dn_bstride, a.dn_cstride);
        stage_params<T>(par, a, at.b, at.live);
        __syncthreads();
        float mean[E], rstd[E], m1[E], m2[E];
        column_stats<LT, E, NW, R>([&](int r, float (&v)[E]) { unpack(v, hr[r]); keep_packed(hr[r]); }, at.rows, C, a.eps, layer, red, mean, rstd);
#pragma unroll
        for (int e = 0; e < E; ++e) m1[e] = m2[e] = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = at.channel(r);
            const float w = r < at.rows ? par[P_WPRE * C + c] : 0.0f;       // a repeated channel counts once
            float v[E], d[E], dw[E];
            unpack(v, hr[r]);
            unpack(d, dr[r]);
            keep_packed(hr[r]);
            keep_packed(dr[r]);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                dw[e] = d[e] * ((v[e] - mean[e]) * rstd[e]);
                m1[e] = fmaf(d[e], w, m1[e]);
                m2[e] = fmaf(dw[e], w, m2[e]);
            }
            const float sw = over_columns(dw), sb = over_columns(d);
            if (at.lt == 0 && r < at.rows) { part[c] = sw; part[C + c] = sb; }
        }
        if (layer) column_sum<LT, E, NW>(m1, red);
        column_sum<LT, E, NW>(m2, red);
#pragma unroll
        for (int e = 0; e < E; ++e) { m1[e] = layer ? m1[e] * inv : 0.0f; m2[e] *= inv; }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float w = par[P_WPRE * C + at.channel(r)];
            float v[E], d[E];
            unpack(v, hr[r]);
            unpack(d, dr[r]);
#pragma unroll
            for (int e = 0; e < E; ++e) g[r][e] = (fmaf(d[e], w, -m1[e]) - (v[e] - mean[e]) * rstd[e] * m2[e]) * rstd[e];
        }
    } else {
        stage_params<T>(par, a, at.b, at.live);
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < E; ++e) g[r][e] = 0.0f;
    }
    if (a.dh)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float d[E];
            unpack(d, at.load_row(a.dh, a.dh_bstride, a.dh_cstride, r));
#pragma unroll
            for (int e = 0; e < E; ++e) g[r][e] += d[e];
        }
    u32x4 yr[R];
    if (a.y) at.load(yr, a.y, a.y_bstride, a.y_cstride);
#pragma unroll
    for (int r = 0; r < R; ++r) at.store_row(a.dx, a.dx_bstride, a.dx_cstride, r, g[r]);
    if (!a.y) return;

    float mean[E], rstd[E], m1[E], m2[E];
    if (a.w_post) column_stats<LT, E, NW, R>([&](int r, float (&v)[E]) { unpack(v, yr[r]); keep_packed(yr[r]); }, at.rows, C, a.eps, layer, red, mean, rstd);
#pragma unroll
    for (int e = 0; e < E; ++e) m1[e] = m2[e] = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int c = at.channel(r);
        const float* q = par + c;
        const float s = q[P_SCALE * C], w = q[P_WPOST * C], bias = q[P_BPOST * C], gi = q[P_GATE * C];
        float gate[E], dg[E], ds[E], dw[E], v[E];
        if (full_gate) unpack(gate, at.load_row(a.gate, a.gate_bstride, a.gate_cstride, r));
        unpack(v, yr[r]);
        keep_packed(yr[r]);
        const float wm = r < at.rows ? w : 0.0f;        // a repeated channel counts once
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float ge = full_gate ? gate[e] : gi;
            if (a.w_post) v[e] = (v[e] - mean[e]) * rstd[e];
            const float z = a.w_post ? fmaf(v[e], w, bias) : v[e];
            dg[e] = g[r][e] * s * z;                    // gradient of the gate
            ds[e] = g[r][e] * ge * z;                   // of the scale
            g[r][e] *= s * ge;                          // of z
            dw[e] = g[r][e] * v[e];                     // of the weight
            m1[e] = fmaf(g[r][e], wm, m1[e]);
            m2[e] = fmaf(dw[e], wm, m2[e]);
        }
        if (a.dgate && full_gate) at.store_row(a.dgate, a.dgate_bstride, a.dgate_cstride, r, dg);
        const float sg = item_gate ? over_columns(dg) : 0.0f;
        const float ss = over_columns(ds), sw = over_columns(dw), sb = over_columns(g[r]);
        if (at.lt == 0 && r < at.rows) {
            part[2 * C + c] = ss;
            part[3 * C + c] = sw;
            part[4 * C + c] = sb;
            if (item_gate) p.part_gate[(int64_t)at.id * C + c] = sg;
        }
    }
    if (a.w_post) {
        if (layer) column_sum<LT, E, NW>(m1, red);
        column_sum<LT, E, NW>(m2, red);
#pragma unroll
        for (int e = 0; e < E; ++e) { m1[e] = layer ? m1[e] * inv : 0.0f; m2[e] *= inv; }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (a.w_post) {
            const float w = par[P_WPOST * C + at.channel(r)];
            float v[E];
            unpack(v, yr[r]);
#pragma unroll
            for (int e = 0; e < E; ++e) g[r][e] = (fmaf(g[r][e], w, -m1[e]) - (v[e] - mean[e]) * rstd[e] * m2[e]) * rstd[e];
        }
        at.store_row(a.dy, a.dy_bstride, a.dy_cstride, r, g[r]);
    }
}

// Sums over the workgroups: blockIdx.y 0..4 a parameter's gradient, 5.. the gate of item blockIdx.y - 5.
constexpr int SUM_C = 32, SUM_P = 32;
template <typename T>
__global__ __launch_bounds__(SUM_C * SUM_P)
void block_norm_sums_kernel(NDev p)
{
    __shared__ float acc[SUM_P][SUM_C];
    const vk_block_norm_args& a = p.a;
    const int which = (int)blockIdx.y, c = (int)blockIdx.x * SUM_C + (int)threadIdx.x % SUM_C, q = (int)threadIdx.x / SUM_C;
    float* outs[5] = {a.dw_pre, a.db_pre, a.dscale, a.dw_post, a.db_post};
    if (which < 5 && !outs[which]) return;
    const int64_t stride = which < 5 ? 5 * (int64_t)a.channels : a.channels;
    const int n = which < 5 ? a.batch * p.windows : p.windows;
    const float* src = which < 5 ? p.part + (int64_t)which * a.channels : p.part_gate + (int64_t)(which - 5) * p.windows * a.channels;
    float s = 0.0f;
    if (c < a.channels)
#pragma unroll 4
        for (int i = q; i < n; i += SUM_P) s += src[i * stride + c];
    acc[q][threadIdx.x % SUM_C] = s;
    __syncthreads();
    if (q || c >= a.channels) return;
    for (int i = 1; i < SUM_P; ++i) s += acc[i][threadIdx.x % SUM_C];
    if (which < 5) outs[which][c] = s;
    else ((T*)a.dgate)[(int64_t)(which - 5) * a.dgate_bstride + (int64_t)c * a.dgate_cstride] = (T)s;
}

int fail(int code, const char* what, const char* msg)
{
    char buf[256];
    snprintf(buf, sizeof(buf), "%s: %s", what, msg);
    return vk_fail(code, buf);
}

// Rows of one item are addressed with 32-bit offsets.
bool item_fits(const void* p, int64_t cstride, const vk_block_norm_args* a)
{
    return !p || ((int64_t)(a->channels - 1) * cstride + a->length) * 4 < (int64_t)1 << 32;
}

bool strides_ok(const void* p, int64_t bstride, int64_t cstride) { return !p || vk_strides_ok(bstride, cstride); }

bool rows_apart(int64_t bstride, int64_t cstride, const vk_block_norm_args* a)
{
    return vk_rows_apart(bstride, cstride, a->channels, a->length, a->batch);
}

// What a workspace depends on.
int check_sizes(const vk_block_norm_args* a, const char* what)
{
    if (!a) return fail(VK_E_ARG, what, "null argument struct");
    if (a->batch < 0 || a->channels <= 0 || a->length < 0) return fail(VK_E_ARG, what, "bad size");
    if (a->dtype != VK_DTYPE_F32 && a->dtype != VK_DTYPE_BF16) return fail(VK_E_UNSUPPORTED, what, "dtype must be VK_DTYPE_F32 or VK_DTYPE_BF16");
    if (a->channels > VK_BLOCK_NORM_MAX_CHANNELS) return fail(VK_E_UNSUPPORTED, what, "more than VK_BLOCK_NORM_MAX_CHANNELS channels");
    if (a->length > (1 << 28)) return fail(VK_E_UNSUPPORTED, what, "length beyond 2^28");
    return VK_OK;
}

int check(const vk_block_norm_args* a, const char* what, bool backward)
{
    const int rc = check_sizes(a, what);
    if (rc != VK_OK) return rc;
    if (a->norm != VK_NORM_LAYER && a->norm != VK_NORM_RMS) return fail(VK_E_ARG, what, "norm must be VK_NORM_LAYER or VK_NORM_RMS");
    if (!(a->eps > 0.0f && a->eps < 1e30f)) return fail(VK_E_ARG, what, "eps must be positive and finite");
    const bool some = a->batch > 0 && a->length > 0;
    if (some && !a->y && (a->gate || a->scale || a->w_post)) return fail(VK_E_ARG, what, "gate, scale and the norm after the block need y");
    if ((!a->w_post && a->b_post) || (!a->w_pre && a->b_pre)) return fail(VK_E_ARG, what, "a norm's bias needs its weight");
    if (!strides_ok(a->x, a->x_bstride, a->x_cstride) || !strides_ok(a->y, a->y_bstride, a->y_cstride)
        || !strides_ok(a->gate, a->gate_bstride, a->gate_cstride) || !strides_ok(a->h, a->h_bstride, a->h_cstride)
        || !strides_ok(a->n, a->n_bstride, a->n_cstride) || !strides_ok(a->dh, a->dh_bstride, a->dh_cstride)
        || !strides_ok(a->dn, a->dn_bstride, a->dn_cstride) || !strides_ok(a->dx, a->dx_bstride, a->dx_cstride)
        || !strides_ok(a->dy, a->dy_bstride, a->dy_cstride) || !strides_ok(a->dgate, a->dgate_bstride, a->dgate_cstride))
        return fail(VK_E_ARG, what, "a stride is negative or beyond 2^40");
    if (!item_fits(a->x, a->x_cstride, a) || !item_fits(a->y, a->y_cstride, a) || !item_fits(a->h, a->h_cstride, a)
        || !item_fits(a->n, a->n_cstride, a) || !item_fits(a->dh, a->dh_cstride, a) || !item_fits(a->dn, a->dn_cstride, a)
        || !item_fits(a->dx, a->dx_cstride, a) || !item_fits(a->dy, a->dy_cstride, a)
        || (!a->gate_per_item && (!item_fits(a->gate, a->gate_cstride, a) || !item_fits(a->dgate, a->dgate_cstride, a))))
        return fail(VK_E_UNSUPPORTED, what, "an item's view spans 2^30 elements or more");
    if (!backward) {
        if (some && (!a->x || (!a->h && !a->n))) return fail(VK_E_ARG, what, "null x, or nothing to write");
        if (some && a->n && !a->w_pre) return fail(VK_E_ARG, what, "n needs w_pre");
        if ((a->h && !rows_apart(a->h_bstride, a->h_cstride, a)) || (a->n && !rows_apart(a->n_bstride, a->n_cstride, a)))
            return fail(VK_E_ARG, what, "rows of an output overlap");
    } else {
        if (some && (!a->dx || (a->y && !a->dy) || (!a->dh && !a->dn))) return fail(VK_E_ARG, what, "null dx or dy, or no gradient came in");
        if (some && a->dn && (!a->w_pre || !a->h)) return fail(VK_E_ARG, what, "dn needs h and w_pre");
        if ((a->dgate && !a->gate) || (a->dscale && !a->scale) || ((a->dw_post || a->db_post) && !a->w_post)
            || ((a->dw_pre || a->db_pre) && !a->w_pre))
            return fail(VK_E_ARG, what, "a gradient of something that was not given");
        if (some && (a->dw_pre || a->db_pre) && !a->dn) return fail(VK_E_ARG, what, "the gradients of w_pre and b_pre need dn");
        if ((a->dx && !rows_apart(a->dx_bstride, a->dx_cstride, a)) || (a->dy && !rows_apart(a->dy_bstride, a->dy_cstride, a))
            || (a->dgate && !a->gate_per_item && !rows_apart(a->dgate_bstride, a->dgate_cstride, a)))
            return fail(VK_E_ARG, what, "rows of an output overlap");
    }
    return VK_OK;
}

// A workgroup's window: LT lanes of 16 bytes along time, NW waves, R channels per thread, so (64 / LT) * NW * R
// channels.  Eight lanes make 128-byte accesses, a whole cache line; narrower windows hold more channels and
// make more workgroups.  Few channels per thread keep several workgroups on a CU, so that one loads while another computes:
// eight waves of four rather than four of eight (fp32 backward, 32 x 256 x 2048: 136 us against 144; 64 x 192 x 862: 99,
// 113), and in bf16, whose lanes hold eight columns, 129..256 channels in half as wide windows (160 channels, 16 x 4095:
// 79 us against 84 and, with four waves of eight, 112; in fp32 not: 32 x 256 x 2048 150 against 136; nor from 512 channels on,
// where rows of 32 bytes cost more than they gain: 8 x 1024 x 2047 147 against 124).
struct Plan { int lt, nw, r; };
Plan plan_of(const vk_block_norm_args* a)
{
    static constexpr int kShapes[3][2] = {{4, 4}, {8, 4}, {8, 8}};
    const int e = a->dtype == VK_DTYPE_BF16 ? 8 : 4;
    Plan pl{8, 8, 8};
    if (e == 8 && a->channels > 128 && a->channels <= 256) pl.lt = 4;
    while (pl.lt > 1 && (64 / pl.lt) * kShapes[2][0] * kShapes[2][1] < a->channels) pl.lt >>= 1;
    // fewer than 256 workgroups: narrower windows spread over more CUs
    while (pl.lt > 1 && (int64_t)a->batch * ((a->length + pl.lt * e - 1) / (pl.lt * e)) < 256) pl.lt >>= 1;
    for (const auto& s : kShapes)
        if ((64 / pl.lt) * s[0] * s[1] >= a->channels) { pl.nw = s[0]; pl.r = s[1]; break; }
    return pl;
}

template <auto KERNEL>
int launch_kernel(const NDev& d, int64_t blocks, int threads, size_t lds, hipStream_t st, const char* what)
{
    static std::atomic<unsigned long long> raised{0};
    hipError_t e = vk_allow_lds(KERNEL, lds, raised);
    if (e != hipSuccess) return fail(VK_E_LAUNCH, what, hipGetErrorString(e));
    hipLaunchKernelGGL(KERNEL, dim3((unsigned)blocks), dim3(threads), lds, st, d);
    e = hipGetLastError();
    return e == hipSuccess ? VK_OK : fail(VK_E_LAUNCH, what, hipGetErrorString(e));
}

template <typename T, int LT, int NW, int R>
int launch(const NDev& d, bool backward, hipStream_t st, const char* what)
{
    const int64_t blocks = ((int64_t)d.a.batch * d.windows + 7) / 8 * 8;       // see Spot
    if (blocks * 64 * NW > 0xffffffffLL) return fail(VK_E_UNSUPPORTED, what, "too many workgroups");     // the limit of a grid, in threads
    const size_t lds = (NW * LT * Pack<T>::E + P_COUNT * (size_t)d.a.channels) * 4;
    return backward ? launch_kernel<block_norm_backward_kernel<T, LT, NW, R>>(d, blocks, 64 * NW, lds, st, what)
                    : launch_kernel<block_norm_kernel<T, LT, NW, R>>(d, blocks, 64 * NW, lds, st, what);
}
template <typename T, int NW, int R>
int by_window(const NDev& d, int lt, bool backward, hipStream_t st, const char* what)
{
    switch (lt) {
    case 8:
        if constexpr (!(Pack<T>::E == 8 && NW == 8 && R == 4)) return launch<T, 8, NW, R>(d, backward, st, what);
        return fail(VK_E_UNSUPPORTED, what, "no such window");      // plan_of takes four lanes there
    case 4: return launch<T, 4, NW, R>(d, backward, st, what);
    case 2: return launch<T, 2, NW, R>(d, backward, st, what);
    default: return launch<T, 1, NW, R>(d, backward, st, what);
    }
}
template <typename T>
int by_shape(const NDev& d, const Plan& pl, bool backward, hipStream_t st, const char* what)
{
    if (pl.nw == 4) return by_window<T, 4, 4>(d, pl.lt, backward, st, what);
    return pl.r == 4 ? by_window<T, 8, 4>(d, pl.lt, backward, st, what) : by_window<T, 8, 8>(d, pl.lt, backward, st, what);
}

int windows_of(const vk_block_norm_args* a, const Plan& pl)
{
    const int w = pl.lt * (a->dtype == VK_DTYPE_BF16 ? 8 : 4);
    return (a->length + w - 1) / w;
}
int64_t workspace_floats(const vk_block_norm_args* a)
{
    return (int64_t)a->batch * windows_of(a, plan_of(a)) * a->channels * (5 + (a->gate && a->gate_per_item ? 1 : 0));
}

}  // namespace

extern "C" int vk_block_norm(const vk_block_norm_args* a, void* stream)
{
    const char* what = "vk_block_norm";
    const int rc = check(a, what, false);
    if (rc != VK_OK) return rc;
    if (a->batch == 0 || a->length == 0) return VK_OK;
    const Plan pl = plan_of(a);
    NDev d{*a, windows_of(a, pl), nullptr, nullptr};
    hipStream_t st = (hipStream_t)stream;
    return a->dtype == VK_DTYPE_BF16 ? by_shape<__bf16>(d, pl, false, st, what) : by_shape<float>(d, pl, false, st, what);
}

extern "C" int64_t vk_block_norm_backward_workspace_bytes(const vk_block_norm_args* a)
{
    const int rc = check_sizes(a, "vk_block_norm_backward_workspace_bytes");
    return rc != VK_OK ? rc : workspace_floats(a) * 4;
}

extern "C" int vk_block_norm_backward(const vk_block_norm_args* a, void* stream)
{
    const char* what = "vk_block_norm_backward";
    int rc = check(a, what, true);
    if (rc != VK_OK) return rc;
    const Plan pl = plan_of(a);
    const bool gates = a->dgate && a->gate_per_item;
    if (gates && a->batch > 65530) return fail(VK_E_UNSUPPORTED, what, "a gate per item: batch > 65530");
    const int64_t need = workspace_floats(a) * 4;
    if (need > 0 && (!a->workspace || a->workspace_bytes < need))
        return fail(VK_E_WORKSPACE, what, "workspace smaller than vk_block_norm_backward_workspace_bytes");
    NDev d{*a, windows_of(a, pl), (float*)a->workspace, nullptr};
    d.part_gate = d.part + (int64_t)a->batch * d.windows * 5 * a->channels;
    hipStream_t st = (hipStream_t)stream;
    if (a->batch > 0 && a->length > 0) {
        rc = a->dtype == VK_DTYPE_BF16 ? by_shape<__bf16>(d, pl, true, st, what) : by_shape<float>(d, pl, true, st, what);
        if (rc != VK_OK) return rc;
    }
    if (!a->dw_pre && !a->db_pre && !a->dscale && !a->dw_post && !a->db_post && !gates) return VK_OK;
    dim3 grid((unsigned)((a->channels + SUM_C - 1) / SUM_C), (unsigned)(5 + (gates ? a->batch : 0)));
    if (a->dtype == VK_DTYPE_BF16) hipLaunchKernelGGL(block_norm_sums_kernel<__bf16>, grid, dim3(SUM_C * SUM_P), 0, st, d);
    else hipLaunchKernelGGL(block_norm_sums_kernel<float>, grid, dim3(SUM_C * SUM_P), 0, st, d);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? VK_OK : fail(VK_E_LAUNCH, what, hipGetErrorString(e));
}
