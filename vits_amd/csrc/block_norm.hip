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
#include <hip/hip_runtime.h>
#include <atomic>
#include <stdint.h>
#include <stdio.h>
#include <string.h>
#include "../../include/vits_amd.h"
#include "api_internal.hpp"
#include "chunk_load.hpp"

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
// Columns t.. of a row of `length`; those at or behind `live` are written as 0.
template <typename T, int E>
__device__ __forceinline__ void store_cols(T* row, const float (&v)[E], int t, int length, int live)
{
    T tmp[E];
#pragma unroll
    for (int e = 0; e < E; ++e) tmp[e] = t + e < live ? (T)v[e] : (T)0.0f;
    if (t + E <= length) {
        __builtin_memcpy(row + t, tmp, E * sizeof(T));
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) if (t + e < length) row[t + e] = tmp[e];
    }
}

// Sum over the channel groups of a workgroup, for every column: lanes of one column group sit LT apart in a wave.
template <int LT, int E, int NW>
__device__ __forceinline__ void column_sum(float (&v)[E], float* red)
{
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, lt = lane % LT;
#pragma unroll
    for (int o = LT; o < 64; o <<= 1)
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] += __shfl_xor(v[e], o);
    __syncthreads();                                        // the previous sum has been read
    if (lane < LT)
#pragma unroll
        for (int e = 0; e < E; ++e) red[(wave * LT + lt) * E + e] = v[e];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) s += red[(w * LT + lt) * E + e];
        v[e] = s;
    }
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
// before `live` count.  LT lanes along time, the other lanes and the waves along the channels.
template <typename T, int LT, int NW>
struct Spot {
    static constexpr int E = Pack<T>::E, CG = 64 / LT * NW;
    int cg, rows, b, t, live, lt, channels;
    __device__ __forceinline__ Spot(const NDev& p)
    {
        const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
        lt = lane % LT;
        cg = wave * (64 / LT) + lane / LT;
        b = (int)blockIdx.x / p.windows;
        t = ((int)blockIdx.x - b * p.windows) * LT * E + lt * E;
        channels = p.a.channels;
        live = p.a.length;
        if (p.a.lengths) { const int64_t n = p.a.lengths[b]; live = (int)(n < 0 ? 0 : n > p.a.length ? p.a.length : n); }
        rows = cg < p.a.channels ? (p.a.channels - cg + CG - 1) / CG : 0;
    }
    __device__ __forceinline__ int channel(int r) const { return cg + r * CG; }
    template <int R>
    __device__ __forceinline__ void load(u32x4 (&v)[R], const void* base, int64_t bstride, int64_t cstride) const
    {
        // threads without a channel read the last one again: the loads stay free of branches
        const T* p = (const T*)base + (int64_t)b * bstride;
#pragma unroll
        for (int r = 0; r < R; ++r) v[r] = load_chunk<T>(p + (int64_t)min(channel(r), channels - 1) * cstride, t, live);
    }
    __device__ __forceinline__ T* row(void* base, int64_t bstride, int64_t cstride, int r) const
    {
        return (T*)base + (int64_t)b * bstride + (int64_t)channel(r) * cstride;
    }
};

template <typename T, int LT, int NW, int R>
__global__ __launch_bounds__(64 * NW)
void block_norm_kernel(NDev p)
{
    using S = Spot<T, LT, NW>;
    constexpr int E = S::E;
    __shared__ float red[NW * LT * E];
    const vk_block_norm_args& a = p.a;
    const S at(p);
    const bool layer = a.norm == VK_NORM_LAYER;
    u32x4 xr[R], yr[R], gr[R];
    at.load(xr, a.x, a.x_bstride, a.x_cstride);
    if (a.y) at.load(yr, a.y, a.y_bstride, a.y_cstride);
    if (a.gate && !a.gate_per_item) at.load(gr, a.gate, a.gate_bstride, a.gate_cstride);
    float h[R][E];
#pragma unroll
    for (int r = 0; r < R; ++r) unpack(h[r], xr[r]);
    if (a.y) {
        float mean[E], rstd[E];
        if (a.w_post) column_stats<LT, E, NW, R>([&](int r, float (&v)[E]) { unpack(v, yr[r]); }, at.rows, a.channels, a.eps, layer, red, mean, rstd);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (r >= at.rows) continue;
            const int c = at.channel(r);
            const float s = a.scale ? a.scale[c] : 1.0f;
            float g[E], z[E];
            if (a.gate && !a.gate_per_item) {
                unpack(g, gr[r]);
#pragma unroll
                for (int e = 0; e < E; ++e) g[e] *= s;
            } else {
                const float q = a.gate ? s * (float)((const T*)a.gate)[(int64_t)at.b * a.gate_bstride + (int64_t)c * a.gate_cstride] : s;
#pragma unroll
                for (int e = 0; e < E; ++e) g[e] = q;
            }
            unpack(z, yr[r]);
            if (a.w_post) {
                const float w = a.w_post[c], bias = a.b_post ? a.b_post[c] : 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) z[e] = fmaf((z[e] - mean[e]) * rstd[e], w, bias);
            }
#pragma unroll
            for (int e = 0; e < E; ++e) h[r][e] = fmaf(g[e], z[e], h[r][e]);
            if (a.h) store_cols<T, E>(at.row(a.h, a.h_bstride, a.h_cstride, r), h[r], at.t, a.length, at.live);
        }
    } else if (a.h) {
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (r < at.rows) store_cols<T, E>(at.row(a.h, a.h_bstride, a.h_cstride, r), h[r], at.t, a.length, at.live);
    }
    if (a.n) {
        float mean[E], rstd[E];
        column_stats<LT, E, NW, R>([&](int r, float (&v)[E]) {
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = h[r][e]; }, at.rows, a.channels, a.eps, layer, red, mean, rstd);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (r >= at.rows) continue;
            const int c = at.channel(r);
            const float w = a.w_pre[c], bias = a.b_pre ? a.b_pre[c] : 0.0f;
            float o[E];
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = fmaf((h[r][e] - mean[e]) * rstd[e], w, bias);
            store_cols<T, E>(at.row(a.n, a.n_bstride, a.n_cstride, r), o, at.t, a.length, at.live);
        }
    }
}

// Gradient through a norm: g -> (g - mean(g) - vhat * mean(g * vhat)) * rstd (layer; without mean(g) for rms).
//
// The gradient of h stays in registers in fp32 from the norm before the next block to the norm after this one.
// Parameter gradients are sums over the columns of a row: over the lanes of a column group (shuffles), then one
// number per row and workgroup goes to memory, and a second kernel adds the workgroups in a fixed order.
template <typename T, int LT, int NW, int R>
__global__ __launch_bounds__(64 * NW)
void block_norm_backward_kernel(NDev p)
{
    using S = Spot<T, LT, NW>;
    constexpr int E = S::E;
    __shared__ float red[NW * LT * E];
    const vk_block_norm_args& a = p.a;
    const S at(p);
    const bool layer = a.norm == VK_NORM_LAYER;
    const float inv = 1.0f / (float)a.channels;
    float* part = p.part + (int64_t)blockIdx.x * 5 * a.channels;
    auto over_columns = [&](const float (&x)[E]) {
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) s += x[e];
#pragma unroll
        for (int o = 1; o < LT; o <<= 1) s += __shfl_xor(s, o);
        return s;
    };

    float g[R][E];              // gradient of h, then of z
    if (a.dn) {
        u32x4 hr[R], dr[R];
        at.load(hr, a.h, a.h_bstride, a.h_cstride);
        at.load(dr, a.dn, a.dn_bstride, a.dn_cstride);
        float mean[E], rstd[E], m1[E], m2[E];
        column_stats<LT, E, NW, R>([&](int r, float (&v)[E]) { unpack(v, hr[r]); }, at.rows, a.channels, a.eps, layer, red, mean, rstd);
#pragma unroll
        for (int e = 0; e < E; ++e) m1[e] = m2[e] = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (r >= at.rows) continue;
            const int c = at.channel(r);
            const float w = a.w_pre[c];
            float v[E], d[E], dw[E];
            unpack(v, hr[r]);
            unpack(d, dr[r]);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float vh = (v[e] - mean[e]) * rstd[e];
                dw[e] = d[e] * vh;
                m1[e] = fmaf(d[e], w, m1[e]);
                m2[e] = fmaf(dw[e], w, m2[e]);
            }
            const float sw = over_columns(dw), sb = over_columns(d);
            if (at.lt == 0) { part[c] = sw; part[a.channels + c] = sb; }
        }
        if (layer) column_sum<LT, E, NW>(m1, red);
        column_sum<LT, E, NW>(m2, red);
#pragma unroll
        for (int e = 0; e < E; ++e) { m1[e] = layer ? m1[e] * inv : 0.0f; m2[e] *= inv; }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float w = r < at.rows ? a.w_pre[at.channel(r)] : 0.0f;
            float v[E], d[E];
            unpack(v, hr[r]);
            unpack(d, dr[r]);
#pragma unroll
            for (int e = 0; e < E; ++e) g[r][e] = (fmaf(d[e], w, -m1[e]) - (v[e] - mean[e]) * rstd[e] * m2[e]) * rstd[e];
        }
    } else {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < E; ++e) g[r][e] = 0.0f;
    }
    u32x4 yr[R];
    if (a.y) at.load(yr, a.y, a.y_bstride, a.y_cstride);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (r >= at.rows) continue;
        if (a.dh) {
            float d[E];
            unpack(d, load_chunk<T>((const T*)a.dh + (int64_t)at.b * a.dh_bstride + (int64_t)at.channel(r) * a.dh_cstride, at.t, at.live));
#pragma unroll
            for (int e = 0; e < E; ++e) g[r][e] += d[e];
        }
        store_cols<T, E>(at.row(a.dx, a.dx_bstride, a.dx_cstride, r), g[r], at.t, a.length, at.live);
    }
    if (!a.y) return;

    float mean[E], rstd[E], m1[E], m2[E];
    if (a.w_post) column_stats<LT, E, NW, R>([&](int r, float (&v)[E]) { unpack(v, yr[r]); }, at.rows, a.channels, a.eps, layer, red, mean, rstd);
#pragma unroll
    for (int e = 0; e < E; ++e) m1[e] = m2[e] = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (r >= at.rows) continue;
        const int c = at.channel(r);
        const float s = a.scale ? a.scale[c] : 1.0f;
        const float w = a.w_post ? a.w_post[c] : 1.0f, bias = a.b_post ? a.b_post[c] : 0.0f;
        float gate[E], dg[E], ds[E], dw[E], v[E];
        if (a.gate && !a.gate_per_item) {
            unpack(gate, load_chunk<T>((const T*)a.gate + (int64_t)at.b * a.gate_bstride + (int64_t)c * a.gate_cstride, at.t, at.live));
        } else {
            const float q = a.gate ? (float)((const T*)a.gate)[(int64_t)at.b * a.gate_bstride + (int64_t)c * a.gate_cstride] : 1.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) gate[e] = q;
        }
        unpack(v, yr[r]);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (a.w_post) v[e] = (v[e] - mean[e]) * rstd[e];
            const float z = a.w_post ? fmaf(v[e], w, bias) : v[e];
            dg[e] = g[r][e] * s * z;                    // gradient of the gate
            ds[e] = g[r][e] * gate[e] * z;              // of the scale
            g[r][e] *= s * gate[e];                     // of z
            dw[e] = g[r][e] * v[e];                     // of the weight
            m1[e] = fmaf(g[r][e], w, m1[e]);
            m2[e] = fmaf(dw[e], w, m2[e]);
        }
        if (a.dgate && !a.gate_per_item)
            store_cols<T, E>(at.row(a.dgate, a.dgate_bstride, a.dgate_cstride, r), dg, at.t, a.length, at.live);
        const float sg = a.dgate && a.gate_per_item ? over_columns(dg) : 0.0f;
        const float ss = over_columns(ds), sw = over_columns(dw), sb = over_columns(g[r]);
        if (at.lt == 0) {
            part[2 * a.channels + c] = ss;
            part[3 * a.channels + c] = sw;
            part[4 * a.channels + c] = sb;
            if (a.dgate && a.gate_per_item) p.part_gate[(int64_t)blockIdx.x * a.channels + c] = sg;
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
        if (r >= at.rows) continue;
        if (a.w_post) {
            const float w = a.w_post[at.channel(r)];
            float v[E];
            unpack(v, yr[r]);
#pragma unroll
            for (int e = 0; e < E; ++e) g[r][e] = (fmaf(g[r][e], w, -m1[e]) - (v[e] - mean[e]) * rstd[e] * m2[e]) * rstd[e];
        }
        store_cols<T, E>(at.row(a.dy, a.dy_bstride, a.dy_cstride, r), g[r], at.t, a.length, at.live);
    }
}

// Sums over the workgroups: blockIdx.y 0..4 a parameter's gradient, 5.. the gate of item blockIdx.y - 5.
constexpr int SUM_C = 32, SUM_P = 8;
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

bool rows_apart(int64_t bstride, int64_t cstride, const vk_block_norm_args* a)
{
    if (a->channels > 1 && cstride < a->length) return false;
    return a->batch <= 1 || bstride >= (int64_t)(a->channels - 1) * (a->channels > 1 ? cstride : 0) + a->length;
}

int check(const vk_block_norm_args* a, const char* what, bool backward)
{
    if (!a) return fail(VK_E_ARG, what, "null argument struct");
    if (a->batch < 0 || a->channels <= 0 || a->length < 0) return fail(VK_E_ARG, what, "bad size");
    if (a->dtype != VK_DTYPE_F32 && a->dtype != VK_DTYPE_BF16) return fail(VK_E_UNSUPPORTED, what, "dtype must be VK_DTYPE_F32 or VK_DTYPE_BF16");
    if (a->norm != VK_NORM_LAYER && a->norm != VK_NORM_RMS) return fail(VK_E_ARG, what, "norm must be VK_NORM_LAYER or VK_NORM_RMS");
    if (a->channels > VK_BLOCK_NORM_MAX_CHANNELS) return fail(VK_E_UNSUPPORTED, what, "more than VK_BLOCK_NORM_MAX_CHANNELS channels");
    if (a->length > (1 << 28)) return fail(VK_E_UNSUPPORTED, what, "length beyond 2^28");
    if (!(a->eps > 0.0f && a->eps < 1e30f)) return fail(VK_E_ARG, what, "eps must be positive and finite");
    const bool some = a->batch > 0 && a->length > 0;
    if (some && !a->y && (a->gate || a->scale || a->w_post)) return fail(VK_E_ARG, what, "gate, scale and the norm after the block need y");
    if ((!a->w_post && a->b_post) || (!a->w_pre && a->b_pre)) return fail(VK_E_ARG, what, "a norm's bias needs its weight");
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
// make more workgroups.
struct Plan { int lt, nw, r; };
Plan plan_of(const vk_block_norm_args* a)
{
    static constexpr int kShapes[4][2] = {{4, 4}, {4, 8}, {8, 8}, {8, 16}};
    const int e = a->dtype == VK_DTYPE_BF16 ? 8 : 4, top = 64 / e;      // at most 64 values of a tensor per thread
    Plan pl{8, 8, top};
    while (pl.lt > 1 && (64 / pl.lt) * 8 * top < a->channels) pl.lt >>= 1;
    // fewer than 256 workgroups: narrower windows spread over more CUs
    while (pl.lt > 1 && (int64_t)a->batch * ((a->length + pl.lt * e - 1) / (pl.lt * e)) < 256) pl.lt >>= 1;
    for (const auto& s : kShapes)
        if ((64 / pl.lt) * s[0] * s[1] >= a->channels) { pl.nw = s[0]; pl.r = s[1]; break; }
    return pl;
}

template <typename T, int LT, int NW, int R>
int launch(const NDev& d, bool backward, hipStream_t st, const char* what)
{
    const int64_t blocks = (int64_t)d.a.batch * d.windows;
    if (blocks > 0x7fffffff) return fail(VK_E_UNSUPPORTED, what, "too many workgroups");
    if (backward) hipLaunchKernelGGL((block_norm_backward_kernel<T, LT, NW, R>), dim3((unsigned)blocks), dim3(64 * NW), 0, st, d);
    else hipLaunchKernelGGL((block_norm_kernel<T, LT, NW, R>), dim3((unsigned)blocks), dim3(64 * NW), 0, st, d);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? VK_OK : fail(VK_E_LAUNCH, what, hipGetErrorString(e));
}
template <typename T, int NW, int R>
int by_window(const NDev& d, int lt, bool backward, hipStream_t st, const char* what)
{
    switch (lt) {
    case 8: return launch<T, 8, NW, R>(d, backward, st, what);
    case 4: return launch<T, 4, NW, R>(d, backward, st, what);
    case 2: return launch<T, 2, NW, R>(d, backward, st, what);
    default: return launch<T, 1, NW, R>(d, backward, st, what);
    }
}
template <typename T>
int by_shape(const NDev& d, const Plan& pl, bool backward, hipStream_t st, const char* what)
{
    if (pl.nw == 4) return pl.r == 4 ? by_window<T, 4, 4>(d, pl.lt, backward, st, what) : by_window<T, 4, 8>(d, pl.lt, backward, st, what);
    if constexpr (Pack<T>::E == 4)
        if (pl.r == 16) return by_window<T, 8, 16>(d, pl.lt, backward, st, what);
    return by_window<T, 8, 8>(d, pl.lt, backward, st, what);
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
    if (!a || a->batch < 0 || a->channels <= 0 || a->length < 0 || a->channels > VK_BLOCK_NORM_MAX_CHANNELS)
        return fail(VK_E_ARG, "vk_block_norm_backward_workspace_bytes", "bad size");
    return workspace_floats(a) * 4;
}

extern "C" int vk_block_norm_backward(const vk_block_norm_args* a, void* stream)
{
    const char* what = "vk_block_norm_backward";
    int rc = check(a, what, true);
    if (rc != VK_OK) return rc;
    const Plan pl = plan_of(a);
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
    const bool gates = a->dgate && a->gate_per_item;
    if (!a->dw_pre && !a->db_pre && !a->dscale && !a->dw_post && !a->db_post && !gates) return VK_OK;
    if (a->batch > 65530) return fail(VK_E_UNSUPPORTED, what, "batch > 65530");
    dim3 grid((unsigned)((a->channels + SUM_C - 1) / SUM_C), (unsigned)(5 + (gates ? a->batch : 0)));
    if (a->dtype == VK_DTYPE_BF16) hipLaunchKernelGGL(block_norm_sums_kernel<__bf16>, grid, dim3(SUM_C * SUM_P), 0, st, d);
    else hipLaunchKernelGGL(block_norm_sums_kernel<float>, grid, dim3(SUM_C * SUM_P), 0, st, d);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? VK_OK : fail(VK_E_LAUNCH, what, hipGetErrorString(e));
}
