// Forward pass of the bucketed-bias attention.  See bucket_attention.hpp for the data layout.
//
// A workgroup owns 4 * 32 * NQ queries of one head and walks over the keys in tiles of 64, one pass,
// with the running maximum and sum of the softmax.  Scores are computed transposed (rows = keys,
// columns = queries), so a query is a lane: its maximum and sum are lane-local but for one exchange
// between the two lane halves, and the probabilities are already the right operand of P V.
#include "bucket_attention.hpp"
#include "api_internal.hpp"
#include "bucket_attention_host.hpp"

namespace {
using namespace vkba;

template <typename T, int DP, int NQ>
__global__ __launch_bounds__(NTHR)
void bucket_attention_kernel(Dev p)
{
    using F = typename Num<T>::frag;
    constexpr int KS = Num<T>::KS, PT = Num<T>::PT, QT = NWAVE * 32 * NQ;
    extern __shared__ __align__(16) unsigned char lds[];
    T* ki = reinterpret_cast<T*>(lds);
    T* vi = ki + DP * PT;
    float* tab = reinterpret_cast<float*>(vi + DP * PT);

    int unit, within;
    if (!place(p, unit, within)) return;
    const int kvh = unit % (p.heads / p.group), b = unit / (p.heads / p.group);
    const int g = within % p.group;
    int rest = within / p.group;
    const int split = rest % p.splits;
    const int qt = p.tiles - 1 - rest / p.splits;          // causal: the longest rows first
    const int head = kvh * p.group + g;
    const Item it = item_of(p, b);
    const int l = threadIdx.x & 63, h = l >> 5, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int q0 = qt * QT + wave * 32 * NQ;

    const T* qg = (const T*)p.q + (int64_t)b * p.qb + (int64_t)head * p.head_dim * p.qc;
    const T* kg = (const T*)p.k + (int64_t)b * p.kb + (int64_t)kvh * p.head_dim * p.kc;
    const T* vg = (const T*)p.v + (int64_t)b * p.vb + (int64_t)kvh * p.head_dim * p.vc;

    // keys this workgroup walks over
    int end = it.nk;
    const int last_q = min(qt * QT + QT, it.nq) - 1;
    if (p.causal) end = clampi(it.start + last_q + 1, 0, end);
    if (qt * QT >= it.nq) end = 0;
    const int first = split * p.per_split * KT;
    end = min(end, first + p.per_split * KT);

    F qf[NQ][DP / KS];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int qi = q0 + 32 * n + (l & 31);
        load_frags<DP>(qf[n], qg + qi, p.qc, p.head_dim, qi < it.nq);
    }
    stage_bias(tab, p, head);

    f32x16 acc[NQ][DP / 32];
    float m[NQ], sum[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        m[n] = -__builtin_inff();
        sum[n] = 0.0f;
#pragma unroll
        for (int blk = 0; blk < DP / 32; ++blk)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[n][blk][r] = 0.0f;
    }

    Tile<T, DP> kt, vt;
    if (first < end) {
        kt.load(kg, p.kc, p.head_dim, first, end);
        vt.load(vg, p.vc, p.head_dim, first, end);
    }
    const float c = p.c;
    for (int j0 = first; j0 < end; j0 += KT) {
        __syncthreads();
        kt.store(ki);
        vt.store(vi);
        __syncthreads();
        if (j0 + KT < end) {
            kt.load(kg, p.kc, p.head_dim, j0 + KT, end);
            vt.load(vg, p.vc, p.head_dim, j0 + KT, end);
        }
        const int pos0 = it.start + q0;
        if (p.causal && j0 > pos0 + 32 * NQ - 1) continue;      // this wave's queries see none of the tile
        f32x16 s[2][NQ];
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[sub][n][r] = 0.0f;
            dot_channels<DP, NQ>(s[sub], ki, 32 * sub, qf);
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const int pos = pos0 + 32 * n + (l & 31);
            float mx = m[n];
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                const int js = j0 + 32 * sub;
                const int lo = js - (pos0 + 32 * n + 31), hi = js + 31 - (pos0 + 32 * n);
                const BlockBias bb = block_bias(tab, p, lo, hi);
                if (bb.near_) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int off = clampi(js + acc_row(r, h) - pos, -p.far_, p.far_);
                        s[sub][n][r] = fmaf(s[sub][n][r], c, tab[off + p.far_]);
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[sub][n][r] = fmaf(s[sub][n][r], c, bb.flat);
                }
                if (js + 32 > end || (p.causal && hi > 0)) {
                    const int stop = p.causal ? min(end, pos + 1) : end;
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (js + acc_row(r, h) >= stop) s[sub][n][r] = -__builtin_inff();
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[sub][n][r]);
            }
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float base = mx == -__builtin_inff() ? 0.0f : mx;
            if (__any(mx > m[n])) {                             // the maximum moved for some query of the wave
                const float alpha = exp2_hw(m[n] - base);
                sum[n] *= alpha;
#pragma unroll
                for (int blk = 0; blk < DP / 32; ++blk)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[n][blk][r] *= alpha;
                m[n] = mx;
            }
            float add = 0.0f;
#pragma unroll
            for (int sub = 0; sub < 2; ++sub)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[sub][n][r] = exp2_hw(s[sub][n][r] - base);
                    add += s[sub][n][r];
                }
            sum[n] += add;
        }
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) dot_positions<DP, NQ>(acc, vi, 32 * sub, s[sub]);
    }

#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int qi = q0 + 32 * n + (l & 31);
        const float total = sum[n] + __shfl_xor(sum[n], 32);
        if (qi >= p.queries) continue;
        const bool live = qi < it.nq && total > 0.0f;
        const bool broken = qi < it.nq && !(total >= 0.0f);     // NaN in the inputs stays visible
        const int64_t row = ((int64_t)b * p.heads + head) * p.queries + qi;
        if (p.splits == 1) {
            const float inv = live || broken ? 1.0f / total : 0.0f;
            T* og = (T*)p.out + (int64_t)b * p.ob + (int64_t)head * p.head_dim * p.oc + qi;
#pragma unroll
            for (int blk = 0; blk < DP / 32; ++blk)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int d = 32 * blk + acc_row(r, h);
                    if (d < p.head_dim) og[(int64_t)d * p.oc] = (T)(live || broken ? acc[n][blk][r] * inv : 0.0f);
                }
            if (h == 0) p.lse[row] = live || broken ? (m[n] + log2f(total)) * LN2 : -__builtin_inff();
        } else {
            const int64_t rows = (int64_t)p.batch * p.heads * p.queries;
            float* po = p.part_o + ((int64_t)split * p.batch * p.heads + (int64_t)b * p.heads + head) * p.head_dim * p.queries + qi;
#pragma unroll
            for (int blk = 0; blk < DP / 32; ++blk)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int d = 32 * blk + acc_row(r, h);
                    if (d < p.head_dim) po[(int64_t)d * p.queries] = acc[n][blk][r];
                }
            if (h == 0) {
                p.part_ml[((int64_t)split * rows + row) * 2] = qi < it.nq ? m[n] : -__builtin_inff();
                p.part_ml[((int64_t)split * rows + row) * 2 + 1] = qi < it.nq ? total : 0.0f;
            }
        }
    }
}

// Joins the shares of the keys: out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s, m = max m_s.
// One thread per query and channel block of a head.
template <typename T>
__global__ __launch_bounds__(256)
void bucket_attention_join_kernel(Dev p)
{
    const int64_t rows = (int64_t)p.batch * p.heads * p.queries;
    const int64_t per_head = (int64_t)p.head_dim * p.queries;
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= rows * p.head_dim) return;
    const int64_t bh = e / per_head, rem = e - bh * per_head;
    const int d = (int)(rem / p.queries), qi = (int)(rem - (int64_t)d * p.queries);
    const int64_t row = bh * p.queries + qi;
    float m = -__builtin_inff();
    for (int s = 0; s < p.splits; ++s) m = fmaxf(m, p.part_ml[((int64_t)s * rows + row) * 2]);
    const float base = m == -__builtin_inff() ? 0.0f : m;
    float o = 0.0f, total = 0.0f;
    for (int s = 0; s < p.splits; ++s) {
        const float l = p.part_ml[((int64_t)s * rows + row) * 2 + 1];
        const float w = exp2_hw(p.part_ml[((int64_t)s * rows + row) * 2] - base);
        if (l != 0.0f) {
            total = fmaf(w, l, total);
            o = fmaf(w, p.part_o[((int64_t)s * p.batch * p.heads + bh) * per_head + rem], o);
        }
    }
    const int b = (int)(bh / p.heads), head = (int)(bh - (int64_t)b * p.heads);
    const bool none = total == 0.0f;
    T* og = (T*)p.out + (int64_t)b * p.ob + ((int64_t)head * p.head_dim + d) * p.oc + qi;
    *og = (T)(none ? 0.0f : o / total);
    if (d == 0) p.lse[row] = none ? -__builtin_inff() : (m + log2f(total)) * LN2;
}

template <typename T, int DP, int NQ>
int launch(const Dev& d, hipStream_t st)
{
    const size_t lds = 2 * (size_t)Tile<T, DP>::BYTES + vkba_table_bytes(d);
    return vkba_launch<bucket_attention_kernel<T, DP, NQ>>(d, vkba_blocks(d), lds, st, "vk_bucket_attention");
}

template <typename T, int NQ>
int by_width(const Dev& d, hipStream_t st)
{
    switch ((d.head_dim + 31) / 32) {
    case 1: return launch<T, 32, NQ>(d, st);
    case 2: return launch<T, 64, NQ>(d, st);
    case 3: return launch<T, 96, NQ>(d, st);
    default: return launch<T, 128, NQ>(d, st);
    }
}

}  // namespace

// Queries per workgroup and shares of the keys' length.  512 workgroups keep two on every CU; with
// fewer the key axis is cut, down to two tiles per share.
static void plan_forward(const vk_bucket_attention_args* a, Dev& d, int& nq)
{
    const int64_t heads = (int64_t)a->batch * a->heads;
    nq = a->dtype == VK_DTYPE_BF16 && heads * ((a->queries + 255) / 256) >= 512 ? 2 : 1;
    d.tiles = (a->queries + 128 * nq - 1) / (128 * nq);
    const int64_t blocks = heads * d.tiles;
    const int key_tiles = (a->keys + KT - 1) / KT;
    int64_t splits = blocks >= 256 || blocks == 0 ? 1 : (512 + blocks - 1) / blocks;
    splits = splits > (key_tiles + 1) / 2 ? (key_tiles + 1) / 2 : splits;
    if (splits < 1) splits = 1;
    d.per_split = (int)((key_tiles + splits - 1) / splits);
    if (d.per_split < 1) d.per_split = 1;
    d.splits = (key_tiles + d.per_split - 1) / d.per_split;
    if (d.splits < 1) d.splits = 1;
    vkba_place(d, (int64_t)d.tiles * d.splits * d.group);
}

extern "C" int64_t vk_bucket_attention_workspace_bytes(const vk_bucket_attention_args* a)
{
    vkba::Dev d;
    int rc = vkba_check(a, d, "vk_bucket_attention_workspace_bytes", false), nq;
    if (rc != VK_OK) return rc;
    plan_forward(a, d, nq);
    return d.splits > 1 ? (int64_t)d.splits * a->batch * a->heads * a->queries * (a->head_dim + 2) * 4 : 0;
}

extern "C" int vk_bucket_attention(const vk_bucket_attention_args* a, void* stream)
{
    Dev d;
    int rc = vkba_check(a, d, "vk_bucket_attention", true), nq;
    if (rc != VK_OK) return rc;
    if (a->batch == 0 || a->queries == 0) return VK_OK;
    if (!a->out || !a->lse) return vk_fail(VK_E_ARG, "vk_bucket_attention: null output");
    if (!vkba_rows_apart(a->out_bstride, a->out_cstride, (int64_t)a->heads * a->head_dim, a->queries, a->batch))
        return vk_fail(VK_E_ARG, "vk_bucket_attention: rows of out overlap");
    plan_forward(a, d, nq);
    const int64_t need = d.splits > 1 ? (int64_t)d.splits * a->batch * a->heads * a->queries * (a->head_dim + 2) * 4 : 0;
    if (need > 0 && (!a->workspace || a->workspace_bytes < need))
        return vk_fail(VK_E_WORKSPACE, "vk_bucket_attention: workspace smaller than vk_bucket_attention_workspace_bytes");
    d.part_ml = (float*)a->workspace;
    d.part_o = d.part_ml + (int64_t)d.splits * a->batch * a->heads * a->queries * 2;
    hipStream_t st = (hipStream_t)stream;
    rc = a->dtype == VK_DTYPE_BF16 ? (nq == 2 ? by_width<__bf16, 2>(d, st) : by_width<__bf16, 1>(d, st))
                                   : by_width<float, 1>(d, st);
    if (rc != VK_OK || d.splits == 1) return rc;
    const int64_t n = (int64_t)a->batch * a->heads * a->head_dim * a->queries;
    dim3 grid((unsigned)((n + 255) / 256));
    if (a->dtype == VK_DTYPE_BF16) hipLaunchKernelGGL(bucket_attention_join_kernel<__bf16>, grid, dim3(256), 0, st, d);
    else hipLaunchKernelGGL(bucket_attention_join_kernel<float>, grid, dim3(256), 0, st, d);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? VK_OK : vk_fail(VK_E_LAUNCH, hipGetErrorString(e));
}
