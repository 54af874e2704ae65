// Backward pass of the bucketed-bias attention: the probabilities are recomputed from the saved
// log-sum-exp, once for the gradient of the queries and of the bias (a workgroup owns queries and
// walks over keys), once for the gradients of the keys and values (a workgroup owns keys and walks
// over the queries of every head that shares them).  Two walks cost 7 products instead of 5, but every
// sum has one owner and a fixed order: no atomics, bit-identical from run to run.
#include "bucket_attention.hpp"
#include "api_internal.hpp"
#include "bucket_attention_host.hpp"

namespace {
using namespace vkba;

constexpr int DGP = 33;         // pitch of a wave's 32 x 32 block of logit gradients

// dq_i = scale * sum_j ds_ij k_j, and the sums of ds over the diagonals j - pos_i = const (the bias
// gradient by offset).  Scores are transposed as in the forward pass: a query is a lane.
template <typename T, int DP>
__global__ __launch_bounds__(NTHR)
void bucket_dq_kernel(Dev p)
{
    using F = typename Num<T>::frag;
    constexpr int KS = Num<T>::KS, PT = Num<T>::PT, QT = NWAVE * 32;
    extern __shared__ __align__(16) unsigned char lds[];
    T* ki = reinterpret_cast<T*>(lds);
    T* vi = ki + DP * PT;
    float* tab = reinterpret_cast<float*>(vi + DP * PT);
    const int offsets = 2 * p.far_ + 1;
    const int l = threadIdx.x & 63, h = l >> 5, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    float* hist = tab + ((offsets + 3) & ~3) + wave * offsets;                  // this wave's diagonal sums
    float* blk_ds = tab + ((offsets + 3) & ~3) + NWAVE * offsets + wave * 32 * DGP;

    int unit, within;
    if (!place(p, unit, within)) return;
    const int kvh = unit % (p.heads / p.group), b = unit / (p.heads / p.group);
    const int head = kvh * p.group + within % p.group;
    const int qt = p.tiles - 1 - within / p.group;
    const Item it = item_of(p, b);
    const int q0 = qt * QT + wave * 32, qi = q0 + (l & 31);
    const bool valid = qi < it.nq;
    const int64_t row = ((int64_t)b * p.heads + head) * p.queries + qi;
    const int64_t hd = (int64_t)head * p.head_dim;

    const T* kg = (const T*)p.k + (int64_t)b * p.kb + (int64_t)kvh * p.head_dim * p.kc;
    const T* vg = (const T*)p.v + (int64_t)b * p.vb + (int64_t)kvh * p.head_dim * p.vc;
    F qf[1][DP / KS], dof[1][DP / KS];
    load_frags<DP>(qf[0], (const T*)p.q + (int64_t)b * p.qb + hd * p.qc + qi, p.qc, p.head_dim, valid);
    load_frags<DP>(dof[0], (const T*)p.dout + (int64_t)b * p.dob + hd * p.doc + qi, p.doc, p.head_dim, valid);
    // delta enters every logit gradient of its row with the same sign, so its error adds up coherently in the
    // bias gradient: summed in 64 bits, rounded once
    double delta64 = 0.0;
    if (valid) {
        const T* og = (const T*)p.o + (int64_t)b * p.ob + hd * p.oc + qi;
        const T* dg = (const T*)p.dout + (int64_t)b * p.dob + hd * p.doc + qi;
        for (int d = h; d < p.head_dim; d += 2) delta64 = fma((double)(float)og[(int64_t)d * p.oc], (double)(float)dg[(int64_t)d * p.doc], delta64);
    }
    delta64 += __shfl_xor(delta64, 32);
    const float delta = (float)delta64;
    float lse2 = __builtin_inff();
    if (valid) {
        const float v = p.lse_in[row];
        lse2 = v == -__builtin_inff() ? __builtin_inff() : v * LOG2E;          // no keys: all probabilities 0
        if (h == 0) p.delta[row] = delta;
    }
    stage_bias(tab, p, head);
    if (p.bias) for (int o = l; o < offsets; o += 64) hist[o] = 0.0f;

    int end = it.nk;
    const int last_q = min(qt * QT + QT, it.nq) - 1;
    if (p.causal) end = clampi(it.start + last_q + 1, 0, end);
    if (qt * QT >= it.nq) end = 0;

    f32x16 acc[1][DP / 32];
#pragma unroll
    for (int blk = 0; blk < DP / 32; ++blk)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[0][blk][r] = 0.0f;
    float far_left = 0.0f, far_right = 0.0f;

    Tile<T, DP> kt, vt;
    if (end > 0) {
        kt.load(kg, p.kc, p.head_dim, 0, end);
        vt.load(vg, p.vc, p.head_dim, 0, end);
    }
    const int pos0 = it.start + q0, pos = pos0 + (l & 31);
    for (int j0 = 0; j0 < end; j0 += KT) {
        __syncthreads();
        kt.store(ki);
        vt.store(vi);
        __syncthreads();
        if (j0 + KT < end) {
            kt.load(kg, p.kc, p.head_dim, j0 + KT, end);
            vt.load(vg, p.vc, p.head_dim, j0 + KT, end);
        }
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            const int js = j0 + 32 * sub;
            if (js >= end || (p.causal && js > pos0 + 31)) continue;
            f32x16 s[1], dp[1];
#pragma unroll
            for (int r = 0; r < 16; ++r) { s[0][r] = 0.0f; dp[0][r] = -delta; }
            dot_channels<DP, 1>(s, ki, 32 * sub, qf);
            dot_channels<DP, 1>(dp, vi, 32 * sub, dof);
            const int lo = js - (pos0 + 31), hi = js + 31 - pos0;
            const BlockBias bb = block_bias(tab, p, lo, hi);
            if (bb.near_) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int off = clampi(js + acc_row(r, h) - pos, -p.far_, p.far_);
                    s[0][r] = fmaf(s[0][r], p.c, tab[off + p.far_] - lse2);
                }
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[0][r] = fmaf(s[0][r], p.c, bb.flat - lse2);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) dp[0][r] *= exp2_hw(s[0][r]);
            if (js + 32 > end || (p.causal && hi > 0)) {
                const int stop = p.causal ? min(end, pos + 1) : end;
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (js + acc_row(r, h) >= stop) dp[0][r] = 0.0f;
            }
            if (p.bias) {
                if (bb.near_) {
                    // transposed through LDS so that a lane owns one diagonal of the block
#pragma unroll
                    for (int r = 0; r < 16; ++r) blk_ds[acc_row(r, h) * DGP + (l & 31)] = dp[0][r];
                    wave_lds_fence();
                    const int dg = l - 31;                      // key index - query index
                    float sum = 0.0f;
                    if (l < 63) {
                        const int i0 = dg < 0 ? -dg : 0, i1 = dg > 0 ? 32 - dg : 32;
                        for (int i = i0; i < i1; ++i) sum += blk_ds[(i + dg) * DGP + i];
                    }
                    const int off = js - pos0 + dg;
                    // offsets beyond the table all fall on its ends: those lanes keep their sum to themselves
                    if (l < 63) {
                        if (off <= -p.far_) far_left += sum;
                        else if (off >= p.far_) far_right += sum;
                        else hist[off + p.far_] += sum;
                    }
                    wave_lds_fence();
                } else {
                    float sum = 0.0f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) sum += dp[0][r];
                    if (hi <= -p.far_) far_left += sum; else far_right += sum;
                }
            }
            dot_positions<DP, 1>(acc, ki, 32 * sub, dp);
        }
    }

    if (qi < p.queries) {
        T* dqg = (T*)p.dq + (int64_t)b * p.dqb + hd * p.dqc + qi;
#pragma unroll
        for (int blk = 0; blk < DP / 32; ++blk)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int d = 32 * blk + acc_row(r, h);
                if (d < p.head_dim) dqg[(int64_t)d * p.dqc] = (T)(valid ? acc[0][blk][r] * p.scale : 0.0f);
            }
    }
    if (p.bias) {
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) { far_left += __shfl_xor(far_left, o); far_right += __shfl_xor(far_right, o); }
        wave_lds_fence();
        if (l == 0) { hist[0] += far_left; hist[offsets - 1] += far_right; }
        __syncthreads();
        const float* all = tab + ((offsets + 3) & ~3);
        float* out = p.part_bias + ((int64_t)(head * p.batch + b) * p.tiles + qt) * offsets;
        for (int o = (int)threadIdx.x; o < offsets; o += NTHR)
            out[o] = ((all[o] + all[offsets + o]) + all[2 * offsets + o]) + all[3 * offsets + o];
    }
}

// dk_j = scale * sum_i ds_ij q_i, dv_j = sum_i p_ij dout_i over all heads that share the kv head.  Scores
// are untransposed here (rows = queries, columns = keys): a key is a lane.
template <typename T, int DP>
__global__ __launch_bounds__(NTHR)
void bucket_dkv_kernel(Dev p)
{
    using F = typename Num<T>::frag;
    constexpr int KS = Num<T>::KS, PT = Num<T>::PT;
    extern __shared__ __align__(16) unsigned char lds[];
    T* qim = reinterpret_cast<T*>(lds);
    T* dim = qim + DP * PT;
    float* st = reinterpret_cast<float*>(dim + DP * PT);        // log-sum-exp and delta of the tile's queries
    float* tab = st + 2 * KT;

    int unit, within;
    if (!place(p, unit, within)) return;
    const int kvh = unit % (p.heads / p.group), b = unit / (p.heads / p.group);
    const Item it = item_of(p, b);
    const int l = threadIdx.x & 63, h = l >> 5, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int kt0 = within * NWAVE * 32, jb = kt0 + wave * 32, j = jb + (l & 31);
    const bool valid = j < it.nk;

    F kf[1][DP / KS], vf[1][DP / KS];
    load_frags<DP>(kf[0], (const T*)p.k + (int64_t)b * p.kb + (int64_t)kvh * p.head_dim * p.kc + j, p.kc, p.head_dim, valid);
    load_frags<DP>(vf[0], (const T*)p.v + (int64_t)b * p.vb + (int64_t)kvh * p.head_dim * p.vc + j, p.vc, p.head_dim, valid);
    f32x16 dk[1][DP / 32], dv[1][DP / 32];
#pragma unroll
    for (int blk = 0; blk < DP / 32; ++blk)
#pragma unroll
        for (int r = 0; r < 16; ++r) { dk[0][blk][r] = 0.0f; dv[0][blk][r] = 0.0f; }

    // queries that see any of these keys: with `causal` those at or behind the first key
    int q_first = 0;
    if (p.causal) q_first = clampi(kt0 - it.start, 0, it.nq) / KT * KT;
    const int tiles = kt0 < it.nk ? (it.nq - q_first + KT - 1) / KT : 0;
    const int steps = tiles > 0 ? tiles * p.group : 0;

    Tile<T, DP> qt, dt;
    float stat = 0.0f;
    auto fetch = [&](int step) {
        const int g = step / tiles, i0 = q_first + (step - g * tiles) * KT;
        const int head = kvh * p.group + g;
        const int64_t hd = (int64_t)head * p.head_dim;
        qt.load((const T*)p.q + (int64_t)b * p.qb + hd * p.qc, p.qc, p.head_dim, i0, it.nq);
        dt.load((const T*)p.dout + (int64_t)b * p.dob + hd * p.doc, p.doc, p.head_dim, i0, it.nq);
        const int64_t row = ((int64_t)b * p.heads + head) * p.queries;
        const int i = i0 + ((int)threadIdx.x & (KT - 1));
        if (threadIdx.x < KT) {
            stat = __builtin_inff();
            if (i < it.nq) { const float v = p.lse_in[row + i]; stat = v == -__builtin_inff() ? __builtin_inff() : v * LOG2E; }
        } else if (threadIdx.x < 2 * KT) {
            stat = i < it.nq ? p.delta[row + i] : 0.0f;
        }
    };
    if (steps > 0) fetch(0);
    for (int step = 0; step < steps; ++step) {
        const int g = step / tiles, tile = step - g * tiles, i0 = q_first + tile * KT;
        __syncthreads();
        qt.store(qim);
        dt.store(dim);
        if (threadIdx.x < 2 * KT) st[threadIdx.x] = stat;
        if (tile == 0) stage_bias(tab, p, kvh * p.group + g);
        __syncthreads();
        if (step + 1 < steps) fetch(step + 1);
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            const int is = i0 + 32 * sub, pos0 = it.start + is;
            if (is >= it.nq || (p.causal && jb > pos0 + 31)) continue;
            f32x16 s[1], dp[1];
#pragma unroll
            for (int r = 0; r < 16; ++r) { s[0][r] = 0.0f; dp[0][r] = -st[KT + 32 * sub + acc_row(r, h)]; }
            dot_channels<DP, 1>(s, qim, 32 * sub, kf);
            dot_channels<DP, 1>(dp, dim, 32 * sub, vf);
            const int lo = jb - (pos0 + 31), hi = jb + 31 - pos0;
            const BlockBias bb = block_bias(tab, p, lo, hi);
            if (bb.near_) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int off = clampi(j - (pos0 + acc_row(r, h)), -p.far_, p.far_);
                    s[0][r] = fmaf(s[0][r], p.c, tab[off + p.far_] - st[32 * sub + acc_row(r, h)]);
                }
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[0][r] = fmaf(s[0][r], p.c, bb.flat - st[32 * sub + acc_row(r, h)]);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) s[0][r] = exp2_hw(s[0][r]);
            if (p.causal && hi > 0) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (j > pos0 + acc_row(r, h)) s[0][r] = 0.0f;
            }
            dot_positions<DP, 1>(dv, dim, 32 * sub, s);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[0][r] *= dp[0][r];
            dot_positions<DP, 1>(dk, qim, 32 * sub, s);
        }
    }
    if (j < p.keys) {
        const int64_t hd = (int64_t)kvh * p.head_dim;
        T* dkg = (T*)p.dk + (int64_t)b * p.dkb + hd * p.dkc + j;
        T* dvg = (T*)p.dv + (int64_t)b * p.dvb + hd * p.dvc + j;
#pragma unroll
        for (int blk = 0; blk < DP / 32; ++blk)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int d = 32 * blk + acc_row(r, h);
                if (d < p.head_dim) {
                    dkg[(int64_t)d * p.dkc] = (T)(valid ? dk[0][blk][r] * p.scale : 0.0f);
                    dvg[(int64_t)d * p.dvc] = (T)(valid ? dv[0][blk][r] : 0.0f);
                }
            }
    }
}

// dbias[h, c] = sum of the diagonal sums whose offset falls into bucket c, over all workgroups of head h.
constexpr int BR_THREADS = 1024;
__global__ __launch_bounds__(BR_THREADS)
void bucket_dbias_kernel(const float* part, const int32_t* bucket_of, float* dbias, int parts, int far_, int buckets)
{
    extern __shared__ float sums[];                     // [4][offsets]
    const int offsets = 2 * far_ + 1, head = (int)blockIdx.x, tid = (int)threadIdx.x;
    const float* src = part + (int64_t)head * parts * offsets;
    const int lane = tid & 255, quarter = tid >> 8;
    for (int o = lane; o < offsets; o += 256) {
        float s = 0.0f;
        for (int i = quarter; i < parts; i += 4) s += src[(int64_t)i * offsets + o];
        sums[quarter * offsets + o] = s;
    }
    __syncthreads();
    for (int c = tid; c < buckets; c += BR_THREADS) {
        float s = 0.0f;
        for (int o = 0; o < offsets; ++o) {
            const int bk = clampi(bucket_of[o], 0, buckets - 1);
            if (bk == c) s += (sums[o] + sums[offsets + o]) + (sums[2 * offsets + o] + sums[3 * offsets + o]);
        }
        dbias[(int64_t)head * buckets + c] = s;
    }
}

template <typename T, int DP>
int launch_both(Dev d, hipStream_t st)
{
    const size_t img = 2 * (size_t)Tile<T, DP>::BYTES, offsets = 2 * (size_t)d.far_ + 1;
    const char* what = "vk_bucket_attention_backward";
    if (d.queries > 0) {
        d.tiles = (d.queries + NWAVE * 32 - 1) / (NWAVE * 32);
        vkba_place(d, (int64_t)d.tiles * d.group);
        const size_t lds = img + vkba_table_bytes(d) + (d.bias ? NWAVE * (offsets + 32 * DGP) * 4 : 0);
        int rc = vkba_launch<bucket_dq_kernel<T, DP>>(d, vkba_blocks(d), lds, st, what);
        if (rc != VK_OK) return rc;
    }
    if (d.keys > 0) {
        vkba_place(d, (d.keys + NWAVE * 32 - 1) / (NWAVE * 32));
        return vkba_launch<bucket_dkv_kernel<T, DP>>(d, vkba_blocks(d), img + 2 * KT * 4 + vkba_table_bytes(d), st, what);
    }
    return VK_OK;
}

template <typename T>
int by_width(const Dev& d, hipStream_t st)
{
    switch ((d.head_dim + 31) / 32) {
    case 1: return launch_both<T, 32>(d, st);
    case 2: return launch_both<T, 64>(d, st);
    case 3: return launch_both<T, 96>(d, st);
    default: return launch_both<T, 128>(d, st);
    }
}

int64_t parts_of_head(const vk_bucket_attention_args* a)
{
    return (int64_t)a->batch * ((a->queries + NWAVE * 32 - 1) / (NWAVE * 32));
}
int64_t workspace_floats(const vk_bucket_attention_args* a)
{
    const int64_t delta = (int64_t)a->batch * a->heads * a->queries;
    return delta + (a->has_bias ? parts_of_head(a) * a->heads * (2 * (int64_t)a->max_distance + 1) : 0);
}

}  // namespace

extern "C" int64_t vk_bucket_attention_backward_workspace_bytes(const vk_bucket_attention_args* a)
{
    vkba::Dev d;
    const int rc = vkba_check(a, d, "vk_bucket_attention_backward_workspace_bytes", false);
    return rc != VK_OK ? rc : workspace_floats(a) * 4;
}

extern "C" int vk_bucket_attention_backward(const vk_bucket_attention_args* a, void* stream)
{
    const char* what = "vk_bucket_attention_backward";
    vkba::Dev d;
    int rc = vkba_check(a, d, what, true);
    if (rc != VK_OK) return rc;
    const bool rows = a->batch > 0 && a->queries > 0, cols = a->batch > 0 && a->keys > 0;
    if (rows && (!a->out || !a->lse || !a->dout || !a->dq)) return vkba_fail(VK_E_ARG, what, "null out, lse, dout or dq");
    if (cols && (!a->dk || !a->dv)) return vkba_fail(VK_E_ARG, what, "null dk or dv");
    if (a->has_bias && !a->dbias) return vkba_fail(VK_E_ARG, what, "null dbias");
    if (!vkba_rows_apart(a->dq_bstride, a->dq_cstride, (int64_t)a->heads * a->head_dim, a->queries, a->batch)
        || !vkba_rows_apart(a->dk_bstride, a->dk_cstride, (int64_t)a->kv_heads * a->head_dim, a->keys, a->batch)
        || !vkba_rows_apart(a->dv_bstride, a->dv_cstride, (int64_t)a->kv_heads * a->head_dim, a->keys, a->batch))
        return vkba_fail(VK_E_ARG, what, "rows of a gradient overlap");
    const int64_t need = workspace_floats(a) * 4;
    if (need > 0 && (!a->workspace || a->workspace_bytes < need))
        return vkba_fail(VK_E_WORKSPACE, what, "workspace smaller than vk_bucket_attention_backward_workspace_bytes");
    d.delta = (float*)a->workspace;
    d.part_bias = d.delta + (int64_t)a->batch * a->heads * a->queries;
    hipStream_t st = (hipStream_t)stream;
    if (a->batch > 0) {
        rc = a->dtype == VK_DTYPE_BF16 ? by_width<__bf16>(d, st) : by_width<float>(d, st);
        if (rc != VK_OK) return rc;
    }
    if (!a->has_bias) return VK_OK;
    const size_t lds = 4 * (2 * (size_t)a->max_distance + 1) * 4;
    hipLaunchKernelGGL(bucket_dbias_kernel, dim3((unsigned)a->heads), dim3(BR_THREADS), lds, st, d.part_bias, a->bucket_of,
                       a->dbias, (int)parts_of_head(a), a->max_distance, a->buckets);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? VK_OK : vkba_fail(VK_E_LAUNCH, what, hipGetErrorString(e));
}
