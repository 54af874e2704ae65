// Backward pass of the bucketed-bias attention: the probabilities are recomputed from the saved
// log-sum-exp, once for the gradient of the queries and of the bias (a workgroup owns queries and
// walks over keys), once for the gradients of the keys and values (a workgroup owns keys and walks
// over the queries of every head that shares them).  Two walks cost 7 products instead of 5, but every
// sum has one owner and a fixed order: no atomics, bit-identical from run to run.
// Measured: 2 x 4095 causal positions, 16 bf16 heads of 128 on 4, 802 us (428 TFLOP/s of the formula's products), bound by
// matrix and vector instructions of two waves per SIMD that overlap little; 16 x up to 697, 2 fp32 heads of 96, 183 us.
#include "bucket_attention.hpp"
#include "api_internal.hpp"
#include "bucket_attention_host.hpp"

namespace {
using namespace vkba;

// How a kernel is built: waves per SIMD, positions of a staged tile, whether dk and dv have workgroups of their own.
// Two waves per SIMD (at most 256 registers each) matter most: one computes while the other waits.  With bf16 and 128
// channels dq fits with tiles of 32 keys (4096 positions, 16 heads: 806 -> 522 us), while dk and dv together with the
// fragments of k and v do not fit at all and are computed by separate workgroups, for one more product (S twice).
template <typename T, int DP, int KW>
struct Shape {
    static constexpr bool BF = sizeof(T) == 2;
    static constexpr bool SPLIT = BF && DP > 96;
    static constexpr int MIN_WAVES = BF || DP <= 64 ? 2 : 1;
    // the next tile is loaded into registers while the present one is computed, unless that makes the rest spill too much
    // (bf16, 8 x 8 heads of 96, 2048 positions: 594 us with, 533 without; 16 heads of 128 on 4, 1024 positions: 131, 110) or,
    // fp32, takes the second wave.  With 128 channels and tiles of 32 dq spills 21 registers with it, 4 without, and it pays
    // all the same where the walk is long (2 x 16 heads on 4, 4095 causal positions: 791 us with, 834 without; two-sided
    // 1419, 1476; 8 x 1024: 425, 413).
    static constexpr bool AHEAD = BF ? DP <= 64 || (DP > 96 && KW == 1) : MIN_WAVES == 1;
    static constexpr int KT_DQ = BF && DP > 96 && KW == 1 ? 32 : 64, KT_DKV = KT_DQ;
    static constexpr int OWN = Tile<T, DP, 64>::BYTES;                  // image of 64 of the workgroup's own rows
    static constexpr int IMAGES = 2 * OWN;                              // as large as two tiles
};

__host__ __device__ inline int64_t kv_elements(const Dev& p) { return (int64_t)p.batch * (p.heads / p.group) * p.head_dim * p.keys; }

// A row whose log-sum-exp is below this (all its keys have a bias that low) passes no gradient back: fp32 does not hold
// what its probabilities need (a step is 2^-3 here and grows), and exp(s - lse) would grow out of bounds.
constexpr float LSE_LEAST = -0x1p20f;

constexpr int DGP = 33;         // pitch of a wave's 32 x 32 block of logit gradients

// dq_i = scale * sum_j ds_ij k_j, and the sums of ds over the diagonals j - pos_i = const (the bias
// gradient by offset).  Scores are transposed as in the forward pass: a query is a lane.
//
// KW = 2: half of the waves take the first, half the second 32 keys of every tile (64 queries per workgroup
// instead of 128) and their sums are joined through LDS at the end.
template <typename T, int DP, int KW>
__global__ __launch_bounds__(NTHR, (Shape<T, DP, KW>::MIN_WAVES))
void bucket_dq_kernel(Dev p)
{
    using F = typename Num<T>::frag;
    using S = Shape<T, DP, KW>;
    constexpr int KT = S::KT_DQ, KS = Num<T>::KS, PT = Tile<T, DP, KT>::PT, QW = NWAVE / KW, QT = QW * 32;
    extern __shared__ __align__(16) unsigned char lds[];
    T* ki = reinterpret_cast<T*>(lds);
    T* vi = reinterpret_cast<T*>(lds + Tile<T, DP, KT>::BYTES);
    T* own = reinterpret_cast<T*>(lds + S::OWN);            // second image of own rows
    float* tab = reinterpret_cast<float*>(lds + S::IMAGES);
    const int offsets = 2 * p.far_ + 1;
    const int l = threadIdx.x & 63, h = l >> 5, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    float* hist = tab + ((offsets + 3) & ~3) + wave * offsets;                  // this wave's diagonal sums
    float* blk_ds = tab + ((offsets + 3) & ~3) + NWAVE * offsets + wave * 32 * DGP;

    const Place at = place(p, (int)blockIdx.x);
    if (!at.any) return;
    const int b = at.b, kvh = at.kvh, head = kvh * p.group + at.within % p.group;
    const int qt = p.tiles - 1 - at.within / p.group;
    const Item it = uniform_item(p, b);
    const int qw = wave / KW, kw = wave % KW;
    const int q0 = qt * QT + qw * 32, qi = q0 + (l & 31);
    const bool valid = qi < it.nq;
    const int64_t row = ((int64_t)b * p.heads + head) * p.queries + qi;
    const int64_t hd = (int64_t)head * p.head_dim;

    const T* kg = (const T*)p.k + (int64_t)b * p.kb + (int64_t)kvh * p.head_dim * p.kc;
    const T* vg = (const T*)p.v + (int64_t)b * p.vb + (int64_t)kvh * p.head_dim * p.vc;
    // keys this workgroup walks over
    int end = it.nk;
    const int last_q = min(qt * QT + QT, it.nq) - 1;
    if (p.causal) end = clampi(it.start + last_q + 1, 0, end);
    if (qt * QT >= it.nq) end = 0;

    Tile<T, DP, KT> kt, vt;
    F qf[DP / KS], dof[DP / KS];
    // delta enters every logit gradient of its row with the same sign, so its error adds up coherently in the
    // bias gradient: summed in 64 bits, rounded once
    float delta = 0.0f;
    // The matrix instruction's rounding leans to one side by some 1e-9 of a product sum, which shows in a bias gradient
    // summed over 10^7 pairs (far bucket of 4095 causal positions: off by 6e-6 of its value).  Every other query takes
    // its gradient with the other sign, so that the lean cancels; the results are turned back at the end.
    const float sgn = (l & 1) ? -1.0f : 1.0f;
    if (qt * QT < it.nq) {
        OwnRows<T, DP, 64, QW> rq, rd;
        rq.load((const T*)p.o + (int64_t)b * p.ob + hd * p.oc, p.oc, p.head_dim, qt * QT, it.nq);
        rd.load((const T*)p.dout + (int64_t)b * p.dob + hd * p.doc, p.doc, p.head_dim, qt * QT, it.nq);
        rq.frags(qf, ki, own, qw);
        rq.load((const T*)p.q + (int64_t)b * p.qb + hd * p.qc, p.qc, p.head_dim, qt * QT, it.nq);
        rd.frags(dof, ki, own, qw);
        delta = (float)dot_frags(qf, dof);
        flip(dof, sgn < 0.0f);
        if (S::AHEAD && end > 0) {
            kt.load(kg, p.kc, p.head_dim, 0, end);
            vt.load(vg, p.vc, p.head_dim, 0, end);
        }
        rq.frags(qf, ki, own, qw);
    }
    // lse2 rounds the row's log-sum-exp in units of log2: a relative error of some 1e-6 that all probabilities of the
    // row share, so it does not average out in the bias gradient.  `off` is that error (below; 64 bits).
    float lse2 = __builtin_inff();
    double off = 0.0;
    if (valid) {
        const float v = p.lse_in[row];
        if (!(v < LSE_LEAST)) {                             // without keys all probabilities are 0
            lse2 = v * LOG2E;
            off = (double)v * 1.4426950408889634 - (double)lse2;
        }
        if (h == 0 && kw == 0) p.delta[row] = delta;
    }
    const float near_fix = sgn * (float)(1.0 - off * (double)LN2);
    const float minus_delta = -sgn * delta;
    stage_bias(tab, p, head);
    if (p.bias) for (int o = l; o < offsets; o += 64) hist[o] = 0.0f;

    f32x16 acc[DP / 32];
#pragma unroll
    for (int blk = 0; blk < DP / 32; ++blk)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[blk][r] = 0.0f;
    double far_left = 0.0, far_right = 0.0;                // this query's sums over the whole blocks beyond the table
    float end_left = 0.0f, end_right = 0.0f;                // of diagonals beyond it in blocks that reach into it

    const int pos0 = it.start + q0, pos = pos0 + (l & 31);
    for (int j0 = 0; j0 < end; j0 += KT) {
        if constexpr (!S::AHEAD) {
            kt.load(kg, p.kc, p.head_dim, j0, end);
            vt.load(vg, p.vc, p.head_dim, j0, end);
        }
        __syncthreads();
        kt.store(ki);
        vt.store(vi);
        __syncthreads();
        if (S::AHEAD && j0 + KT < end) {
            kt.load(kg, p.kc, p.head_dim, j0 + KT, end);
            vt.load(vg, p.vc, p.head_dim, j0 + KT, end);
        }
#pragma unroll
        for (int i = 0; i < KT / 32 / KW; ++i) {
            const int c0 = 32 * (kw * (KT / 32 / KW) + i), js = j0 + c0;
            if (js >= end || (p.causal && js > pos0 + 31)) continue;
            const int lo = js - (pos0 + 31), hi = js + 31 - pos0, side = bias_side(p, lo, hi);
            f32x16 s, dp;
#pragma unroll
            for (int r = 0; r < 16; ++r) { s[r] = 0.0f; dp[r] = minus_delta; }
            dot_channels<DP, PT>(s, ki, c0, qf);
            dot_channels<DP, PT>(dp, vi, c0, dof);
            if (side != BIAS_NEAR && js + 32 <= end && !(p.causal && hi > 0)) {
                const float shift = bias_flat(tab, p, side) - lse2;
#pragma unroll
                for (int r = 0; r < 16; ++r) dp[r] *= exp2_hw(fmaf(s[r], p.c, shift));
            } else {
                const int stop = (p.causal ? min(end, pos + 1) : end) - js;
                const float flat = bias_flat(tab, p, side);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int row = acc_row(r, h);
                    const float bias = side == BIAS_NEAR ? tab[clampi(js + row - pos, -p.far_, p.far_) + p.far_] : flat;
                    dp[r] *= exp2_hw(fmaf(s[r], p.c, bias - lse2));
                    if (row >= stop) dp[r] = 0.0f;
                }
            }
            if (side == BIAS_NEAR) {
                // transposed through LDS so that a lane owns one diagonal of the block
#pragma unroll
                for (int r = 0; r < 16; ++r) blk_ds[acc_row(r, h) * DGP + (l & 31)] = dp[r] * near_fix;
                wave_lds_fence();
                const int dg = l - 31;                          // key index - query index
                float sum = 0.0f;
                if (l < 63) {
                    const int i0 = dg < 0 ? -dg : 0, i1 = dg > 0 ? 32 - dg : 32;
                    for (int e = i0; e < i1; ++e) sum += blk_ds[(e + dg) * DGP + e];
                }
                const int o = js - pos0 + dg;
                // offsets beyond the table all fall on its ends
                if (l < 63) {
                    if (o <= -p.far_) end_left += sum;
                    else if (o >= p.far_) end_right += sum;
                    else hist[o + p.far_] += sum;
                }
                wave_lds_fence();
            } else if (side != BIAS_NONE) {
                float sum = 0.0f;
#pragma unroll
                for (int r = 0; r < 16; ++r) sum += dp[r];
                if (side == BIAS_LEFT) far_left += sum; else far_right += sum;
            }
            dot_positions<DP, PT>(acc, ki, c0, dp);
        }
    }

    if constexpr (KW == 2) {
        __syncthreads();                                    // the images are free
        float* red = reinterpret_cast<float*>(lds) + qw * DP * 32 + (l & 31);
        if (kw == 1)
#pragma unroll
            for (int blk = 0; blk < DP / 32; ++blk)
#pragma unroll
                for (int r = 0; r < 16; ++r) red[(32 * blk + acc_row(r, h)) * 32] = acc[blk][r];
        __syncthreads();
        if (kw == 0)
#pragma unroll
            for (int blk = 0; blk < DP / 32; ++blk)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[blk][r] += red[(32 * blk + acc_row(r, h)) * 32];
    }
    if (qi < p.queries && kw == 0) {
        store_rows((T*)p.dq + (int64_t)b * p.dqb + hd * p.dqc + qi, p.dqc, p.head_dim, acc, h, valid, sgn * p.scale);
    }
    if (p.bias) {
        if (lse2 < __builtin_inff()) {                      // what the rounding of (bias - lse2) and of lse2 left out
            // (a bias of -inf: all probabilities there are 0, and -inf - (-inf) is no rounding)
            const float left = tab[0] - lse2, right = tab[2 * p.far_] - lse2;
            if (left != -__builtin_inff()) far_left *= 1.0 + (((double)tab[0] - (double)lse2 - (double)left) - off) * (double)LN2;
            if (right != -__builtin_inff()) far_right *= 1.0 + (((double)tab[2 * p.far_] - (double)lse2 - (double)right) - off) * (double)LN2;
        }
        far_left = (double)sgn * far_left + end_left;
        far_right = (double)sgn * far_right + end_right;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) { far_left += __shfl_xor(far_left, o); far_right += __shfl_xor(far_right, o); }
        wave_lds_fence();
        if (l == 0) { hist[0] = (float)((double)hist[0] + far_left); hist[offsets - 1] = (float)((double)hist[offsets - 1] + far_right); }
        __syncthreads();
        const float* all = tab + ((offsets + 3) & ~3);
        float* out = p.part_bias + ((int64_t)(head * p.batch + b) * p.tiles + qt) * offsets;
        for (int o = (int)threadIdx.x; o < offsets; o += NTHR)
            out[o] = ((all[o] + all[offsets + o]) + all[2 * offsets + o]) + all[3 * offsets + o];
    }
}

// dk_j = scale * sum_i ds_ij q_i, dv_j = sum_i p_ij dout_i over all heads that share the kv head.  Scores
// are untransposed here (rows = queries, columns = keys): a key is a lane.
//
// KW = 2: half of the waves take the first, half the second 32 queries of every tile (64 keys per workgroup).
// DK, DV: which of the two this workgroup computes.
template <typename T, int DP, int KW, bool DK, bool DV>
__device__ __forceinline__ void key_side(const Dev& p, int id, unsigned char* lds, bool reverse = false)
{
    using F = typename Num<T>::frag;
    using S = Shape<T, DP, KW>;
    constexpr int KT = S::KT_DKV, NS = KT / 32 / KW, KS = Num<T>::KS, PT = Tile<T, DP, KT>::PT, CW = NWAVE / KW;
    T* qim = reinterpret_cast<T*>(lds);
    T* dim = reinterpret_cast<T*>(lds + S::OWN);
    float* st = reinterpret_cast<float*>(lds + S::IMAGES);      // log-sum-exp and -delta of the tile's queries
    float* tab = st + 2 * KT;

    const Place at = place(p, id);
    if (!at.any) return;
    const int b = at.b, kvh = at.kvh;
    const Item it = uniform_item(p, b);
    const int l = threadIdx.x & 63, h = l >> 5, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int cw = wave / KW, kw = wave % KW;
    const int within = reverse ? p.per_unit - 1 - at.within : at.within;
    const int share = within % p.shares;
    const int kt0 = within / p.shares * CW * 32, jb = kt0 + cw * 32, j = jb + (l & 31);
    const bool valid = j < it.nk;
    const int64_t hd = (int64_t)kvh * p.head_dim;

    F kf[DP / KS], vf[DK ? DP / KS : 1];
    if (kt0 < it.nk) {
        OwnRows<T, DP, 64, CW> rk, rv;
        rk.load((const T*)p.k + (int64_t)b * p.kb + hd * p.kc, p.kc, p.head_dim, kt0, it.nk);
        if constexpr (DK) rv.load((const T*)p.v + (int64_t)b * p.vb + hd * p.vc, p.vc, p.head_dim, kt0, it.nk);
        rk.frags(kf, qim, dim, cw);
        if constexpr (DK) rv.frags(vf, qim, dim, cw);
    }
    f32x16 dk[DK ? DP / 32 : 1], dv[DV ? DP / 32 : 1];
#pragma unroll
    for (int blk = 0; blk < DP / 32; ++blk)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            if constexpr (DK) dk[blk][r] = 0.0f;
            if constexpr (DV) dv[blk][r] = 0.0f;
        }

    // queries that see any of these keys: with `causal` those at or behind the first key
    int q_first = 0;
    if (p.causal) q_first = clampi(kt0 - it.start, 0, it.nq) / KT * KT;
    const int tiles = kt0 < it.nk ? (it.nq - q_first + KT - 1) / KT : 0;
    const int steps = tiles > 0 ? tiles * p.group : 0;                          // (head, query tile), of which this share has
    const int first = (int)((int64_t)steps * share / p.shares), last = (int)((int64_t)steps * (share + 1) / p.shares);

    Tile<T, DP, KT> qt, dt;
    float stat = 0.0f;
    auto fetch = [&](int step) {
        const int g = step / tiles, i0 = q_first + (step - g * tiles) * KT;
        const int head = kvh * p.group + g;
        qt.load((const T*)p.q + (int64_t)b * p.qb + (int64_t)head * p.head_dim * p.qc, p.qc, p.head_dim, i0, it.nq);
        dt.load((const T*)p.dout + (int64_t)b * p.dob + (int64_t)head * p.head_dim * p.doc, p.doc, p.head_dim, i0, it.nq);
        const int64_t row = ((int64_t)b * p.heads + head) * p.queries;
        const int i = i0 + ((int)threadIdx.x & (KT - 1));
        if (threadIdx.x < 2 * KT) {                 // converted when it is stored: using it here would wait for all loads
            const float* src = threadIdx.x < KT ? p.lse_in : p.delta;
            stat = i < it.nq ? src[row + i] : threadIdx.x < KT ? -__builtin_inff() : 0.0f;
        }
    };
    if (S::AHEAD && first < last) fetch(first);
    for (int step = first; step < last; ++step) {
        const int g = step / tiles, tile = step - g * tiles, i0 = q_first + tile * KT;
        if constexpr (!S::AHEAD) fetch(step);
        __syncthreads();
        qt.store(qim);
        dt.store(dim);
        if (threadIdx.x < KT) st[threadIdx.x] = stat < LSE_LEAST ? __builtin_inff() : stat * LOG2E;    // no keys: all probabilities 0
        else if (threadIdx.x < 2 * KT) st[threadIdx.x] = -stat;
        if (tile == 0 || step == first) stage_bias(tab, p, kvh * p.group + g);
        __syncthreads();
        if (S::AHEAD && step + 1 < last) fetch(step + 1);
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int c0 = 32 * (kw * NS + i), is = i0 + c0, pos0 = it.start + is;     // this block's queries
            if (is >= it.nq || (p.causal && jb > pos0 + 31)) continue;
            const int lo = jb - (pos0 + 31), hi = jb + 31 - pos0, side = bias_side(p, lo, hi);
            f32x16 s, dp;
#pragma unroll
            for (int r = 0; r < 16; ++r) { s[r] = 0.0f; if constexpr (DK) dp[r] = st[KT + c0 + acc_row(r, h)]; }
            dot_channels<DP, PT>(s, qim, c0, kf);
            if constexpr (DK) dot_channels<DP, PT>(dp, dim, c0, vf);
            const float flat = bias_flat(tab, p, side);
            if (side != BIAS_NEAR) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = exp2_hw(fmaf(s[r], p.c, flat - st[c0 + acc_row(r, h)]));
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int row = acc_row(r, h);
                    const float bias = tab[clampi(j - (pos0 + row), -p.far_, p.far_) + p.far_];
                    s[r] = exp2_hw(fmaf(s[r], p.c, bias - st[c0 + row]));
                }
            }
            // queries behind their length are masked too: a key that only they would see may hold anything
            const int stop = it.nq - is;
            if (p.causal && (hi > 0 || stop < 32)) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int row = acc_row(r, h);
                    if (j > pos0 + row || row >= stop) {
                        s[r] = 0.0f;
                        if constexpr (DK) dp[r] = 0.0f;
                    }
                }
            }
            if constexpr (DV) dot_positions<DP, PT>(dv, dim, c0, s);
            if constexpr (DK) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] *= dp[r];
                dot_positions<DP, PT>(dk, qim, c0, s);
            }
        }
    }
    float* red = reinterpret_cast<float*>(lds) + cw * DP * 32 + (l & 31);
    auto finish = [&](f32x16 (&x)[DP / 32], float* part, void* out, int64_t bstride, int64_t cstride, float scale) {
        if constexpr (KW == 2) {
            __syncthreads();
            if (kw == 1)
#pragma unroll
                for (int blk = 0; blk < DP / 32; ++blk)
#pragma unroll
                    for (int r = 0; r < 16; ++r) red[(32 * blk + acc_row(r, h)) * 32] = x[blk][r];
            __syncthreads();
            if (kw == 0)
#pragma unroll
                for (int blk = 0; blk < DP / 32; ++blk)
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[blk][r] += red[(32 * blk + acc_row(r, h)) * 32];
        }
        if (j >= p.keys || kw != 0) return;
        if (p.shares > 1) {
            float* g = part + (((int64_t)share * p.batch + b) * (p.heads / p.group) * p.head_dim + hd) * p.keys + j;
            store_rows(g, p.keys, p.head_dim, x, h, valid, scale);
        } else {
            store_rows((T*)out + (int64_t)b * bstride + hd * cstride + j, cstride, p.head_dim, x, h, valid, scale);
        }
    };
    if constexpr (DK) finish(dk, p.part_kv, p.dk, p.dkb, p.dkc, p.scale);
    if constexpr (DV) finish(dv, p.part_kv + p.shares * kv_elements(p), p.dv, p.dvb, p.dvc, 1.0f);
}

// dbias[h, c] = sum of the diagonal sums whose offset falls into bucket c, over all workgroups of head h, in 64 bits
// (the sums of a row cancel to zero).
__device__ __forceinline__ void dbias_of_head(const Dev& p, int head, unsigned char* lds)
{
    const int offsets = 2 * p.far_ + 1, tid = (int)threadIdx.x, parts = p.batch * p.tiles;
    float* sums = reinterpret_cast<float*>(lds);
    int* bucket = reinterpret_cast<int*>(sums + offsets);
    const float* src = p.part_bias + (int64_t)head * parts * offsets;
    for (int o = tid; o < offsets; o += NTHR) {
        double s = 0.0;
        int i = 0;
        for (; i + 8 <= parts; i += 8) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = src[(int64_t)(i + e) * offsets + o];
#pragma unroll
            for (int e = 0; e < 8; ++e) s += v[e];
        }
        for (; i < parts; ++i) s += src[(int64_t)i * offsets + o];
        sums[o] = (float)s;
        bucket[o] = clampi(p.bucket_of[o], 0, p.buckets - 1);
    }
    __syncthreads();
    for (int c0 = 0; c0 < p.buckets; c0 += NTHR / 32) {
        const int c = c0 + tid / 32;
        double s = 0.0;
        for (int o = tid & 31; o < offsets; o += 32) s += bucket[o] == c ? (double)sums[o] : 0.0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor(s, o, 32);
        if ((tid & 31) == 0 && c < p.buckets) p.dbias[(int64_t)head * p.buckets + c] = (float)s;
    }
}

// The gradients of keys and values; the last workgroups of the launch do the sums of the bias gradient.
template <typename T, int DP, int KW>
__global__ __launch_bounds__(NTHR, (Shape<T, DP, KW>::MIN_WAVES))
void bucket_dkv_kernel(Dev p)
{
    extern __shared__ __align__(16) unsigned char lds[];
    int id = (int)blockIdx.x;
    if constexpr (Shape<T, DP, KW>::SPLIT) {
        if (id < p.kv_blocks) return key_side<T, DP, KW, true, false>(p, id, lds);
        id -= p.kv_blocks;
        if (id < p.kv_blocks) return key_side<T, DP, KW, false, true>(p, id, lds, p.fold);
    } else {
        if (id < p.kv_blocks) return key_side<T, DP, KW, true, true>(p, id, lds);
    }
    dbias_of_head(p, id - p.kv_blocks, lds);
}

// Sum of the shares of dk and dv; a workgroup has 1024 keys of a row.
template <typename T>
__global__ __launch_bounds__(256) void bucket_kv_sum_kernel(Dev p)
{
    const int per_row = (p.keys + 1023) / 1024, rows_of_item = p.heads / p.group * p.head_dim;
    const int64_t rows = (int64_t)p.batch * rows_of_item, n = kv_elements(p);
    int64_t row = blockIdx.x / per_row;
    const int j0 = (int)(blockIdx.x - row * per_row) * 1024 + (int)threadIdx.x;
    const bool is_v = row >= rows;
    const float* part = p.part_kv + (is_v ? p.shares * n : 0);
    if (is_v) row -= rows;
    const int64_t b = row / rows_of_item, c = row - b * rows_of_item;
    T* out = is_v ? (T*)p.dv + b * p.dvb + c * p.dvc : (T*)p.dk + b * p.dkb + c * p.dkc;
    part += row * p.keys;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int j = j0 + 256 * i;
        if (j >= p.keys) return;
        float x = 0.0f;
        for (int s = 0; s < p.shares; ++s) x += part[s * n + j];
        out[j] = (T)x;
    }
}

template <typename T, int DP, int KW>
int launch_both(Dev d, hipStream_t st)
{
    using S = Shape<T, DP, KW>;
    const size_t offsets = 2 * (size_t)d.far_ + 1;
    const char* what = "vk_bucket_attention_backward";
    constexpr int ROWS = NWAVE / KW * 32;
    d.tiles = (d.queries + ROWS - 1) / ROWS;
    if (d.queries > 0) {
        vkba_place(d, (int64_t)d.tiles * d.group);
        const size_t lds = S::IMAGES + vkba_table_bytes(d) + (d.bias ? NWAVE * (offsets + 32 * DGP) * 4 : 0);
        int rc = vkba_launch<bucket_dq_kernel<T, DP, KW>>(d, vkba_blocks(d), lds, st, what);
        if (rc != VK_OK) return rc;
    }
    vkba_place(d, (int64_t)(d.keys + ROWS - 1) / ROWS * d.shares);
    const int64_t blocks = d.keys > 0 ? vkba_blocks(d) : 0;
    if (blocks > 0x7fffffff) return vkba_fail(VK_E_UNSUPPORTED, what, "too many workgroups");
    d.kv_blocks = (int)blocks;
    // causal: the first keys have the most queries.  Where all workgroups find a place at once (two on every CU),
    // those of dv come in the other order, so that a CU gets a long and a short one (heads of 128: 16 of 1000 positions 90 us
    // without, 86 with; 8 of 2000: 140, 135; launches that leave CUs empty are the same)
    d.fold = d.causal && 2 * blocks <= 512;
    const size_t need = S::IMAGES + 2 * S::KT_DKV * 4 + vkba_table_bytes(d);
    int rc = vkba_launch<bucket_dkv_kernel<T, DP, KW>>(d, (S::SPLIT ? 2 : 1) * blocks + (d.bias ? d.heads : 0),
                                                       need > offsets * 8 ? need : offsets * 8, st, what);
    if (rc != VK_OK || d.shares == 1) return rc;
    return vkba_launch<bucket_kv_sum_kernel<T>>(d, 2 * (kv_elements(d) / d.keys) * ((d.keys + 1023) / 1024), 0, st, what);
}

template <typename T, int KW>
int by_width(const Dev& d, hipStream_t st)
{
    switch ((d.head_dim + 31) / 32) {
    case 1: return launch_both<T, 32, KW>(d, st);
    case 2: return launch_both<T, 64, KW>(d, st);
    case 3: return launch_both<T, 96, KW>(d, st);
    default: return launch_both<T, 128, KW>(d, st);
    }
}

// Rows (queries of the first, keys of the second kernel) per workgroup.
int key_waves(const vk_bucket_attention_args* a)
{
    return a->dtype == VK_DTYPE_F32 || (int64_t)a->batch * a->heads * ((a->queries + 127) / 128) < 256 ? 2 : 1;
}
int64_t parts_of_head(const vk_bucket_attention_args* a)
{
    const int rows = 128 / key_waves(a);
    return (int64_t)a->batch * ((a->queries + rows - 1) / rows);
}
// Shares of the queries (of all heads of the group), each with workgroups of its own for dk and dv; a third launch sums
// them.  Where the workgroups would fill less than half of the chip (one bf16 head of 128 shared by 16, 2048 causal
// positions: 1510 us without, 233 with shares; two fp32 heads of 96, 697 positions: 177, 130; not above: four
// times 8 bf16 heads of 64, 2048 positions, 512 workgroups: 156, 170).  With `causal` also where each walks far: the
// first keys have nearly twice the mean work, and the chip waits for them (4095 positions, 16 heads on 4, batch 2,
// 512 workgroups: 755 us for dk and dv without, 602 + 20 with two shares and their sum).
int key_shares(const vk_bucket_attention_args* a)
{
    const int group = a->kv_heads > 0 ? a->heads / a->kv_heads : 1, rows = 128 / key_waves(a);
    const bool split = a->dtype == VK_DTYPE_BF16 && a->head_dim > 96;
    const int64_t blocks = (int64_t)a->batch * a->kv_heads * ((a->keys + rows - 1) / rows) * (split ? 2 : 1);
    const int64_t steps = (int64_t)group * ((a->queries + 63) / 64), slots = a->dtype == VK_DTYPE_F32 && a->head_dim > 64 ? 256 : 512;
    const int64_t target = a->causal && steps >= 64 ? 1024 : blocks < slots / 2 ? slots : 0;
    if (blocks == 0 || blocks >= target) return 1;
    const int64_t want = (target + blocks - 1) / blocks, most = steps / 2;
    return (int)(want < most ? want : most < 1 ? 1 : most);
}
int64_t workspace_floats(const vk_bucket_attention_args* a)
{
    const int64_t delta = (int64_t)a->batch * a->heads * a->queries;
    const int64_t shares = key_shares(a);
    const int64_t kv = shares > 1 ? 2 * shares * a->batch * a->kv_heads * a->head_dim * a->keys : 0;
    return delta + kv + (a->has_bias ? parts_of_head(a) * a->heads * (2 * (int64_t)a->max_distance + 1) : 0);
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
    if (!vk_strides_ok(a->dout_bstride, a->dout_cstride) || !vk_strides_ok(a->dq_bstride, a->dq_cstride)
        || !vk_strides_ok(a->dk_bstride, a->dk_cstride) || !vk_strides_ok(a->dv_bstride, a->dv_cstride))
        return vkba_fail(VK_E_ARG, what, "a stride of dout, dq, dk or dv is negative or beyond 2^40");
    if (!vk_rows_apart(a->dq_bstride, a->dq_cstride, (int64_t)a->heads * a->head_dim, a->queries, a->batch)
        || !vk_rows_apart(a->dk_bstride, a->dk_cstride, (int64_t)a->kv_heads * a->head_dim, a->keys, a->batch)
        || !vk_rows_apart(a->dv_bstride, a->dv_cstride, (int64_t)a->kv_heads * a->head_dim, a->keys, a->batch))
        return vkba_fail(VK_E_ARG, what, "rows of a gradient overlap");
    const int64_t need = workspace_floats(a) * 4;
    if (need > 0 && (!a->workspace || a->workspace_bytes < need))
        return vkba_fail(VK_E_WORKSPACE, what, "workspace smaller than vk_bucket_attention_backward_workspace_bytes");
    d.delta = (float*)a->workspace;
    d.shares = key_shares(a);
    d.part_kv = d.delta + (int64_t)a->batch * a->heads * a->queries;
    d.part_bias = d.part_kv + (d.shares > 1 ? 2 * d.shares * kv_elements(d) : 0);
    d.dbias = a->dbias;
    hipStream_t st = (hipStream_t)stream;
    if (key_waves(a) == 2) return a->dtype == VK_DTYPE_BF16 ? by_width<__bf16, 2>(d, st) : by_width<float, 2>(d, st);
    return by_width<__bf16, 1>(d, st);
}
