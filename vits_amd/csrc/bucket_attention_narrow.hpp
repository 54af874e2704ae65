#pragma once
// Forward pass for few rows: new tokens over a long cache, and short sequences.  See bucket_attention.hpp.
//
// A workgroup owns 16 rows of one kv head - a row is a (head of the group, query) pair, so the heads that share keys
// and values share one pass over them - and a share of the keys; each of its four waves walks over tiles of its
// own, with a softmax of its own, and nothing is staged: keys and values go from memory to registers once.
//   * Values are the left operand of P V as they lie in memory (16 channels x consecutive positions).
//   * Keys are needed with the channels consecutive, memory has the positions consecutive: a lane loads the same 8
//     positions of 8 channels (bf16) and turns the 8 x 8 block in registers, one byte permute per output dword.
//     In fp32 a lane needs one channel at a time and nothing is turned.
// The order of the keys in the score tiles is chosen so that a lane's scores are consecutive positions, the right
// operand of P V without crossing lanes.  The next tile's keys are requested before the present one's softmax.
// Bound by memory with one row tile: keys and values are read once (a token over 16 x up to 16384 positions, 16 heads of
// 128 on 4, bf16: 94 us, 3.8 TB/s; 128 bf16 channels spill 10 registers); a sentence of 43 positions takes 14 us, all latency.
#include "bucket_attention.hpp"

namespace vkba {

typedef float f32x4v __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4v mma16(bf16x8 a, bf16x8 b, f32x4v c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4v mma16(float a, float b, f32x4v c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

template <typename T, int DP>
struct Narrow {
    static constexpr int E = Num<T>::EPC, TK = 16 * E;              // positions per 16-byte load, of a tile
    static constexpr int CK = sizeof(T) == 2 ? 32 : 4;              // channels of a score step
    static constexpr int NK = DP / 4;                               // 16-byte loads of a tile's keys per lane
    using frag = typename Num<T>::frag;

    // Keys: load n of a lane is channel row(n), positions base + E * order(lane).
    __device__ __forceinline__ static int order(int m) { return 4 * (m & 3) + (m >> 2); }
    __device__ __forceinline__ static int krow(int n, int q4) { return sizeof(T) == 2 ? 32 * (n >> 3) + 8 * q4 + (n & 7) : 4 * n + q4; }

    __device__ __forceinline__ static void load_keys(u32x4 (&k)[NK], const T* base, int64_t cstride, int d_real, int t0, int length)
    {
        const int l = threadIdx.x & 63, q4 = l >> 4, col = min(t0 + E * order(l & 15), length - E);
        if (d_real == DP && cstride < (int64_t)(1 << 24)) {
            const unsigned lane = ((unsigned)(krow(0, 1) - krow(0, 0)) * (unsigned)q4 * (unsigned)cstride + (unsigned)col) * (unsigned)sizeof(T);
            const char* p = (const char*)base;
#pragma unroll
            for (int n = 0; n < NK; ++n) __builtin_memcpy(&k[n], p + (int64_t)krow(n, 0) * cstride * (int64_t)sizeof(T) + lane, 16);
            return;
        }
        // Channels that are not there, among the last 32, are zero: another channel's infinity would make a NaN of the
        // queries' zero.
        int real = d_real;
        asm volatile("" : "+s"(real));                              // masks made where they are used, not kept over the loop
#pragma unroll
        for (int n = 0; n < NK; ++n) {
            const int d = krow(n, q4);
            if (krow(n, 0) < DP - 32) {
                __builtin_memcpy(&k[n], base + (int64_t)d * cstride + col, 16);
            } else {
                __builtin_memcpy(&k[n], base + (int64_t)min(d, real - 1) * cstride + col, 16);
                k[n] &= (unsigned)((d - real) >> 31);
            }
        }
    }
    // Values: load (blk, r) of a lane is channel 16 blk + lane % 16, positions base + 4 E r + E (lane / 16); zero at and
    // behind `limit`, whatever lies there.
    __device__ __forceinline__ static void load_values(u32x4 (&v)[DP / 4], const T* base, int64_t cstride, int d_real, int t0, int length, int limit)
    {
        const int l = threadIdx.x & 63, row = l & 15;
        int col[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) col[r] = min(t0 + 4 * E * r + E * (l >> 4), length - E);
        if (d_real == DP && cstride < (int64_t)(1 << 24)) {
            const unsigned lane = (unsigned)row * (unsigned)cstride * (unsigned)sizeof(T);
            const char* p = (const char*)base;
#pragma unroll
            for (int n = 0; n < DP / 4; ++n)
                __builtin_memcpy(&v[n], p + (int64_t)(16 * (n >> 2)) * cstride * (int64_t)sizeof(T) + (lane + (unsigned)col[n & 3] * (unsigned)sizeof(T)), 16);
        } else {
#pragma unroll
            for (int n = 0; n < DP / 4; ++n)
                __builtin_memcpy(&v[n], base + (int64_t)min(16 * (n >> 2) + row, d_real - 1) * cstride + col[n & 3], 16);
        }
        if (t0 + TK <= limit) return;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            u32x4 keep;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (E == 4) keep[j] = col[r] + j < limit ? 0xffffffffu : 0u;
                else keep[j] = (col[r] + 2 * j < limit ? 0xffffu : 0u) | (col[r] + 2 * j + 1 < limit ? 0xffff0000u : 0u);
            }
#pragma unroll
            for (int blk = 0; blk < DP / 16; ++blk) v[4 * blk + r] &= keep;
        }
    }
};

// s[o][r]: key base + 4 E r + E (lane / 16) + o of row lane % 16.
template <int DP>
__device__ __forceinline__ void narrow_scores(f32x4v (&s)[8], const u32x4 (&k)[DP / 4], const bf16x8 (&q)[DP / 32])
{
#pragma unroll
    for (int st = 0; st < DP / 32; ++st)
#pragma unroll
        for (int o = 0; o < 8; ++o) {
            u32x4 a;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                a[j] = __builtin_amdgcn_perm(k[8 * st + 2 * j + 1][o >> 1], k[8 * st + 2 * j][o >> 1], (o & 1) ? 0x07060302u : 0x05040100u);
            bf16x8 f;
            __builtin_memcpy(&f, &a, 16);
            s[o] = mma16(f, q[st], s[o]);
        }
}
template <int DP>
__device__ __forceinline__ void narrow_scores(f32x4v (&s)[4], const u32x4 (&k)[DP / 4], const float (&q)[DP / 4])
{
#pragma unroll
    for (int st = 0; st < DP / 4; ++st)
#pragma unroll
        for (int o = 0; o < 4; ++o) s[o] = mma16(__uint_as_float(k[st][o]), q[st], s[o]);
}
template <int DP>
__device__ __forceinline__ void narrow_values(f32x4v (&acc)[DP / 16], const u32x4 (&v)[DP / 4], const f32x4v (&p)[8])
{
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        bf16x8 b;
#pragma unroll
        for (int o = 0; o < 8; ++o) b[o] = (__bf16)p[o][r];
#pragma unroll
        for (int blk = 0; blk < DP / 16; ++blk) {
            bf16x8 a;
            __builtin_memcpy(&a, &v[4 * blk + r], 16);
            acc[blk] = mma16(a, b, acc[blk]);
        }
    }
}
template <int DP>
__device__ __forceinline__ void narrow_values(f32x4v (&acc)[DP / 16], const u32x4 (&v)[DP / 4], const f32x4v (&p)[4])
{
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int o = 0; o < 4; ++o)
#pragma unroll
            for (int blk = 0; blk < DP / 16; ++blk) acc[blk] = mma16(__uint_as_float(v[4 * blk + r][o]), p[o][r], acc[blk]);
}

template <typename T, int DP>
__global__ __launch_bounds__(NTHR, 1)
void bucket_attention_narrow_kernel(Dev p)
{
    using N = Narrow<T, DP>;
    constexpr int E = N::E, TK = N::TK, NQ = DP / N::CK;
    extern __shared__ __align__(16) unsigned char lds[];
    float* tab = reinterpret_cast<float*>(lds);
    const Place at = place(p, (int)blockIdx.x);
    if (!at.any) return;
    const int b = at.b, kvh = at.kvh, split = at.within % p.splits, r0 = 16 * (at.within / p.splits);
    const Item it = uniform_item(p, b);
    const int l = threadIdx.x & 63, q4 = l >> 4, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int rows = p.group * p.queries, row = r0 + (l & 15), rc = row < rows ? row : rows - 1;
    const int g = rc / p.queries, qi = rc - g * p.queries, head = kvh * p.group + g;
    const bool valid = row < rows && qi < it.nq;
    const int pos = it.start + qi;
    // positions of the tile's rows: one head's queries, or all of them
    const int last = min(r0 + 15, rows - 1), g0 = r0 / p.queries, g1 = last / p.queries;
    const int i_lo = g0 == g1 ? r0 - g0 * p.queries : 0, i_hi = g0 == g1 ? last - g0 * p.queries : p.queries - 1;

    int end = it.nk;
    if (p.causal) end = clampi(it.start + min(i_hi, it.nq - 1) + 1, 0, end);      // behind it may lie anything
    if (i_lo >= it.nq) end = 0;
    const int first = split * p.per_split * TK;
    end = min(end, first + p.per_split * TK);
    const int offsets = 2 * p.far_ + 1;
    const T* kg = (const T*)p.k + (int64_t)b * p.kb + (int64_t)kvh * p.head_dim * p.kc;
    const T* vg = (const T*)p.v + (int64_t)b * p.vb + (int64_t)kvh * p.head_dim * p.vc;

    float m = -__builtin_inff(), sum = 0.0f;
    f32x4v acc[DP / 16];
#pragma unroll
    for (int blk = 0; blk < DP / 16; ++blk) acc[blk] = f32x4v{0.0f, 0.0f, 0.0f, 0.0f};
    if (first < end) {
        u32x4 kr[N::NK], vr[DP / 4];
        const int t_first = first + wave * TK;
        // the rows' own queries: few, and read once
        typename N::frag qf[NQ];
        {
            const T* col = (const T*)p.q + (int64_t)b * p.qb + (int64_t)head * p.head_dim * p.qc + qi;
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int s = 0; s < NQ; ++s)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int d = 32 * s + 8 * q4 + e;
                        const T v = col[(int64_t)(d < p.head_dim ? d : p.head_dim - 1) * p.qc];
                        qf[s][e] = valid && d < p.head_dim ? v : (T)0.0f;
                    }
            } else {
#pragma unroll
                for (int s = 0; s < NQ; ++s) {
                    const int d = 4 * s + q4;
                    const T v = col[(int64_t)(d < p.head_dim ? d : p.head_dim - 1) * p.qc];
                    qf[s] = valid && d < p.head_dim ? v : 0.0f;
                }
            }
        }
        // bias: the table of the heads at hand, where these keys come near their queries; else its ends
        const int gap_lo = first - (it.start + i_hi), gap_hi = end - 1 - (it.start + i_lo);
        const int reach = bias_side(p, gap_lo, gap_hi);
        float left = 0.0f, right = 0.0f;
        const float* mine = tab + (g - g0) * offsets;
        if (reach == BIAS_NEAR) {
            for (int o = (int)threadIdx.x; o < offsets; o += NTHR) {
                const int bk = clampi(p.bucket_of[o], 0, p.buckets - 1);
                for (int h = g0; h <= g1; ++h) tab[(h - g0) * offsets + o] = p.bias[(int64_t)(kvh * p.group + h) * p.buckets + bk] * LOG2E;
            }
        }
        if (p.bias) {
            left = p.bias[(int64_t)head * p.buckets + clampi(p.bucket_of[0], 0, p.buckets - 1)] * LOG2E;
            right = p.bias[(int64_t)head * p.buckets + clampi(p.bucket_of[2 * p.far_], 0, p.buckets - 1)] * LOG2E;
        }
        __syncthreads();
        // one round more than tiles: the first only requests keys
        for (int j0 = t_first - NWAVE * TK; j0 < end; j0 += NWAVE * TK) {
            const bool here = j0 >= t_first;
            f32x4v s[E];
            if (here) {
                N::load_values(vr, vg, p.vc, p.head_dim, j0, p.keys, end);
#pragma unroll
                for (int o = 0; o < E; ++o) s[o] = f32x4v{0.0f, 0.0f, 0.0f, 0.0f};
                narrow_scores<DP>(s, kr, qf);
            }
            if (j0 + NWAVE * TK < end) N::load_keys(kr, kg, p.kc, p.head_dim, j0 + NWAVE * TK, p.keys);
            if (!here) continue;
            // by the keys that are there, as for the whole share above: where the table was not staged, no tile takes it
            const int side = bias_side(p, j0 - (it.start + i_hi), min(j0 + TK, end) - 1 - (it.start + i_lo));
            const float flat = side == BIAS_LEFT ? left : side == BIAS_RIGHT ? right : 0.0f;
            const bool whole = j0 + TK <= end && !(p.causal && j0 + TK - 1 > it.start + i_lo);
            const int stop = p.causal ? min(end, pos + 1) : end;
            float mx = -__builtin_inff();
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int first_j = j0 + 4 * E * r + E * q4, j8 = min(first_j, p.keys - E);     // see load_keys
#pragma unroll
                for (int o = 0; o < E; ++o) {
                    const int j = j8 + o;
                    const float bias = side == BIAS_NEAR ? mine[clampi(j - pos, -p.far_, p.far_) + p.far_] : flat;
                    s[o][r] = fmaf(s[o][r], p.c, bias);
                    if (!whole && (j < first_j || j >= stop)) s[o][r] = -__builtin_inff();
                    mx = fmaxf(mx, s[o][r]);
                }
            }
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            if (__any(mx > m + 8.0f)) {                     // as in the kernel for many rows: m follows in large steps
                const float top = fmaxf(mx, m), alpha = exp2_hw(m - (top == -__builtin_inff() ? 0.0f : top));
                sum *= alpha;
#pragma unroll
                for (int blk = 0; blk < DP / 16; ++blk) acc[blk] *= alpha;
                m = top;
            }
            const float base = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
            for (int o = 0; o < E; ++o)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[o][r] = exp2_hw(s[o][r] - base);
                    sum += s[o][r];
                }
            narrow_values<DP>(acc, vr, s);
        }
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);

    // the four waves' results
    __syncthreads();
    float* red = reinterpret_cast<float*>(lds);             // [wave][DP + 2][16]
    float* my = red + wave * (DP + 2) * 16 + (l & 15);
#pragma unroll
    for (int blk = 0; blk < DP / 16; ++blk)
#pragma unroll
        for (int r = 0; r < 4; ++r) my[(16 * blk + 4 * q4 + r) * 16] = acc[blk][r];
    if (q4 == 0) { my[DP * 16] = m; my[(DP + 1) * 16] = sum; }
    __syncthreads();
    if (row >= rows) return;
    const float* all = red + (l & 15);
    float top = -__builtin_inff(), w[NWAVE], total = 0.0f;
#pragma unroll
    for (int i = 0; i < NWAVE; ++i) top = fmaxf(top, all[(i * (DP + 2) + DP) * 16]);
    const float base = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
    for (int i = 0; i < NWAVE; ++i) {
        w[i] = exp2_hw(all[(i * (DP + 2) + DP) * 16] - base);
        total = fmaf(w[i], all[(i * (DP + 2) + DP + 1) * 16], total);
    }
    const bool some = qi < it.nq && !(total == 0.0f);       // NaN in the inputs stays visible
    const int64_t lrow = ((int64_t)b * p.heads + head) * p.queries + qi, lrows = (int64_t)p.batch * p.heads * p.queries;
    T* og = (T*)p.out + (int64_t)b * p.ob + (int64_t)head * p.head_dim * p.oc + qi;
    float* po = p.part_o + ((int64_t)split * p.batch * p.heads + (int64_t)b * p.heads + head) * p.head_dim * p.queries + qi;
    const float inv = 1.0f / total;
    for (int d = (int)threadIdx.x >> 4; d < p.head_dim; d += NTHR / 16) {
        float o = 0.0f;
#pragma unroll
        for (int i = 0; i < NWAVE; ++i) o = fmaf(w[i], all[(i * (DP + 2) + d) * 16], o);
        if (p.splits == 1) og[(int64_t)d * p.oc] = (T)(some ? o * inv : 0.0f);
        else if (some) po[(int64_t)d * p.queries] = o;
    }
    if (threadIdx.x < 16) {
        if (p.splits == 1) {
            p.lse[lrow] = some ? (top + log2f(total)) * LN2 : -__builtin_inff();
        } else {
            p.part_ml[((int64_t)split * lrows + lrow) * 2] = some ? top : -__builtin_inff();
            p.part_ml[((int64_t)split * lrows + lrow) * 2 + 1] = some ? total : 0.0f;
        }
    }
}

}  // namespace vkba
