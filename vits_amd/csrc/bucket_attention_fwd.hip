// Forward pass of the bucketed-bias attention.  See bucket_attention.hpp for the data layout.
//
// A workgroup owns 128 or 64 queries of one head and walks over the keys in tiles of 64, one pass,
// with the running maximum and sum of the softmax.  Scores are computed transposed (rows = keys,
// columns = queries), so a query is a lane: its maximum and sum are lane-local but for one exchange
// between the two lane halves, and the probabilities are already the right operand of P V.
//
// Bound in bf16 by matrix and vector instructions one after the other (4 x 8191 positions, 8 heads of 64: 718 us,
// 765 TFLOP/s; per 32 x 32 scores 256 cycles of matrix and some 640 of vector instructions, 765 us if none overlap; 8192
// positions, whose rows are aligned: 675 us), in fp32 by the matrix instruction's rate and unequal lengths (16 x up to 1001
// positions, 2 heads of 96: 101 us, 59 TFLOP/s; all 1001 long: 122 us, 101 TFLOP/s).  Of the variants only fp32 with 128
// channels spills registers (36).
#include "bucket_attention.hpp"
#include "bucket_attention_narrow.hpp"
#include "api_internal.hpp"
#include "bucket_attention_host.hpp"

namespace {
using namespace vkba;

constexpr int FWD_TILE = 64;    // keys of a staged tile
// A bias that a whole block shares enters the exponents as flat - maximum, exactly, while the maximum is rounded with the
// bias in it: they differ by up to half a step of the bias, 16 just below FLAT_MAX, and an exponent is that much too large.
// Ends of the table (bits: left, right) that are larger, but finite, are looked up like near ones.
constexpr float FLAT_MAX = 0x1p29f;
__device__ __forceinline__ int steep_ends(const float* tab, const Dev& p)
{
    auto steep = [](float x) { return fabsf(x) >= FLAT_MAX && fabsf(x) < __builtin_inff(); };
    return __builtin_amdgcn_readfirstlane((steep(tab[0]) ? 1 << BIAS_LEFT : 0) | (steep(tab[2 * p.far_]) ? 1 << BIAS_RIGHT : 0));
}

// KW = 2: half of the waves take the first, half the second 32 keys of every tile (64 queries per workgroup
// instead of 128), each with a maximum, sum and output of its own, joined through LDS at the end.  The staging of
// a tile is then shared by half the work, but there are twice the workgroups.
template <typename T, int DP, int KW>
__global__ __launch_bounds__(NTHR, (sizeof(T) == 2 && DP <= 64 ? 3 : 2))
void bucket_attention_kernel(Dev p)
{
    using F = typename Num<T>::frag;
    constexpr int KT = FWD_TILE, KS = Num<T>::KS, PT = Tile<T, DP, KT>::PT, QW = NWAVE / KW, QT = QW * 32;
    constexpr int NS = KT / 32 / KW;                              // 32-key blocks of a tile per wave
    // the next tile is loaded into registers while the present one is computed; in fp32, where a tile takes four times
    // the matrix cycles, those registers are worth more as a second wave per SIMD
    constexpr bool AHEAD = sizeof(T) == 2;
    constexpr int SP = sizeof(T) == 4 ? 1 : NS;             // of them in one softmax step (fp32: 1, to keep the registers)
    extern __shared__ __align__(16) unsigned char lds[];
    T* ki = reinterpret_cast<T*>(lds);
    T* vi = ki + DP * PT;
    float* tab = reinterpret_cast<float*>(vi + DP * PT);

    const Place at = place(p, (int)blockIdx.x);
    if (!at.any) return;
    const int b = at.b, kvh = at.kvh, g = at.within % p.group, rest = at.within / p.group;
    const int split = rest % p.splits;
    const int qt = p.tiles - 1 - rest / p.splits;           // causal: the longest rows first
    const int head = kvh * p.group + g;
    const Item it = uniform_item(p, b);
    const int l = threadIdx.x & 63, h = l >> 5, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int qw = wave / KW, kw = wave % KW;
    const int q0 = qt * QT + qw * 32, qi = q0 + (l & 31);

    const T* kg = (const T*)p.k + (int64_t)b * p.kb + (int64_t)kvh * p.head_dim * p.kc;
    const T* vg = (const T*)p.v + (int64_t)b * p.vb + (int64_t)kvh * p.head_dim * p.vc;

    // keys this workgroup walks over
    int end = it.nk;
    const int last_q = min(qt * QT + QT, it.nq) - 1;
    if (p.causal) end = clampi(it.start + last_q + 1, 0, end);
    if (qt * QT >= it.nq) end = 0;
    const int first = split * p.per_split * KT;
    end = min(end, first + p.per_split * KT);

    Tile<T, DP, KT> kt, vt;
    F qf[DP / KS];
    if (first < end) {
        OwnRows<T, DP, KT, QW> rows;
        rows.load((const T*)p.q + (int64_t)b * p.qb + (int64_t)head * p.head_dim * p.qc, p.qc, p.head_dim, qt * QT, it.nq);
        if constexpr (AHEAD) {
            kt.load(kg, p.kc, p.head_dim, first, end);
            vt.load(vg, p.vc, p.head_dim, first, end);
        }
        stage_bias(tab, p, head);
        rows.frags(qf, ki, vi, qw);
    }

    f32x16 acc[DP / 32];
    float m = -__builtin_inff(), sum = 0.0f;
#pragma unroll
    for (int blk = 0; blk < DP / 32; ++blk)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[blk][r] = 0.0f;

    const float c = p.c;
    const int pos0 = it.start + q0, pos = pos0 + (l & 31);
    const int steep = p.bias && first < end ? steep_ends(tab, p) : 0;
    for (int j0 = first; j0 < end; j0 += KT) {
        if constexpr (!AHEAD) {
            kt.load(kg, p.kc, p.head_dim, j0, end);
            vt.load(vg, p.vc, p.head_dim, j0, end);
        }
        __syncthreads();
        kt.store(ki);
        vt.store(vi);
        __syncthreads();
        if (AHEAD && j0 + KT < end) {
            kt.load(kg, p.kc, p.head_dim, j0 + KT, end);
            vt.load(vg, p.vc, p.head_dim, j0 + KT, end);
        }
#pragma unroll
        for (int step = 0; step < NS / SP; ++step) {
            const int c0 = 32 * (kw * NS + step * SP), js = j0 + c0;            // this step's keys: SP * 32 from here
            if (js >= end || (p.causal && js > pos0 + 31)) continue;            // none in sight of this wave
            f32x16 s[SP];
#pragma unroll
            for (int i = 0; i < SP; ++i) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[i][r] = 0.0f;
                dot_channels<DP, PT>(s[i], ki, c0 + 32 * i, qf);
            }
            float mul = c, flat = 0.0f;                                         // logit = mul * s + flat
            const int lo = js - (pos0 + 31), hi = js + 32 * SP - 1 - pos0;
            int side = bias_side(p, lo, hi);
            if (steep >> side & 1) side = BIAS_NEAR;
            if (side == BIAS_NEAR) {
                mul = 1.0f;
#pragma unroll
                for (int i = 0; i < SP; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int off = clampi(js + 32 * i + acc_row(r, h) - pos, -p.far_, p.far_);
                        s[i][r] = fmaf(s[i][r], c, tab[off + p.far_]);
                    }
            } else {
                flat = bias_flat(tab, p, side);
            }
            if (js + 32 * SP > end || (p.causal && hi > 0)) {
                const int stop = (p.causal ? min(end, pos + 1) : end) - js;
#pragma unroll
                for (int i = 0; i < SP; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (32 * i + acc_row(r, h) >= stop) s[i][r] = -__builtin_inff();
            }
            float mx = s[0][0];
#pragma unroll
            for (int i = 0; i < SP; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[i][r]);
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            mx = fmaf(mx, mul, flat);                                           // the scale is positive: the maximum stays the maximum
            // m is the exponents' reference, not the exact maximum: it follows when some query of the wave is more
            // than 8 (a factor of 256) above it, so that the sums and the output are rarely scaled anew
            if (__any(mx > m + 8.0f)) {
                const float top = fmaxf(mx, m), alpha = exp2_hw(m - (top == -__builtin_inff() ? 0.0f : top));
                sum *= alpha;
#pragma unroll
                for (int blk = 0; blk < DP / 32; ++blk)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[blk][r] *= alpha;
                m = top;
            }
            const float base = m == -__builtin_inff() ? 0.0f : m;
            const float shift = flat - base;
            float add = 0.0f;
#pragma unroll
            for (int i = 0; i < SP; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[i][r] = exp2_hw(fmaf(s[i][r], mul, shift));
                    add += s[i][r];
                }
            sum += add;
#pragma unroll
            for (int i = 0; i < SP; ++i) dot_positions<DP, PT>(acc, vi, c0 + 32 * i, s[i]);
        }
    }

    float total = sum + __shfl_xor(sum, 32);
    if constexpr (KW == 2) {
        __syncthreads();                                    // the images are free
        float* red = reinterpret_cast<float*>(lds) + qw * (DP + 2) * 32 + (l & 31);
        if (kw == 1) {
#pragma unroll
            for (int blk = 0; blk < DP / 32; ++blk)
#pragma unroll
                for (int r = 0; r < 16; ++r) red[(32 * blk + acc_row(r, h)) * 32] = acc[blk][r];
            red[DP * 32] = m;
            red[(DP + 1) * 32] = total;
        }
        __syncthreads();
        if (kw == 1) return;
        const float m1 = red[DP * 32], t1 = red[(DP + 1) * 32];
        const float mx = fmaxf(m, m1), base = mx == -__builtin_inff() ? 0.0f : mx;
        const float w0 = exp2_hw(m - base), w1 = exp2_hw(m1 - base);
        m = mx;
        total = total * w0 + t1 * w1;
#pragma unroll
        for (int blk = 0; blk < DP / 32; ++blk)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[blk][r] = acc[blk][r] * w0 + red[(32 * blk + acc_row(r, h)) * 32] * w1;
    }
    if (qi >= p.queries) return;
    const bool some = qi < it.nq && !(total == 0.0f);       // NaN in the inputs stays visible
    const int64_t row = ((int64_t)b * p.heads + head) * p.queries + qi;
    if (p.splits == 1) {
        const float inv = 1.0f / total;
        T* og = (T*)p.out + (int64_t)b * p.ob + (int64_t)head * p.head_dim * p.oc + qi;
#pragma unroll
        for (int blk = 0; blk < DP / 32; ++blk)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int d = 32 * blk + acc_row(r, h);
                if (d < p.head_dim) og[(int64_t)d * p.oc] = (T)(some ? acc[blk][r] * inv : 0.0f);
            }
        if (h == 0) p.lse[row] = some ? (m + log2f(total)) * LN2 : -__builtin_inff();
    } else {
        const int64_t rows = (int64_t)p.batch * p.heads * p.queries;
        float* po = p.part_o + ((int64_t)split * p.batch * p.heads + (int64_t)b * p.heads + head) * p.head_dim * p.queries + qi;
#pragma unroll
        for (int blk = 0; blk < DP / 32; ++blk)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int d = 32 * blk + acc_row(r, h);
                if (d < p.head_dim) po[(int64_t)d * p.queries] = acc[blk][r];
            }
        if (h == 0) {
            p.part_ml[((int64_t)split * rows + row) * 2] = some ? m : -__builtin_inff();
            p.part_ml[((int64_t)split * rows + row) * 2 + 1] = some ? total : 0.0f;
        }
    }
}

// Joins the shares of the keys: out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s, m = max m_s.
// One thread per query and channel of a head; the shares' numbers are requested eight at a time.
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
    const int64_t row = bh * p.queries + qi, o_step = (int64_t)p.batch * p.heads * per_head;
    float m = -__builtin_inff(), o = 0.0f, total = 0.0f;
    for (int s0 = 0; s0 < p.splits; s0 += 8) {
        float ms[8], ls[8], os[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t s = min(s0 + i, p.splits - 1);
            const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + (s * rows + row) * 2);
            ms[i] = s0 + i < p.splits ? ml.x : -__builtin_inff();
            ls[i] = s0 + i < p.splits ? ml.y : 0.0f;
            os[i] = p.part_o[s * o_step + bh * per_head + rem];
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, ms[i]);
        const float base = top == -__builtin_inff() ? 0.0f : top, keep = exp2_hw(m - base);
        o *= keep;
        total *= keep;
        m = top;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float w = exp2_hw(ms[i] - base);
            total = fmaf(w, ls[i], total);
            o = ls[i] != 0.0f ? fmaf(w, os[i], o) : o;     // a share without keys left its sums unwritten
        }
    }
    const int b = (int)(bh / p.heads), head = (int)(bh - (int64_t)b * p.heads);
    const bool none = total == 0.0f;
    T* og = (T*)p.out + (int64_t)b * p.ob + ((int64_t)head * p.head_dim + d) * p.oc + qi;
    *og = (T)(none ? 0.0f : o / total);
    if (d == 0) p.lse[row] = none ? -__builtin_inff() : (m + log2f(total)) * LN2;
}

template <typename T, int DP>
int launch(const Dev& d, int kw, hipStream_t st)
{
    const size_t lds = 2 * (size_t)Tile<T, DP, FWD_TILE>::BYTES + vkba_table_bytes(d);
    if constexpr (sizeof(T) == 2)
        if (kw == 1) return vkba_launch<bucket_attention_kernel<T, DP, 1>>(d, vkba_blocks(d), lds, st, "vk_bucket_attention");
    return vkba_launch<bucket_attention_kernel<T, DP, 2>>(d, vkba_blocks(d), lds, st, "vk_bucket_attention");
}

template <typename T>
int by_width(const Dev& d, int kw, hipStream_t st)
{
    switch ((d.head_dim + 31) / 32) {
    case 1: return launch<T, 32>(d, kw, st);
    case 2: return launch<T, 64>(d, kw, st);
    case 3: return launch<T, 96>(d, kw, st);
    default: return launch<T, 128>(d, kw, st);
    }
}

template <typename T>
int narrow_by_width(const Dev& d, hipStream_t st)
{
    const char* what = "vk_bucket_attention";
    const int heads = d.group < 16 ? d.group : 16;              // of which a tile of 16 rows can hold rows
    const size_t tab = (size_t)heads * (2 * d.far_ + 1) * 4;
    auto lds = [&](int dp) { const size_t red = (size_t)NWAVE * (dp + 2) * 16 * 4; return red > tab ? red : tab; };
    switch ((d.head_dim + 31) / 32) {
    case 1: return vkba_launch<bucket_attention_narrow_kernel<T, 32>>(d, vkba_blocks(d), lds(32), st, what);
    case 2: return vkba_launch<bucket_attention_narrow_kernel<T, 64>>(d, vkba_blocks(d), lds(64), st, what);
    case 3: return vkba_launch<bucket_attention_narrow_kernel<T, 96>>(d, vkba_blocks(d), lds(96), st, what);
    default: return vkba_launch<bucket_attention_narrow_kernel<T, 128>>(d, vkba_blocks(d), lds(128), st, what);
    }
}

// Which kernel (kw = 0: the one for few rows), queries per workgroup (128 or, with the waves in two key halves, 64)
// and shares of the keys' length.
//  * Few rows.  That kernel makes 16-row tiles over all rows of a kv head, the other 64-row tiles of one head each, and
//    both read the keys and values once per tile.  In bf16 it pays where it makes fewer tiles (a token, 16 heads on one kv
//    head, 8 x 8192 positions: 29 us against 63) or as many in a part of the chip (16 rows, 128 kv heads, 4096 positions:
//    34 against 34; 512 heads of 1024: 45 against 33); in fp32, whose wide tiles take longer, up to twice as many (32
//    rows, 128 heads: 77 against 102; 64 rows: 133 against 100) unless many short rows fill the chip (512 heads, 8 rows
//    of 64 positions: 29 against 18).  And where few workgroups have little to do: eight bf16 heads of 256 positions,
//    batch 2, 18 against 21; two fp32 heads of 301, 21 against 21, of 697, 33 against 22.
//    A workgroup per CU: a token over 16 x 16384 positions took 207 us with shares for 256, 213 with shares for 512.
//  * Two key halves: fp32 always (half the accumulators per wave; with one, two waves per SIMD do not fit), bf16 where
//    128-row tiles would make no more than one workgroup per CU (8 heads of 128, 2048 positions: 46 us against 53; four
//    times 8 heads of 96, 512 workgroups: 103 against 76) or stay half empty (one row, 512 heads of 1024: 33 against 41).
void plan_forward(const vk_bucket_attention_args* a, Dev& d, int& kw)
{
    const int64_t heads = (int64_t)a->batch * a->heads;
    const int64_t rows = (int64_t)d.group * a->queries;
    int64_t blocks, splits;
    int key_tiles, least;                                       // tiles of the key axis, the fewest in a share
    int row_tiles;
    const bool bf = a->dtype == VK_DTYPE_BF16;
    const int chunk = bf ? 8 : 4;                               // positions of a load there
    const int64_t units = (int64_t)a->batch * a->kv_heads, few = (rows + 15) / 16, wide = (int64_t)d.group * ((a->queries + 63) / 64);
    const bool shared = bf ? few < wide || (few == wide && units * few <= 128)
                           : few <= 2 * wide && (a->keys >= 512 || units * few <= 256);
    if (a->keys >= chunk && (shared || (units * few <= 256 && a->keys <= 320))) {
        const int tk = bf ? 128 : 64;
        kw = 0;
        d.tiles = (int)few;
        row_tiles = d.tiles;
        blocks = units * few;
        key_tiles = (a->keys + tk - 1) / tk;
        least = NWAVE;
        splits = blocks == 0 ? 1 : (256 + blocks - 1) / blocks;
    } else {
        kw = !bf || a->queries <= 64 || heads * ((a->queries + 127) / 128) <= 256 ? 2 : 1;
        d.tiles = (a->queries + 128 / kw - 1) / (128 / kw);
        row_tiles = d.tiles * d.group;
        blocks = heads * d.tiles;
        key_tiles = (a->keys + FWD_TILE - 1) / FWD_TILE;
        least = 2;
        splits = blocks >= 256 || blocks == 0 ? 1 : (512 + blocks - 1) / blocks;
    }
    const int64_t most = (key_tiles + least - 1) / least;
    if (splits > most) splits = most;
    if (splits < 1) splits = 1;
    d.per_split = (int)((key_tiles + splits - 1) / splits);
    if (kw == 0) d.per_split = (d.per_split + NWAVE - 1) / NWAVE * NWAVE;
    if (d.per_split < 1) d.per_split = 1;
    d.splits = (key_tiles + d.per_split - 1) / d.per_split;
    if (d.splits < 1) d.splits = 1;
    vkba_place(d, (int64_t)row_tiles * d.splits);
}

}  // namespace

extern "C" int64_t vk_bucket_attention_workspace_bytes(const vk_bucket_attention_args* a)
{
    vkba::Dev d;
    int rc = vkba_check(a, d, "vk_bucket_attention_workspace_bytes", false), kw;
    if (rc != VK_OK) return rc;
    plan_forward(a, d, kw);
    return d.splits > 1 ? (int64_t)d.splits * a->batch * a->heads * a->queries * (a->head_dim + 2) * 4 : 0;
}

extern "C" int vk_bucket_attention(const vk_bucket_attention_args* a, void* stream)
{
    vkba::Dev d;
    int rc = vkba_check(a, d, "vk_bucket_attention", true), kw;
    if (rc != VK_OK) return rc;
    if (a->batch == 0 || a->queries == 0) return VK_OK;
    if (!a->out || !a->lse) return vk_fail(VK_E_ARG, "vk_bucket_attention: null output");
    if (!vk_rows_apart(a->out_bstride, a->out_cstride, (int64_t)a->heads * a->head_dim, a->queries, a->batch))
        return vk_fail(VK_E_ARG, "vk_bucket_attention: rows of out overlap");
    plan_forward(a, d, kw);
    const int64_t need = d.splits > 1 ? (int64_t)d.splits * a->batch * a->heads * a->queries * (a->head_dim + 2) * 4 : 0;
    if (need > 0 && (!a->workspace || a->workspace_bytes < need))
        return vk_fail(VK_E_WORKSPACE, "vk_bucket_attention: workspace smaller than vk_bucket_attention_workspace_bytes");
    d.part_ml = (float*)a->workspace;
    d.part_o = d.part_ml + (int64_t)d.splits * a->batch * a->heads * a->queries * 2;
    hipStream_t st = (hipStream_t)stream;
    if (kw == 0) rc = a->dtype == VK_DTYPE_BF16 ? narrow_by_width<__bf16>(d, st) : narrow_by_width<float>(d, st);
    else rc = a->dtype == VK_DTYPE_BF16 ? by_width<__bf16>(d, kw, st) : by_width<float>(d, kw, st);
    if (rc != VK_OK || d.splits == 1) return rc;
    const int64_t n = (int64_t)a->batch * a->heads * a->head_dim * a->queries;
    dim3 grid((unsigned)((n + 255) / 256));
    if (a->dtype == VK_DTYPE_BF16) hipLaunchKernelGGL(bucket_attention_join_kernel<__bf16>, grid, dim3(256), 0, st, d);
    else hipLaunchKernelGGL(bucket_attention_join_kernel<float>, grid, dim3(256), 0, st, d);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? VK_OK : vk_fail(VK_E_LAUNCH, hipGetErrorString(e));
}
