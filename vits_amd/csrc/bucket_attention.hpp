#pragma once
// Attention with a learned relative position bias by buckets: what the forward and the backward
// kernels share.
//
//   s_ij = scale * q_i . k_j + bias[h, bucket_of(j - pos_i)],  pos_i = start + i
//   lse_i = log sum_j exp(s_ij),  o_i = sum_j exp(s_ij - lse_i) v_j
//
// Tensors are channel-major (time contiguous), so an LDS image of a tile is [channel][64 positions].
// Every product of the passes contracts either the channels (scores: rows = positions of the image)
// or the positions (rows = channels of the image), and both read the same image:
//   * contraction over channels: bf16 needs 8 channels of one position in a lane; the transposing
//     LDS read (4 channel rows x 16 positions per 16 lanes) delivers them.  Which 8 channels a
//     k-step takes is free as long as both operands agree, and rows 8 apart are taken, which puts
//     the four rows of a read 16 banks apart (pitch 34 dwords): no bank conflicts.  fp32 needs one
//     channel per lane half: a plain row read.
//   * contraction over positions: the other operand is a 32x32 accumulator tile whose lane holds
//     positions 8 * (r / 4) + 4 * half + r % 4 (r = register).  The image is read at exactly those
//     positions, so probabilities go from the softmax straight into the next matrix instruction,
//     without crossing lanes or LDS.
// Softmax statistics and all sums are fp32.  In bf16 the probabilities (and the logit gradients) are
// rounded to bf16 where they enter a matrix instruction: one relative rounding of at most 2^-8 per term,
// of random sign, under sums that are rounded to bf16 once more when they are stored.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>
#include "../../include/vits_amd.h"

namespace vkba {

typedef float  f32x4  __attribute__((ext_vector_type(4)));
typedef float  f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short  s16x4  __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int KT = 64;          // positions of a staged tile
constexpr int NWAVE = 4;        // waves of a workgroup
constexpr int NTHR = 64 * NWAVE;

template <typename T> struct Num;
template <> struct Num<__bf16> {
    static constexpr int KS = 16, EPC = 8, PT = 68;     // channels per k-step, elements per 16-byte chunk, image pitch
    using frag = bf16x8;
};
template <> struct Num<float> {
    static constexpr int KS = 2, EPC = 4, PT = 66;
    using frag = float;
};

__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(float a, float b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// 16 bytes of a row at position t; positions at or behind `limit` are zero and not read.  Rows of odd
// length start anywhere, so the load is declared unaligned (the memory system takes it as one access).
template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const T* row, int t, int limit)
{
    constexpr int E = Num<T>::EPC;
    u32x4 r = {0u, 0u, 0u, 0u};
    if (t + E <= limit) {
        __builtin_memcpy(&r, row + t, 16);
    } else if (t < limit) {
        T tmp[E];
#pragma unroll
        for (int e = 0; e < E; ++e) tmp[e] = t + e < limit ? row[t + e] : (T)0.0f;
        __builtin_memcpy(&r, tmp, 16);
    }
    return r;
}

// A [DP channels][KT positions] tile on its way from memory to its LDS image, through registers.
template <typename T, int DP>
struct Tile {
    static constexpr int E = Num<T>::EPC, PT = Num<T>::PT, CPR = KT / E;      // chunks per row
    static constexpr int ROWS = NTHR / CPR, N = DP / ROWS;                     // rows per pass, passes
    static constexpr int BYTES = DP * PT * (int)sizeof(T);
    u32x4 c[N];
    __device__ __forceinline__ void load(const T* base, int64_t cstride, int d_real, int t0, int limit)
    {
        const int row = (int)threadIdx.x / CPR, t = t0 + ((int)threadIdx.x % CPR) * E;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int d = row + i * ROWS;
            c[i] = d < d_real ? load_chunk<T>(base + (int64_t)d * cstride, t, limit) : u32x4{0u, 0u, 0u, 0u};
        }
    }
    __device__ __forceinline__ void store(T* img) const
    {
        const int row = (int)threadIdx.x / CPR, col = ((int)threadIdx.x % CPR) * E;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            u32x2* p = reinterpret_cast<u32x2*>(img + (row + i * ROWS) * PT + col);
            p[0] = u32x2{c[i][0], c[i][1]};
            p[1] = u32x2{c[i][2], c[i][3]};
        }
    }
};

// Channel of element e of k-step s in lane half h (the order both operands of a contraction over
// channels use).
__device__ __forceinline__ constexpr int bf16_channel(int s, int h, int e)
{
    return 32 * (s >> 1) + 8 * (e & 3) + 4 * (s & 1) + 2 * h + (e >> 2);
}

// The fragments of one position per lane (col: pointer to its channel 0), for contraction over channels.
template <int DP>
__device__ __forceinline__ void load_frags(bf16x8 (&f)[DP / 16], const __bf16* col, int64_t cstride, int d_real, bool valid)
{
    const int h = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int d = bf16_channel(s, h, e);
            f[s][e] = (valid && d < d_real) ? col[(int64_t)d * cstride] : (__bf16)0.0f;
        }
}
template <int DP>
__device__ __forceinline__ void load_frags(float (&f)[DP / 2], const float* col, int64_t cstride, int d_real, bool valid)
{
    const int h = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int s = 0; s < DP / 2; ++s) {
        const int d = 2 * s + h;
        f[s] = (valid && d < d_real) ? col[(int64_t)d * cstride] : 0.0f;
    }
}

// acc[n] (rows: positions col0 + 0..31 of the image, columns: the lanes' positions) += sum over channels.
template <int DP, int N>
__device__ __forceinline__ void dot_channels(f32x16 (&acc)[N], const __bf16* img, int col0, const bf16x8 (&f)[N][DP / 16])
{
    constexpr int PT = Num<__bf16>::PT;
    const int l = threadIdx.x & 63, h = l >> 5;
    const int row = 8 * ((l & 15) >> 2) + 2 * h, col = col0 + (l & 16) + 4 * (l & 3);
    const __bf16* p = img + row * PT + col;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        typedef __attribute__((address_space(3))) s16x4 lds4;
        const __bf16* ps = p + (32 * (s >> 1) + 4 * (s & 1)) * PT;
        const s16x4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)ps);
        const s16x4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(ps + PT));
        bf16x8 a;
        __builtin_memcpy(&a, &a0, 8);
        __builtin_memcpy((char*)&a + 8, &a1, 8);
#pragma unroll
        for (int n = 0; n < N; ++n) acc[n] = mma(a, f[n][s], acc[n]);
    }
}
template <int DP, int N>
__device__ __forceinline__ void dot_channels(f32x16 (&acc)[N], const float* img, int col0, const float (&f)[N][DP / 2])
{
    constexpr int PT = Num<float>::PT;
    const int l = threadIdx.x & 63, h = l >> 5;
    const float* p = img + h * PT + col0 + (l & 31);
#pragma unroll
    for (int s = 0; s < DP / 2; ++s) {
        const float a = p[2 * s * PT];
#pragma unroll
        for (int n = 0; n < N; ++n) acc[n] = mma(a, f[n][s], acc[n]);
    }
}

// acc[n][b] (rows: channels 32 b + 0..31 of the image, columns: the lanes' positions) += sum over the 32
// positions col0.. of image * w[n], w[n] in accumulator layout (rows: those 32 positions).
template <int DP, int N>
__device__ __forceinline__ void dot_positions(f32x16 (&acc)[N][DP / 32], const __bf16* img, int col0, const f32x16 (&w)[N])
{
    constexpr int PT = Num<__bf16>::PT;
    const int l = threadIdx.x & 63, h = l >> 5;
    const __bf16* p = img + (l & 31) * PT + col0 + 4 * h;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
        bf16x8 b[N];
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < 8; ++e) b[n][e] = (__bf16)w[n][8 * ks + e];
#pragma unroll
        for (int blk = 0; blk < DP / 32; ++blk) {
            const __bf16* pb = p + blk * 32 * PT + 16 * ks;
            bf16x8 a;
            __builtin_memcpy(&a, __builtin_assume_aligned(pb, 8), 8);
            __builtin_memcpy((char*)&a + 8, __builtin_assume_aligned(pb + 8, 8), 8);
#pragma unroll
            for (int n = 0; n < N; ++n) acc[n][blk] = mma(a, b[n], acc[n][blk]);
        }
    }
}
template <int DP, int N>
__device__ __forceinline__ void dot_positions(f32x16 (&acc)[N][DP / 32], const float* img, int col0, const f32x16 (&w)[N])
{
    constexpr int PT = Num<float>::PT;
    const int l = threadIdx.x & 63, h = l >> 5;
    const float* p = img + (l & 31) * PT + col0 + 4 * h;
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4)
#pragma unroll
        for (int blk = 0; blk < DP / 32; ++blk) {
            const float* pb = p + blk * 32 * PT + 8 * r4;
            float a[4];
            __builtin_memcpy(a, __builtin_assume_aligned(pb, 8), 8);
            __builtin_memcpy(a + 2, __builtin_assume_aligned(pb + 2, 8), 8);
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int n = 0; n < N; ++n) acc[n][blk] = mma(a[r], w[n][4 * r4 + r], acc[n][blk]);
        }
}

// Row (position within 32) of accumulator register r in lane half h.
__device__ __forceinline__ constexpr int acc_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

struct Dev {
    const void* q; const void* k; const void* v; const void* o; const void* dout;
    void* out; void* dq; void* dk; void* dv;
    const float* lse_in; float* lse;
    int64_t qb, qc, kb, kc, vb, vc, ob, oc, dob, doc, dqb, dqc, dkb, dkc, dvb, dvc;
    const float* bias; const int32_t* bucket_of;
    const int64_t* nk; const int64_t* nq; const int64_t* start;
    int batch, heads, group, head_dim, queries, keys, buckets, far_, causal;
    float scale, c;                 // c = scale * log2(e)
    int tiles, splits, per_split;   // row tiles of a head, shares of the other axis, its tiles per share
    int units, spread;              // (item, kv head) pairs; 1: a pair's workgroups on one XCD
    int per_unit;
    float* part_o; float* part_ml;  // forward: partial results of the shares
    float* delta; float* part_bias; // backward: row sums of out * dout; diagonal sums of the logit gradients
};

// Lengths and positions of item b, clamped to what the tensors hold.
struct Item { int nk, nq, start; };
__device__ __forceinline__ Item item_of(const Dev& p, int b)
{
    Item it;
    auto clamp = [](int64_t v, int hi) { return (int)(v < 0 ? 0 : v > hi ? hi : v); };
    it.nk = p.nk ? clamp(p.nk[b], p.keys) : p.keys;
    it.nq = p.nq ? clamp(p.nq[b], p.queries) : p.queries;
    it.start = 0;
    if (p.start) { const int64_t s = p.start[b]; it.start = (int)(s < -(1 << 29) ? -(1 << 29) : s > (1 << 29) ? (1 << 29) : s); }
    return it;
}

// Workgroup -> (unit, index within the unit).  Workgroups go round robin over the 8 XCDs; with `spread`
// all workgroups of a unit share one XCD, so the keys and values of a head stay in that XCD's L2.
__device__ __forceinline__ bool place(const Dev& p, int& unit, int& within)
{
    const int id = (int)blockIdx.x;
    if (p.spread) {
        const int slot = id >> 3;
        unit = (id & 7) + 8 * (slot / p.per_unit);
        within = slot % p.per_unit;
        return unit < p.units;
    }
    unit = id / p.per_unit;
    within = id - unit * p.per_unit;
    return true;
}

// bias by offset (in units of log2) of one head into LDS: tab[o + far] for o = -far .. far.
__device__ __forceinline__ void stage_bias(float* tab, const Dev& p, int head)
{
    if (!p.bias) return;
    for (int o = (int)threadIdx.x; o < 2 * p.far_ + 1; o += (int)blockDim.x) {
        int b = p.bucket_of[o];
        b = b < 0 ? 0 : b >= p.buckets ? p.buckets - 1 : b;
        tab[o] = p.bias[(int64_t)head * p.buckets + b] * LOG2E;
    }
}

// Offsets (row - column or column - row in absolute positions) of one 32 x 32 block against the bias table.
// Beyond `far` on either side the whole block shares one value.
struct BlockBias { bool near_; float flat; };
__device__ __forceinline__ BlockBias block_bias(const float* tab, const Dev& p, int lo, int hi)
{
    BlockBias r{false, 0.0f};
    if (!p.bias) return r;
    if (hi <= -p.far_) r.flat = tab[0];
    else if (lo >= p.far_) r.flat = tab[2 * p.far_];
    else r.near_ = true;
    return r;
}

// LDS written by some lanes of a wave and read by others: a wave's LDS accesses complete in order, so only
// the compiler has to keep them in order.
__device__ __forceinline__ void wave_lds_fence()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

}  // namespace vkba
