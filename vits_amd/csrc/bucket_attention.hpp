#pragma once
// Attention with a learned relative position bias by buckets: what the forward and the backward
// kernels share.
//
//   s_ij = scale * q_i . k_j + bias[h, bucket_of(j - pos_i)],  pos_i = start + i
//   lse_i = log sum_j exp(s_ij),  o_i = sum_j exp(s_ij - lse_i) v_j
//
// Tensors are channel-major (time contiguous), so an LDS image of a tile is [channel][32, 64 or 128 positions].
// Every product of the passes contracts either the channels (scores: rows = positions of the image)
// or the positions (rows = channels of the image), and both read the same image:
//   * contraction over channels: bf16 needs 8 channels of one position in a lane; the transposing
//     LDS read (4 channel rows x 16 positions per 16 lanes) delivers them.  Which 8 channels a
//     k-step takes is free as long as both operands agree, and rows 8 apart are taken, which puts
//     the four rows of a read 16 banks apart (pitch 2 dwords above a multiple of 32): no bank conflicts.  fp32 needs one
//     channel per lane half: a plain row read.
//   * contraction over positions: the other operand is a 32x32 accumulator tile whose lane holds
//     positions 8 * (r / 4) + 4 * half + r % 4 (r = register).  The image is read at exactly those
//     positions, so probabilities go from the softmax straight into the next matrix instruction,
//     without crossing lanes or LDS.
// Softmax statistics and all sums are fp32.  In bf16 the probabilities (and the logit gradients) are
// rounded to bf16 where they enter a matrix instruction: one relative rounding of at most 2^-8 per term,
// of random sign, under sums that are rounded to bf16 once more when they are stored.  Chosen because fp32 products take
// eight times as long and a second bf16 slice of them would double these products: the results' distance from 64 bits,
// in the 2-norm, is 2.1e-3 to 2.4e-3 instead of the 1.7e-3 that storing them in bf16 costs alone.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>
#include "../../include/vits_amd.h"
#include "chunk_load.hpp"

namespace vkba {

typedef float  f32x4  __attribute__((ext_vector_type(4)));
typedef float  f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short  s16x4  __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef chunk_t u32x4;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int NWAVE = 4;        // waves of a workgroup
constexpr int NTHR = 64 * NWAVE;

template <typename T> struct Num;
template <> struct Num<__bf16> {
    static constexpr int KS = 16, EPC = 8, PAD = 4;     // channels per k-step, elements per 16-byte chunk, pitch of an image - positions
    using frag = bf16x8;
};
template <> struct Num<float> {
    static constexpr int KS = 2, EPC = 4, PAD = 2;
    using frag = float;
};

__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(float a, float b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// A [DP channels][KT positions] tile on its way from memory to its LDS image, through registers.
template <typename T, int DP, int KT>
struct Tile {
    static constexpr int E = Num<T>::EPC, PT = KT + Num<T>::PAD, CPR = KT / E; // chunks per row
    static constexpr int ROWS = NTHR / CPR, N = DP / ROWS;                     // rows per pass, passes
    static_assert(DP % ROWS == 0, "whole passes");
    static constexpr int BYTES = DP * PT * (int)sizeof(T);
    u32x4 c[N];
    // Positions t0 .. t0 + KT - 1 of d_real channels; what is at or behind `limit`, and channels up to DP, is zero.
    // A whole tile is loaded without a branch, from uniform row pointers and one 32-bit offset per lane.
    __device__ __forceinline__ void load(const T* base, int64_t cstride, int d_real, int t0, int limit)
    {
        const int row = (int)threadIdx.x / CPR, col = ((int)threadIdx.x % CPR) * E;
        if (t0 + KT <= limit && d_real == DP && cstride < (int64_t)(1 << 24)) {
            const unsigned lane = ((unsigned)row * (unsigned)cstride + (unsigned)col) * (unsigned)sizeof(T);
            const char* p = (const char*)(base + t0);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const char* q = p + (int64_t)i * ROWS * cstride * (int64_t)sizeof(T);
                __builtin_memcpy(&c[i], q + lane, 16);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int d = row + i * ROWS;
            const u32x4 v = load_chunk<T>(base + (int64_t)(d < d_real ? d : d_real - 1) * cstride, t0 + col, limit);
            c[i] = d < d_real ? v : u32x4{0u, 0u, 0u, 0u};
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

// The fragments of the positions col0 + 0..31 of an image, one position per lane, for contraction over channels.
template <int DP, int PT>
__device__ __forceinline__ void read_frags(bf16x8 (&f)[DP / 16], const __bf16* img, int col0)
{
    typedef __attribute__((address_space(3))) s16x4 lds4;
    const int l = threadIdx.x & 63, h = l >> 5;
    const __bf16* p = img + (8 * ((l & 15) >> 2) + 2 * h) * PT + col0 + (l & 16) + 4 * (l & 3);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        const __bf16* ps = p + (32 * (s >> 1) + 4 * (s & 1)) * PT;
        const s16x4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)ps);
        const s16x4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(ps + PT));
        __builtin_memcpy(&f[s], &a0, 8);
        __builtin_memcpy((char*)&f[s] + 8, &a1, 8);
    }
}
template <int DP, int PT>
__device__ __forceinline__ void read_frags(float (&f)[DP / 2], const float* img, int col0)
{
    const int l = threadIdx.x & 63;
    const float* p = img + (l >> 5) * PT + col0 + (l & 31);
#pragma unroll
    for (int s = 0; s < DP / 2; ++s) f[s] = p[2 * s * PT];
}
// A workgroup's own rows (QW waves of 32 positions from t0) as fragments, by way of the two image buffers: 16-byte
// loads of whole rows, where a lane that gathered its own position would touch one row per load (2048 causal
// positions of 128 channels in bf16: 131 us against 199).
template <typename T, int DP, int KT, int QW>
struct OwnRows {
    static constexpr int NT = (QW * 32 + KT - 1) / KT, PT = Tile<T, DP, KT>::PT;
    static_assert(NT <= 2, "two images");
    Tile<T, DP, KT> t[NT];
    __device__ __forceinline__ void load(const T* base, int64_t cstride, int d_real, int t0, int limit)
    {
#pragma unroll
        for (int i = 0; i < NT; ++i) t[i].load(base, cstride, d_real, t0 + i * KT, limit);
    }
    // `slot`: which of the workgroup's 32-position groups this wave takes.  The images are free before and after.
    __device__ __forceinline__ void frags(typename Num<T>::frag (&f)[DP / Num<T>::KS], T* img0, T* img1, int slot) const
    {
        t[0].store(img0);
        if constexpr (NT == 2) t[1].store(img1);
        __syncthreads();
        read_frags<DP, PT>(f, 32 * slot >= KT ? img1 : img0, 32 * slot % KT);
        __syncthreads();
    }
};

// The product of two such fragment sets, summed over the channels in 64 bits (both halves of the wave get the sum).
template <int N>
__device__ __forceinline__ double dot_frags(const bf16x8 (&a)[N], const bf16x8 (&b)[N])
{
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fma((double)(float)a[i][e], (double)(float)b[i][e], s);
    return s + __shfl_xor(s, 32);
}
template <int N>
__device__ __forceinline__ double dot_frags(const float (&a)[N], const float (&b)[N])
{
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fma((double)a[i], (double)b[i], s);
    return s + __shfl_xor(s, 32);
}

// acc (rows: positions col0 + 0..31 of the image, columns: the lanes' positions) += sum over channels.
template <int DP, int PT>
__device__ __forceinline__ void dot_channels(f32x16& acc, const __bf16* img, int col0, const bf16x8 (&f)[DP / 16])
{
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
        acc = mma(a, f[s], acc);
    }
}
template <int DP, int PT>
__device__ __forceinline__ void dot_channels(f32x16& acc, const float* img, int col0, const float (&f)[DP / 2])
{
    const int l = threadIdx.x & 63, h = l >> 5;
    const float* p = img + h * PT + col0 + (l & 31);
#pragma unroll
    for (int s = 0; s < DP / 2; ++s) {
        acc = mma(p[2 * s * PT], f[s], acc);
    }
}

// acc[b] (rows: channels 32 b + 0..31 of the image, columns: the lanes' positions) += sum over the 32
// positions col0.. of image * w, w in accumulator layout (rows: those 32 positions).
template <int DP, int PT>
__device__ __forceinline__ void dot_positions(f32x16 (&acc)[DP / 32], const __bf16* img, int col0, const f32x16& w)
{
    const int l = threadIdx.x & 63, h = l >> 5;
    const __bf16* p = img + (l & 31) * PT + col0 + 4 * h;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
        bf16x8 b;
#pragma unroll
        for (int e = 0; e < 8; ++e) b[e] = (__bf16)w[8 * ks + e];
#pragma unroll
        for (int blk = 0; blk < DP / 32; ++blk) {
            const __bf16* pb = p + blk * 32 * PT + 16 * ks;
            bf16x8 a;
            __builtin_memcpy(&a, __builtin_assume_aligned(pb, 8), 8);
            __builtin_memcpy((char*)&a + 8, __builtin_assume_aligned(pb + 8, 8), 8);
            acc[blk] = mma(a, b, acc[blk]);
        }
    }
}
template <int DP, int PT>
__device__ __forceinline__ void dot_positions(f32x16 (&acc)[DP / 32], const float* img, int col0, const f32x16& w)
{
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
            for (int r = 0; r < 4; ++r) acc[blk] = mma(a[r], w[4 * r4 + r], acc[blk]);
        }
}

template <int N>
__device__ __forceinline__ void flip(bf16x8 (&f)[N], bool neg)
{
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) f[i][e] = neg ? -f[i][e] : f[i][e];
}
template <int N>
__device__ __forceinline__ void flip(float (&f)[N], bool neg)
{
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = neg ? -f[i] : f[i];
}

// Row (position within 32) of accumulator register r in lane half h.
__device__ __forceinline__ constexpr int acc_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }
// Accumulators (32 channels x 32 positions each), times f, to rows of a tensor; g: channel 0, this lane's position.
template <typename T, int NB>
__device__ __forceinline__ void store_rows(T* g, int64_t cstride, int d_real, const f32x16 (&x)[NB], int h, bool valid, float f)
{
#pragma unroll
    for (int blk = 0; blk < NB; ++blk)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int d = 32 * blk + acc_row(r, h);
            if (d < d_real) g[(int64_t)d * cstride] = (T)(valid ? x[blk][r] * f : 0.0f);
        }
}

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
    int units, spread, mix, sort;   // (item, kv head) pairs; a pair's workgroups on one XCD, its pairs side by side; items by their work
    int per_unit, elem;             // bytes of an element
    float* part_o; float* part_ml;  // forward: partial results of the shares
    float* dbias; int kv_blocks, fold;   // backward: bias gradient; workgroups before those that sum it; the order of the dv ones
    int shares; float* part_kv;     // backward: shares of the queries, their sums for dk and dv
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

// The same for the workgroup's own item, in scalar registers: everything that branches on it is uniform.
__device__ __forceinline__ Item uniform_item(const Dev& p, int b)
{
    Item it = item_of(p, b);
    it.nk = __builtin_amdgcn_readfirstlane(it.nk);
    it.nq = __builtin_amdgcn_readfirstlane(it.nq);
    it.start = __builtin_amdgcn_readfirstlane(it.start);
    return it;
}

// Workgroup -> (item, kv head, index within the pair).  Workgroups go round robin over the 8 XCDs; with `spread` all
// workgroups of a pair share one XCD, so the keys and values of a head stay in that XCD's L2 (pairs are dealt back and
// forth, 0..7 then 7..0).  With `mix` an XCD's pairs go on side by side instead of one after the other, so that the
// longest workgroups of all of them come first.  With lengths, items go in the order of their work, the largest first: the XCDs then get
// like shares, and what starts last is short.
struct Place { int b, kvh, within; bool any; };
__device__ __forceinline__ Place place(const Dev& p, int id)
{
    const int kv_heads = p.heads / p.group;
    int unit;
    Place r;
    if (p.spread) {
        const int slot = id >> 3, rounds = (p.units + 7) >> 3;
        const int turn = slot / rounds;
        const int round = p.mix ? (slot + turn) % rounds : slot / p.per_unit;
        unit = 8 * round + ((round & 1) ? 7 - (id & 7) : id & 7);
        r.within = p.mix ? turn : slot - round * p.per_unit;
    } else {
        unit = id / p.per_unit;
        r.within = id - unit * p.per_unit;
    }
    unit = __builtin_amdgcn_readfirstlane(unit);
    r.within = __builtin_amdgcn_readfirstlane(r.within);
    r.any = unit < p.units;
    r.b = unit / kv_heads;
    r.kvh = unit - r.b * kv_heads;
    if (p.sort && r.any) {                                  // at most 64 items: a lane each
        const int lane = (int)threadIdx.x & 63;
        const Item it = item_of(p, lane < p.batch ? lane : p.batch - 1);
        const float mine = (float)it.nq * (float)it.nk;
        int rank = 0;
        for (int o = 0; o < p.batch; ++o) {
            const float other = __shfl(mine, o);
            rank += other > mine || (other == mine && o < lane);
        }
        const unsigned long long hit = __ballot(lane < p.batch && rank == r.b);
        r.b = __builtin_amdgcn_readfirstlane(hit ? (int)__builtin_ctzll(hit) : 0);     // ranks are a permutation: exactly one
    }
    return r;
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

// Offsets lo .. hi (key - query) of a block against the bias table.  Beyond `far` on either side all of it shares
// one value; without a bias the table is not there.
enum { BIAS_LEFT, BIAS_RIGHT, BIAS_NEAR, BIAS_NONE };
__device__ __forceinline__ int bias_side(const Dev& p, int lo, int hi)
{
    return !p.bias ? BIAS_NONE : hi <= -p.far_ ? BIAS_LEFT : lo >= p.far_ ? BIAS_RIGHT : BIAS_NEAR;
}
__device__ __forceinline__ float bias_flat(const float* tab, const Dev& p, int side)
{
    return side == BIAS_LEFT ? tab[0] : side == BIAS_RIGHT ? tab[2 * p.far_] : 0.0f;
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
