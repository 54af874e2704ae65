#pragma once
// Host side shared by the forward and the backward pass of the bucketed-bias attention: argument
// checks, placement of the workgroups, launches.
#include <atomic>
#include <math.h>
#include <stdio.h>
#include "bucket_attention.hpp"
#include "api_internal.hpp"
#include "conv_mfma.hpp"      // vk_allow_lds

inline int vkba_fail(int code, const char* what, const char* msg)
{
    char buf[256];
    snprintf(buf, sizeof(buf), "%s: %s", what, msg);
    return vk_fail(code, buf);
}

// Fills the device struct with everything that does not depend on the pass.  `pointers`: also check them
// (the workspace queries look at the sizes only).
inline int vkba_check(const vk_bucket_attention_args* a, vkba::Dev& d, const char* what, bool pointers)
{
    if (!a) return vkba_fail(VK_E_ARG, what, "null argument struct");
    if (a->batch < 0 || a->queries < 0 || a->keys < 0 || a->heads <= 0 || a->kv_heads <= 0 || a->heads % a->kv_heads)
        return vkba_fail(VK_E_ARG, what, "bad batch, length or head count (heads must be a multiple of kv_heads)");
    if (a->dtype != VK_DTYPE_F32 && a->dtype != VK_DTYPE_BF16) return vkba_fail(VK_E_UNSUPPORTED, what, "dtype must be VK_DTYPE_F32 or VK_DTYPE_BF16");
    if (a->head_dim < 1 || a->head_dim > VK_BUCKET_MAX_HEAD_DIM) return vkba_fail(VK_E_UNSUPPORTED, what, "head_dim must be 1..128");
    if ((int64_t)a->batch * a->heads > 0x7fffff) return vkba_fail(VK_E_UNSUPPORTED, what, "batch x heads beyond 2^23");
    if (a->queries > VK_BUCKET_MAX_LENGTH || a->keys > VK_BUCKET_MAX_LENGTH) return vkba_fail(VK_E_UNSUPPORTED, what, "length beyond VK_BUCKET_MAX_LENGTH");
    if (!(a->scale > 0.0f && a->scale < 1e30f)) return vkba_fail(VK_E_ARG, what, "scale must be positive and finite");
    if (a->has_bias && (a->buckets < 1 || a->max_distance < 1 || a->max_distance > VK_BUCKET_MAX_DISTANCE))
        return vkba_fail(VK_E_UNSUPPORTED, what, "bias needs at least one bucket and max_distance in 1..VK_BUCKET_MAX_DISTANCE");
    if (pointers) {
        if ((uintptr_t)a->workspace & 15) return vkba_fail(VK_E_ARG, what, "workspace must be 16-byte aligned");
        if (a->has_bias && (!a->bias || !a->bucket_of)) return vkba_fail(VK_E_ARG, what, "null bias or bucket table");
        if (a->batch && a->queries && !a->q) return vkba_fail(VK_E_ARG, what, "null queries");
        if (a->batch && a->keys && (!a->k || !a->v)) return vkba_fail(VK_E_ARG, what, "null keys or values");
        if (!vk_strides_ok(a->q_bstride, a->q_cstride) || !vk_strides_ok(a->k_bstride, a->k_cstride)
            || !vk_strides_ok(a->v_bstride, a->v_cstride) || !vk_strides_ok(a->out_bstride, a->out_cstride))
            return vkba_fail(VK_E_ARG, what, "a stride of q, k, v or out is negative or beyond 2^40");
    }
    memset(&d, 0, sizeof(d));
    d.q = a->q; d.qb = a->q_bstride; d.qc = a->q_cstride;
    d.k = a->k; d.kb = a->k_bstride; d.kc = a->k_cstride;
    d.v = a->v; d.vb = a->v_bstride; d.vc = a->v_cstride;
    d.out = a->out; d.o = a->out; d.ob = a->out_bstride; d.oc = a->out_cstride;
    d.lse = a->lse; d.lse_in = a->lse;
    d.dout = a->dout; d.dob = a->dout_bstride; d.doc = a->dout_cstride;
    d.dq = a->dq; d.dqb = a->dq_bstride; d.dqc = a->dq_cstride;
    d.dk = a->dk; d.dkb = a->dk_bstride; d.dkc = a->dk_cstride;
    d.dv = a->dv; d.dvb = a->dv_bstride; d.dvc = a->dv_cstride;
    d.bias = a->has_bias ? a->bias : nullptr;
    d.bucket_of = a->bucket_of;
    d.nk = a->key_lengths; d.nq = a->query_lengths; d.start = a->query_start;
    d.batch = a->batch; d.heads = a->heads; d.group = a->heads / a->kv_heads; d.head_dim = a->head_dim;
    d.queries = a->queries; d.keys = a->keys;
    d.buckets = a->has_bias ? a->buckets : 0;
    d.far_ = a->has_bias ? a->max_distance : 0;
    d.causal = a->causal != 0;
    d.scale = a->scale;
    d.c = a->scale * vkba::LOG2E;
    d.units = a->batch * a->kv_heads;
    d.elem = a->dtype == VK_DTYPE_BF16 ? 2 : 4;
    return VK_OK;
}

// `per_unit` workgroups for every (item, kv head) pair.  The pairs are dealt over the XCDs where that
// leaves no XCD more than a tenth above the average; few pairs go round robin instead.
inline void vkba_place(vkba::Dev& d, int64_t per_unit)
{
    d.per_unit = (int)(per_unit > 0x7fffffff ? 0x7fffffff : per_unit);
    const int64_t rounds = (d.units + 7) / 8;
    d.spread = d.units >= 8 && rounds * 8 * 10 <= (int64_t)d.units * 11;
    // causal: tiles differ in length most, and an XCD's pairs side by side (2048 causal positions: 128 -> 120 us) are
    // worth it while their keys and values fit its 4 MiB of L2; padded batches alone lose by it (16 x 1001 fp32: 102 -> 121)
    d.mix = d.spread && d.causal
            && rounds * (int64_t)d.head_dim * 2 * (d.keys > d.queries ? d.keys : d.queries) * d.elem <= 4 << 20;
    d.sort = (d.nk || d.nq) && d.batch > 1 && d.batch <= 64;
}
inline int64_t vkba_blocks(const vkba::Dev& d)
{
    return (int64_t)d.per_unit * (d.spread ? (d.units + 7) / 8 * 8 : d.units);
}

inline size_t vkba_table_bytes(const vkba::Dev& d) { return ((size_t)(2 * d.far_ + 1) * 4 + 15) & ~(size_t)15; }

template <auto KERNEL>
int vkba_launch(const vkba::Dev& d, int64_t blocks, size_t lds, hipStream_t st, const char* what)
{
    if (blocks <= 0) return VK_OK;
    if (blocks * vkba::NTHR > 0xffffffffLL) return vkba_fail(VK_E_UNSUPPORTED, what, "too many workgroups");    // the limit of a grid, in threads
    static std::atomic<unsigned long long> raised{0};
    hipError_t e = vk_allow_lds(KERNEL, lds, raised);
    if (e != hipSuccess) return vkba_fail(VK_E_LAUNCH, what, hipGetErrorString(e));
    hipLaunchKernelGGL(KERNEL, dim3((unsigned)blocks), dim3(vkba::NTHR), lds, st, d);
    e = hipGetLastError();
    return e == hipSuccess ? VK_OK : vkba_fail(VK_E_LAUNCH, what, hipGetErrorString(e));
}
