// attn.cuh -- what the attention operators share (kv_cache.cu, attn_prefill.cu,
// attn_decode.cu): element types, the paged cache as kernels see it, argument checks.
#pragma once

#include "../../include/amoe.h"
#include "amoe_internal.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>
#include <cmath>
#include <string>

namespace amoe {
namespace attn {

constexpr int kMaxGroup = 128;
constexpr int kMaxPageSize = 4096;
constexpr float kLog2e = 1.4426950408889634f;

// Weights of the softmax meet the values in 16 bits.  A running maximum that is left as it is until a weight has
// outgrown it by 2^lazy gives weights up to 2^lazy; float32 sums hold 2^8, and bf16 has float32's exponents.  f16 does
// not: below 2^-14 it loses bits and below 2^-25 everything, while the sum in the denominator keeps it, so that a long
// flat tail beside one large weight counts short (131071 keys at 2^-25.1 gave 0 of 0.0036).  Its weights therefore carry
// the factor 2^shift, which brings the largest to 2^15 (65504 is the last): whole precision down to 2^-25 of the row's
// largest weight, 2^-36 of it lost of a key below.  The less the maximum may lag the wider that range, and the more
// often the sums are rescaled: 8192 tokens of 64 f16 heads 690 us with 2^8, 697 with 2^4, 728 with 2^2, 777 with 1;
// decode of 48 sequences of 4096-8192 over E4M3 66.6 and 66.7 us with 2^8 and 2^4, 2 % and 6 % more with 2^2 and 1.
__host__ __device__ constexpr float weight_lazy(int type) { return type == AMOE_GGUF_F16 ? 4.0f : 8.0f; }
__host__ __device__ constexpr float weight_shift(int type) { return type == AMOE_GGUF_F16 ? 15.0f - weight_lazy(type) : 0.0f; }

// ---- device side -------------------------------------------------------------------
// Packed rows with strides in bytes.
struct RowsDev {
    char *p;
    int64_t ts, hs;
};

struct CacheDev {
    char *k, *v;
    uint8_t *ks, *vs;
    int32_t *status;
    const int32_t *table;
    int64_t pages;
    int table_stride, shift, heads;  // page_size = 1 << shift
};

// The sequences of packed rows t, t + 1, ... t + N - 1: how many end at or before each (empty sequences before a row's
// share its start).  Always in [0, seqs), whatever cu holds; the caller checks that the sequence holds the row.  A whole
// warp calls it, with a load for every 32 sequences instead of a chain of them; the host, for checks, looks at the same
// 32 in turn.
template <int N>
__host__ __device__ __forceinline__ void find_seqs(const int32_t *cu, int seqs, int t, int (&s)[N]) {
#pragma unroll
    for (int k = 0; k < N; ++k) s[k] = 0;
    for (int s0 = 0; s0 < seqs; s0 += 32) {
        auto end_of = [&](int i) { return s0 + i < seqs ? cu[s0 + i + 1] : INT_MAX; };
#ifdef __CUDA_ARCH__
        const int end = end_of(threadIdx.x % 32);
        auto ended = [&](int row) { return __ballot_sync(0xffffffffu, end <= row); };
        auto count = [](uint32_t bits) { return __popc(bits); };
#else
        auto ended = [&](int row) {
            uint32_t bits = 0;
            for (int i = 0; i < 32; ++i) bits |= (uint32_t)(end_of(i) <= row) << i;
            return bits;
        };
        auto count = [](uint32_t bits) { return __builtin_popcount(bits); };
#endif
        uint32_t bits = 0;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            bits = ended(t + k);
            const int upto = s[k] + count(bits);
            s[k] = upto < seqs ? upto : seqs - 1;
        }
        if (bits != 0xffffffffu) break;  // the last row's sequence, and so every one's, is found
    }
}

// One row's, on the host.
inline int find_seq(const int32_t *cu, int seqs, int t) {
    int s[1];
    find_seqs(cu, seqs, t, s);
    return s[0];
}

// Page of position pos (>= 0) of sequence s, or the negated status bit where the table has none.
__host__ __device__ inline int lookup_page(const CacheDev &c, int s, int64_t pos) {
    const int64_t i = pos >> c.shift;
    if (i >= c.table_stride) return -AMOE_KV_PAST_TABLE;
    const int page = c.table[(int64_t)s * c.table_stride + i];
    return page >= 0 && page < c.pages ? page : -AMOE_KV_BAD_PAGE;
}

// The same with the bit set in the cache's status.
__device__ __forceinline__ int page_of(const CacheDev &c, int s, int64_t pos) {
    const int page = lookup_page(c, s, pos);
    if (page < 0) atomicOr(c.status, -page);
    return page;
}

// The last of `fills` fills (the i-th goes to stage i % stages) that went to this stage; -1: none did.
__host__ __device__ inline int last_fill(int fills, int stage, int stages) {
    return fills > stage ? (fills - 1 - stage) / stages * stages + stage : -1;
}

// Row index of (page, head, slot) in the pages.
__host__ __device__ inline int64_t cache_row(const CacheDev &c, int page, int head, int64_t pos) {
    return ((((int64_t)page * c.heads + head) << c.shift) | (pos & ((1 << c.shift) - 1)));
}

template <int TYPE>
__device__ __forceinline__ void load8(const char *p, float (&x)[8]) {
    if constexpr (TYPE == AMOE_GGUF_F32) {
        const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const uint4 w = *reinterpret_cast<const uint4 *>(p);
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float2 f;
            if constexpr (TYPE == AMOE_GGUF_F16) f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
            else f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&u[i]));
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
}

template <int TYPE>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (TYPE == AMOE_GGUF_F16) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}

template <int TYPE>
__device__ __forceinline__ void store8(char *p, const float (&x)[8]) {
    if constexpr (TYPE == AMOE_GGUF_F32) {
        reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        *reinterpret_cast<uint4 *>(p) = make_uint4(pack2<TYPE>(x[0], x[1]), pack2<TYPE>(x[2], x[3]),
                                                   pack2<TYPE>(x[4], x[5]), pack2<TYPE>(x[6], x[7]));
    }
}

// Element size of a type known at run time, and a store that branches on it (uniform).
__host__ __device__ __forceinline__ int elem_size(int type) {
    return type == AMOE_GGUF_F32 ? 4 : type == AMOE_KV_E4M3 ? 1 : 2;
}
__device__ __forceinline__ void store8_any(char *p, int type, const float (&x)[8]) {
    if (type == AMOE_GGUF_F32) store8<AMOE_GGUF_F32>(p, x);
    else if (type == AMOE_GGUF_F16) store8<AMOE_GGUF_F16>(p, x);
    else store8<AMOE_GGUF_BF16>(p, x);
}

// Two E4M3 codes -> f16x2 (exact: every code is an f16 value).
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
    uint32_t r;
    asm("{\n .reg .b16 t;\n cvt.u16.u32 t, %1;\n cvt.rn.f16x2.e4m3x2 %0, t;\n}" : "=r"(r) : "r"(two));
    return r;
}

// Four codes of a word, the first two and the last two.
__device__ __forceinline__ void e4m3x4_to_f16x2(uint32_t four, uint32_t &lo, uint32_t &hi) {
    asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}"
        : "=r"(lo), "=r"(hi)
        : "r"(four));
}

// ---- host side ----------------------------------------------------------------------
inline int reject(const std::string &msg) {
    set_thread_error(msg);
    return AMOE_ERR_INVALID;
}

inline int cuda_error(cudaError_t e, const char *what) {
    set_thread_error(std::string(what) + ": " + cudaGetErrorString(e));
    return e == cudaErrorMemoryAllocation ? AMOE_ERR_NOMEM : AMOE_ERR_CUDA;
}

// Makes `device` current for a call and gives the thread back the device it had.
struct DeviceScope {
    int prev = -1;
    cudaError_t enter(int device) {
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        return prev == device ? cudaSuccess : cudaSetDevice(device);
    }
    ~DeviceScope() {
        int now = -1;
        if (prev >= 0 && cudaGetDevice(&now) == cudaSuccess && now != prev) cudaSetDevice(prev);
    }
};

inline bool float_type(int type) {
    return type == AMOE_GGUF_F32 || type == AMOE_GGUF_F16 || type == AMOE_GGUF_BF16;
}

// Rows `name` with elements of `type` (-1: any float type), heads heads.  AMOE_OK or an error.
inline int check_rows(const amoe_rows *r, const char *name, int head_dim, int heads, int tokens, int type) {
    const std::string n(name);
    if (!r || !r->data) return reject(n + " must not be NULL");
    if (!float_type(r->type) || (type >= 0 && r->type != type))
        return reject(n + " has element type " + std::to_string(r->type) + ", which this call does not take");
    if (heads > 0 && r->heads != heads)
        return reject(n + " has " + std::to_string(r->heads) + " heads, want " + std::to_string(heads));
    if (r->heads < 1) return reject(n + " must have at least one head");
    const int per16 = 16 / elem_size(r->type);
    if ((reinterpret_cast<uintptr_t>(r->data) & 15) || (r->heads > 1 && r->head_stride % per16) ||
        (tokens > 1 && r->token_stride % per16))
        return reject(n + ": data and strides must be multiples of 16 bytes");
    if (r->token_stride < 0 || r->head_stride < 0) return reject(n + ": strides must not be negative");
    // far from where 64-bit byte offsets could overflow
    const int64_t lim = INT64_MAX / 64;
    if ((tokens > 0 && r->token_stride > lim / tokens) || r->head_stride > lim / r->heads || head_dim > 4096)
        return reject(n + ": strides too large");
    return AMOE_OK;
}

inline RowsDev rows_dev(const amoe_rows *r) {
    if (!r) return {nullptr, 0, 0};
    const int64_t e = elem_size(r->type);
    return {static_cast<char *>(r->data), r->token_stride * e, r->head_stride * e};
}

inline int check_head_dim(int head_dim) {
    if (head_dim != 64 && head_dim != 128)
        return reject("head_dim " + std::to_string(head_dim) + " is not 64 or 128");
    return AMOE_OK;
}

inline int check_group(int q_heads, int kv_heads) {
    if (kv_heads < 1 || q_heads < 1 || q_heads % kv_heads)
        return reject("query heads must be a positive multiple of kv heads");
    if (q_heads / kv_heads > kMaxGroup)
        return reject("more than " + std::to_string(kMaxGroup) + " query heads to one kv head");
    return AMOE_OK;
}

inline int check_attn(const amoe_attn *a) {
    if (!a) return reject("attn must not be NULL");
    if (a->window < 0) return reject("sliding window must be non-negative");
    if (!(a->scale >= 0.0f) || std::isinf(a->scale * kLog2e)) return reject("scale must be finite and non-negative");
    return AMOE_OK;
}

inline float attn_scale(const amoe_attn *a, int head_dim) {
    return a->scale > 0.0f ? a->scale : 1.0f / std::sqrt((float)head_dim);
}

inline int check_cache(const amoe_kv_cache *c, const amoe_kv_seqs *s) {
    if (!c) return reject("cache must not be NULL");
    if (int rc = check_head_dim(c->head_dim)) return rc;
    if (c->type != AMOE_GGUF_F16 && c->type != AMOE_GGUF_BF16 && c->type != AMOE_KV_E4M3)
        return reject("cache type " + std::to_string(c->type) + " is not F16, BF16 or E4M3");
    if (c->page_size < 1 || c->page_size > kMaxPageSize || (c->page_size & (c->page_size - 1)))
        return reject("page_size must be a power of two up to " + std::to_string(kMaxPageSize));
    if (c->kv_heads < 1) return reject("kv_heads must be positive");
    if (c->pages < 1 || c->pages > INT_MAX) return reject("pages outside [1, 2^31)");
    if (c->pages * c->page_size > (int64_t)UINT32_MAX / c->kv_heads) return reject("cache of 2^32 rows or more");
    if (!c->k || !c->v || !c->status) return reject("cache k, v and status must not be NULL");
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15)
        return reject("cache k and v must be 16-byte aligned");
    if (c->type == AMOE_KV_E4M3 && (!c->k_scale || !c->v_scale))
        return reject("an E4M3 cache needs k_scale and v_scale");
    if ((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) & 15)
        return reject("cache k_scale and v_scale must be 16-byte aligned");
    if (!s || !s->page_table) return reject("page_table must not be NULL");
    if (s->seqs < 1 || s->table_stride < 1) return reject("seqs and table_stride must be positive");
    return AMOE_OK;
}

inline CacheDev cache_dev(const amoe_kv_cache *c, const amoe_kv_seqs *s) {
    int shift = 0;
    while ((1 << shift) < c->page_size) ++shift;
    return {static_cast<char *>(c->k), static_cast<char *>(c->v), c->k_scale, c->v_scale, c->status,
            s->page_table, c->pages, s->table_stride, shift, c->kv_heads};
}

}  // namespace attn
}  // namespace amoe
