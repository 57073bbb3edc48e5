// attn_decode.cu -- attention of one new token a sequence over the paged cache
// (CausalAttentionWithConfig with one query, internal/backend/cpuref/attention.go:82-171).
//
// One CTA takes one (sequence, query head); its warps split the keys, each with a running
// maximum and sum, and join through shared memory.
#include "attn.cuh"

namespace amoe {
namespace attn {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

struct DecodeParams {
    CacheDev c;
    RowsDev q, out;
    const int32_t *kv_len;
    const float *sinks;
    float scale_log2;
    int window, seqs, group;
};

template <int D, int CACHE, int TYPE>
__global__ void __launch_bounds__(kThreads) decode_attn_kernel(const __grid_constant__ DecodeParams p) {
    constexpr int E = D / 32;
    __shared__ float sm[kWarps], sl[kWarps], so[kWarps][D];
    const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
    const int s = blockIdx.y, h = blockIdx.x, kvh = h / p.group;
    const int len = p.kv_len[s];
    if (len < 0 && threadIdx.x == 0) atomicOr(p.c.status, AMOE_KV_BAD_LENGTHS);
    const int from = p.window > 0 ? max(0, len - p.window) : 0;
    float q[E], acc[E] = {}, m = -INFINITY, l = 0.0f;
    auto f16_or = [](const char *src, int i) {
        return TYPE == AMOE_GGUF_F16 ? __half2float(reinterpret_cast<const __half *>(src)[i])
                                     : __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(src)[i]);
    };
    const char *qs = p.q.p + s * p.q.ts + h * p.q.hs + lane * E * 2;
#pragma unroll
    for (int i = 0; i < E; ++i) q[i] = f16_or(qs, i);
    for (int j = from + w; j < len; j += kWarps) {
        const int page = page_of(p.c, s, j);
        if (page < 0) continue;
        const int64_t row = cache_row(p.c, page, kvh, j);
        float k[E], v[E], dot = 0.0f;
        if constexpr (CACHE == AMOE_KV_E4M3) {
            auto val = [&](const char *pages, const uint8_t *sc, int i) {
                const uint32_t hh = e4m3x2_to_f16x2((uint8_t)pages[row * D + lane * E + i]);
                return __low2float(*reinterpret_cast<const __half2 *>(&hh)) * e8m0_to_float(sc[row]);
            };
#pragma unroll
            for (int i = 0; i < E; ++i) k[i] = val(p.c.k, p.c.ks, i), v[i] = val(p.c.v, p.c.vs, i);
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i)
                k[i] = f16_or(p.c.k + (row * D + lane * E) * 2, i), v[i] = f16_or(p.c.v + (row * D + lane * E) * 2, i);
        }
#pragma unroll
        for (int i = 0; i < E; ++i) dot = fmaf(q[i], k[i], dot);
#pragma unroll
        for (int x = 16; x; x >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, x);
        const float x = dot * p.scale_log2, mm = fmaxf(m, x);
        const float keep = mm == -INFINITY ? 1.0f : exp2f(m - mm), e = mm == -INFINITY ? 0.0f : exp2f(x - mm);
        m = mm;
        l = l * keep + e;
#pragma unroll
        for (int i = 0; i < E; ++i) acc[i] = acc[i] * keep + e * v[i];
    }
    if (lane == 0) sm[w] = m, sl[w] = l;
#pragma unroll
    for (int i = 0; i < E; ++i) so[w][lane * E + i] = acc[i];
    __syncthreads();
    if (w) return;
    const float sink = p.sinks ? p.sinks[h] * kLog2e : -INFINITY;
    float top = sink;
    for (int i = 0; i < kWarps; ++i) top = fmaxf(top, sm[i]);
    float sum = top == -INFINITY ? 0.0f : exp2f(sink - top), o[E] = {};
    for (int i = 0; i < kWarps; ++i) {
        if (sm[i] == -INFINITY && sl[i] == 0.0f) continue;
        const float f = exp2f(sm[i] - top);
        sum += sl[i] * f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] += so[i][lane * E + e] * f;
    }
    const float r = sum == 0.0f ? 0.0f : 1.0f / sum;
    char *dst = p.out.p + s * p.out.ts + h * p.out.hs + lane * E * 2;
#pragma unroll
    for (int e = 0; e < E; e += 2)
        reinterpret_cast<uint32_t *>(dst)[e / 2] = pack2<TYPE>(o[e] * r, o[e + 1] * r);
}

template <int D>
void launch(const DecodeParams &p, int cache, int type, dim3 grid, cudaStream_t st) {
    if (cache == AMOE_GGUF_F16) decode_attn_kernel<D, AMOE_GGUF_F16, AMOE_GGUF_F16><<<grid, kThreads, 0, st>>>(p);
    else if (cache == AMOE_GGUF_BF16)
        decode_attn_kernel<D, AMOE_GGUF_BF16, AMOE_GGUF_BF16><<<grid, kThreads, 0, st>>>(p);
    else if (type == AMOE_GGUF_F16) decode_attn_kernel<D, AMOE_KV_E4M3, AMOE_GGUF_F16><<<grid, kThreads, 0, st>>>(p);
    else decode_attn_kernel<D, AMOE_KV_E4M3, AMOE_GGUF_BF16><<<grid, kThreads, 0, st>>>(p);
}

}  // namespace
}  // namespace attn
}  // namespace amoe

using namespace amoe;
using namespace amoe::attn;

extern "C" int amoe_attn_decode(const amoe_kv_cache *cache, const amoe_kv_seqs *seqs, const amoe_attn *attn,
                                const amoe_rows *q, const amoe_rows *out, const int32_t *kv_len, int32_t max_len,
                                void *stream) {
    if (int rc = check_cache(cache, seqs)) return rc;
    if (int rc = check_attn(attn)) return rc;
    const int D = cache->head_dim;
    if (int rc = check_rows(q, "q", D, 0, seqs->seqs, -1)) return rc;
    if (q->type == AMOE_GGUF_F32) return reject("decode takes F16 or BF16 queries");
    if (cache->type != AMOE_KV_E4M3 && q->type != cache->type) return reject("q and the cache have different types");
    if (int rc = check_rows(out, "out", D, q->heads, seqs->seqs, q->type)) return rc;
    if (int rc = check_group(q->heads, cache->kv_heads)) return rc;
    if (!kv_len) return reject("kv_len must not be NULL");
    if (max_len < 0) return reject("max_len must not be negative");
    if (seqs->seqs > 65535) return reject("more than 65535 sequences in one decode call");
    DecodeParams p{};
    p.c = cache_dev(cache, seqs);
    p.q = rows_dev(q), p.out = rows_dev(out);
    p.kv_len = kv_len, p.sinks = attn->sinks;
    p.scale_log2 = attn_scale(attn, D) * kLog2e;
    p.window = attn->window, p.seqs = seqs->seqs, p.group = q->heads / cache->kv_heads;
    DeviceScope scope;
    cudaError_t e = scope.enter(cache->device);
    if (e != cudaSuccess) return cuda_error(e, "cudaSetDevice");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const dim3 grid(q->heads, seqs->seqs);
    if (D == 64) launch<64>(p, cache->type, q->type, grid, st);
    else launch<128>(p, cache->type, q->type, grid, st);
    e = cudaGetLastError();
    return e == cudaSuccess ? AMOE_OK : cuda_error(e, "decode kernel");
}
