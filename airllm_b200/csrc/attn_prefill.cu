// attn_prefill.cu -- causal attention of packed prompts with grouped heads, learned sinks
// and a sliding window (CausalAttentionWithConfig, internal/backend/cpuref/attention.go:82-171).
//
//   s_j = scale q.k_j over the visible keys, m = max s_j,
//   out = sum exp(s_j - m) v_j / (sum exp(s_j - m) + exp(sink - m))
//
// One warp takes one query head's row and walks its keys with a running maximum and sum.
#include "attn.cuh"

namespace amoe {
namespace attn {
namespace {

constexpr int kThreads = 128;

struct PrefillParams {
    RowsDev q, k, v, out;
    const int32_t *cu_q, *cu_k;
    const float *sinks;
    float scale_log2;
    int window, q_tokens, k_tokens, seqs, q_heads, group;
};

template <int D, int TYPE>
__global__ void __launch_bounds__(kThreads) prefill_kernel(const __grid_constant__ PrefillParams p) {
    constexpr int E = D / 32;  // elements of a lane
    const int lane = threadIdx.x % 32;
    const int t = blockIdx.x, h = blockIdx.y * (kThreads / 32) + threadIdx.x / 32;
    if (h >= p.q_heads) return;
    if (t >= p.cu_q[p.seqs]) return;
    const int s = find_seq(p.cu_q, p.seqs, t);
    const int q0 = p.cu_q[s], q1 = min(p.cu_q[s + 1], p.q_tokens);
    if (q0 < 0 || t < q0 || t >= q1) return;
    const int k0 = max(p.cu_k[s], 0), k1 = min(p.cu_k[s + 1], p.k_tokens);
    const int at = (k1 - k0) - (q1 - t);  // this query's position among its keys
    const int from = p.window > 0 ? max(0, at - p.window + 1) : 0;
    auto row = [&](const RowsDev &r, int tok, int head, float (&x)[E]) {
        const char *src = r.p + tok * r.ts + head * r.hs + lane * E * 2;
#pragma unroll
        for (int i = 0; i < E; ++i)
            x[i] = TYPE == AMOE_GGUF_F16 ? __half2float(reinterpret_cast<const __half *>(src)[i])
                                         : __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(src)[i]);
    };
    float q[E], acc[E] = {}, m = -INFINITY, l = 0.0f;
    row(p.q, t, h, q);
    for (int j = from; j <= at; ++j) {
        float k[E], v[E], dot = 0.0f;
        row(p.k, k0 + j, h / p.group, k);
        row(p.v, k0 + j, h / p.group, v);
#pragma unroll
        for (int i = 0; i < E; ++i) dot = fmaf(q[i], k[i], dot);
#pragma unroll
        for (int w = 16; w; w >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, w);
        const float x = dot * p.scale_log2, mm = fmaxf(m, x);
        const float keep = mm == -INFINITY ? 1.0f : exp2f(m - mm), e = mm == -INFINITY ? 0.0f : exp2f(x - mm);
        m = mm;
        l = l * keep + e;
#pragma unroll
        for (int i = 0; i < E; ++i) acc[i] = acc[i] * keep + e * v[i];
    }
    if (p.sinks) {
        const float x = p.sinks[h] * kLog2e, mm = fmaxf(m, x);
        const float keep = mm == -INFINITY ? 1.0f : exp2f(m - mm);
        l = l * keep + (mm == -INFINITY ? 0.0f : exp2f(x - mm));
#pragma unroll
        for (int i = 0; i < E; ++i) acc[i] *= keep;
    }
    char *dst = p.out.p + t * p.out.ts + h * p.out.hs + lane * E * 2;
#pragma unroll
    for (int i = 0; i < E; i += 2) {
        const float r = l == 0.0f ? 0.0f : 1.0f / l;
        reinterpret_cast<uint32_t *>(dst)[i / 2] = pack2<TYPE>(acc[i] * r, acc[i + 1] * r);
    }
}

}  // namespace
}  // namespace attn
}  // namespace amoe

using namespace amoe;
using namespace amoe::attn;

extern "C" int amoe_attn_prefill(int32_t device, int32_t head_dim, const amoe_attn *attn, const amoe_rows *q,
                                 const amoe_rows *k, const amoe_rows *v, const amoe_rows *out, int32_t q_tokens,
                                 int32_t k_tokens, const int32_t *cu_q, const int32_t *cu_k, int32_t seqs,
                                 void *stream) {
    if (int rc = check_attn(attn)) return rc;
    if (int rc = check_head_dim(head_dim)) return rc;
    if (q_tokens < 0 || k_tokens < 0) return reject("q_tokens and k_tokens must not be negative");
    if (int rc = check_rows(q, "q", head_dim, 0, q_tokens, -1)) return rc;
    if (q->type != AMOE_GGUF_F16 && q->type != AMOE_GGUF_BF16) return reject("prefill takes F16 or BF16 rows");
    if (int rc = check_rows(k, "k", head_dim, 0, k_tokens, q->type)) return rc;
    if (int rc = check_rows(v, "v", head_dim, k->heads, k_tokens, q->type)) return rc;
    if (int rc = check_rows(out, "out", head_dim, q->heads, q_tokens, q->type)) return rc;
    if (int rc = check_group(q->heads, k->heads)) return rc;
    if (!cu_q || !cu_k) return reject("cu_q and cu_k must not be NULL");
    if (seqs < 1) return reject("seqs must be positive");
    if (q_tokens == 0) return AMOE_OK;
    PrefillParams p{};
    p.q = rows_dev(q), p.k = rows_dev(k), p.v = rows_dev(v), p.out = rows_dev(out);
    p.cu_q = cu_q, p.cu_k = cu_k;
    p.sinks = attn->sinks;
    p.scale_log2 = attn_scale(attn, head_dim) * kLog2e;
    p.window = attn->window, p.q_tokens = q_tokens, p.k_tokens = k_tokens, p.seqs = seqs;
    p.q_heads = q->heads, p.group = q->heads / k->heads;
    DeviceScope scope;
    cudaError_t e = scope.enter(device);
    if (e != cudaSuccess) return cuda_error(e, "cudaSetDevice");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const dim3 grid(q_tokens, (q->heads + 3) / 4);
    if (head_dim == 64 && q->type == AMOE_GGUF_F16) prefill_kernel<64, AMOE_GGUF_F16><<<grid, kThreads, 0, st>>>(p);
    else if (head_dim == 64) prefill_kernel<64, AMOE_GGUF_BF16><<<grid, kThreads, 0, st>>>(p);
    else if (q->type == AMOE_GGUF_F16) prefill_kernel<128, AMOE_GGUF_F16><<<grid, kThreads, 0, st>>>(p);
    else prefill_kernel<128, AMOE_GGUF_BF16><<<grid, kThreads, 0, st>>>(p);
    e = cudaGetLastError();
    return e == cudaSuccess ? AMOE_OK : cuda_error(e, "prefill kernel");
}
