// kv_cache.cu -- the paged key-value cache's writes and reads: rotation, quantisation and
// append (yarnHeads, internal/model/gptoss/layer.go:189-207; YaRNRoPE,
// internal/backend/cpuref/rope.go:17-86; KVCache.Append, attention.go:40-59), and the gather
// of a sequence's pages back into packed rows.
//
// append.  Element i and i + d/2 of a head turn by the angle pos * freq[i]:
//   y[i] = x[i] c - x[i + d/2] s,  y[i + d/2] = x[i + d/2] c + x[i] s,
// c and s = cos, sin (angle) * concentration.  Angles of far positions lose float32, and a
// value that lands next to a rounding border of the cache's type must fall on the side the
// definition says, so angles, sines and products are float64 as in the reference, rounded
// once to float32 (its stored type) and from there to the cache's.  A warp or four take a token:
// their lanes compute the angles, then d/16 lanes a head row turn eight pairs each with the sines of
// their eight pairs in registers for every row they visit, the next row's loads in flight as they come (converted
// on arrival they held up the row before: 6000 tokens of 32 + 8 + 8 f16 heads of 128 to E4M3 with their read 78 us, now 63;
// two rows ahead 68).
// Measured: 8192 tokens of 64 + 8 + 8 f32 heads of 64, 252 MB: 48 us, 5.2 TB/s, 0.80 of the copy bandwidth.
//
// E4M3 rows: the scale is a power of two, so scaling is exact and only the rounding to E4M3
// loses bits; the row's maximum is reduced over the d/16 lanes that hold it.
#include "attn.cuh"

namespace amoe {
namespace attn {
namespace {

constexpr int kAppendWarps = 4;  // of a CTA, at most
constexpr int kReadThreads = 256;
constexpr int kReadTokens = 4;  // rows of a warp
constexpr int kNoRow = INT_MIN;  // in the place of a page: not a row of this call

struct RopeDev {
    double freq[AMOE_ROPE_MAX_HALF];
    double conc;
    int on;
};

struct AppendParams {
    CacheDev c;
    RowsDev q, k, v, q_out, k_out, v_out;
    const int32_t *cu, *past;
    int tokens, seqs, q_heads, q_out_type, k_out_type, v_out_type;
    RopeDev rope;
};

// Starts that are negative, decrease or pass the rows given leave rows that no CTA looks at, or that it takes for rows
// behind the last sequence.  The grid's last CTA, which has no row, looks at all of them.
__device__ __forceinline__ void check_starts(const int32_t *cu, int seqs, int tokens, int32_t *status) {
    bool bad = false;
    for (int s = threadIdx.x; s < seqs; s += blockDim.x) {
        const int a = cu[s], b = cu[s + 1];
        bad |= a < 0 || b < a || b > tokens;
    }
    if (bad) atomicOr(status, AMOE_KV_BAD_LENGTHS);
}

// Smallest e with amax <= 448 * 2^e, at least -127; 0 for amax == 0.  amax = 1.f * 2^(E - 127)
// and 448 * 2^e = 1.75 * 2^(e + 8).
__device__ __forceinline__ int e4m3_exp(float amax) {
    const uint32_t b = __float_as_uint(amax);
    if (b == 0u) return 0;
    const int e = (int)(b >> 23) - 135 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < -127 ? -127 : e;
}

// 2^e, e in [-127, 127].
__device__ __forceinline__ float exp2i(int e) {
    return e == -127 ? __uint_as_float(0x00400000u) : __uint_as_float((uint32_t)(e + 127) << 23);
}

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint32_t r;
    asm("{\n .reg .b16 t;\n cvt.rn.satfinite.e4m3x2.f32 t, %1, %2;\n cvt.u32.u16 %0, t;\n}"
        : "=r"(r)
        : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ uint2 e4m3x8(const float (&x)[8], float by) {
    return make_uint2(e4m3x2(x[0] * by, x[1] * by) | e4m3x2(x[2] * by, x[3] * by) << 16,
                      e4m3x2(x[4] * by, x[5] * by) | e4m3x2(x[6] * by, x[7] * by) << 16);
}

// One thread's two groups of eight (elements i0.. and i0 + D/2..) of one row into the cache.
// All D/16 lanes of the row call it together.
template <int D, int CACHE>
__device__ __forceinline__ void cache_store(char *pages, uint8_t *scales, int64_t row, int part, const float (&a)[8],
                                            const float (&b)[8], bool write) {
    if constexpr (CACHE == AMOE_KV_E4M3) {
        float amax = 0.0f;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            amax = fmaxf(amax, fmaxf(fabsf(a[i]), fabsf(b[i])));
            bad |= !isfinite(a[i]) || !isfinite(b[i]);
        }
        if (bad) amax = INFINITY;
#pragma unroll
        for (int m = 1; m < D / 16; m <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, m));
        if (!write) return;
        char *dst = pages + row * D + part * 8;
        if (amax == INFINITY) {
            *reinterpret_cast<uint2 *>(dst) = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
            *reinterpret_cast<uint2 *>(dst + D / 2) = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
            if (part == 0) scales[row] = 255;
            return;
        }
        const int e = e4m3_exp(amax);
        const float by = exp2i(-e);
        *reinterpret_cast<uint2 *>(dst) = e4m3x8(a, by);
        *reinterpret_cast<uint2 *>(dst + D / 2) = e4m3x8(b, by);
        if (part == 0) scales[row] = (uint8_t)(e + 127);
    } else {
        if (!write) return;
        char *dst = pages + (row * D + part * 8) * 2;
        store8<CACHE>(dst, a);
        store8<CACHE>(dst + D, b);
    }
}

template <int D, int SRC, int CACHE>
__global__ void __launch_bounds__(32 * kAppendWarps) append_kernel(const __grid_constant__ AppendParams p) {
    constexpr int L = D / 16;  // lanes of a row
    constexpr int STEP = 32 / L;  // rows of a warp at a time
    constexpr int ES = SRC == AMOE_GGUF_F32 ? 4 : 2;
    __shared__ double2 cs[D / 2];
    const int lane = threadIdx.x % 32, part = lane % L, warp = threadIdx.x / 32, warps = blockDim.x / 32;
    if (blockIdx.x == gridDim.x - 1) return check_starts(p.cu, p.seqs, p.tokens, p.c.status);
    const int t = blockIdx.x, r0 = warp * STEP + lane / L, rows = p.q_heads + 2 * p.c.heads;

    struct Row {  // as loaded: a conversion would wait for it
        uint4 a[ES / 2], b[ES / 2];
    };
    auto load = [&](int r, Row &x) {
        if (r >= rows) return;
        const bool is_q = r < p.q_heads, is_k = !is_q && r < p.q_heads + p.c.heads;
        const RowsDev &src = is_q ? p.q : is_k ? p.k : p.v;
        const int h = is_q ? r : is_k ? r - p.q_heads : r - p.q_heads - p.c.heads;
        const char *at = src.p + t * src.ts + h * src.hs + part * 8 * ES;
#pragma unroll
        for (int i = 0; i < ES / 2; ++i) {
            x.a[i] = reinterpret_cast<const uint4 *>(at)[i];
            x.b[i] = reinterpret_cast<const uint4 *>(at + D / 2 * ES)[i];
        }
    };
    Row next{};
    load(r0, next);  // on its way while the position and its sines are found

    const int last = p.cu[p.seqs];
    int found[1];
    find_seqs(p.cu, p.seqs, t, found);
    const int s = found[0], start = p.cu[s], past = p.past[s];
    if (t >= last) return;  // rows behind the last sequence
    if (start > t || start < 0 || p.cu[s + 1] <= t || past < 0) {
        if (threadIdx.x == 0) atomicOr(p.c.status, AMOE_KV_BAD_LENGTHS);
        return;
    }
    const int64_t pos = (int64_t)past + (t - start);
    const int page = page_of(p.c, s, pos);
    double2 w[8];
    if (p.rope.on) {
        // the token's warps share its sines
        for (int i = threadIdx.x; i < D / 2; i += blockDim.x) {
            double sn, c;
            sincos((double)pos * p.rope.freq[i], &sn, &c);
            cs[i] = make_double2(c * p.rope.conc, sn * p.rope.conc);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = cs[part * 8 + i];
    }
    // the warp stays together for the row maximum's shuffles: the bound is the warp's first row
    for (int r = r0; r - lane / L < rows; r += STEP * warps) {
        struct {
            float a[8], b[8];
        } x;
        load8<SRC>(reinterpret_cast<const char *>(next.a), x.a);
        load8<SRC>(reinterpret_cast<const char *>(next.b), x.b);
        load(r + STEP * warps, next);
        const bool live = r < rows;
        const bool is_q = r < p.q_heads, is_k = !is_q && r < p.q_heads + p.c.heads;
        const int h = is_q ? r : is_k ? r - p.q_heads : r - p.q_heads - p.c.heads;
        if (p.rope.on && live && (is_q || is_k)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const double f = x.a[i], g = x.b[i];
                x.a[i] = (float)(f * w[i].x - g * w[i].y);
                x.b[i] = (float)(g * w[i].x + f * w[i].y);
            }
        }
        const RowsDev &dst = is_q ? p.q_out : is_k ? p.k_out : p.v_out;
        if (live && dst.p) {
            const int type = is_q ? p.q_out_type : is_k ? p.k_out_type : p.v_out_type;
            const int es = elem_size(type);
            char *y = dst.p + t * dst.ts + h * dst.hs + part * 8 * es;
            store8_any(y, type, x.a);
            store8_any(y + D / 2 * es, type, x.b);
        }
        const bool write = live && !is_q && page >= 0;
        if (__any_sync(0xffffffffu, write)) {
            const int64_t row = write ? cache_row(p.c, page, h, pos) : 0;
            cache_store<D, CACHE>(is_k ? p.c.k : p.c.v, is_k ? p.c.ks : p.c.vs, row, part, x.a, x.b, write);
        }
    }
}

struct ReadParams {
    CacheDev c;
    RowsDev k, v;
    const int32_t *cu, *first;
    int tokens, seqs, k_type, v_type;
};

// A warp takes four rows of the output; its lanes walk (head, token) pairs, token first: four
// tokens of a head are one run of the page, and a lane moves 16 bytes of it.
template <int D, int CACHE>
__global__ void __launch_bounds__(kReadThreads, 4) read_kernel(const __grid_constant__ ReadParams p) {
    constexpr int E = CACHE == AMOE_KV_E4M3 ? 16 : 8;  // elements of 16 bytes
    constexpr int C = D / E, RPI = 32 / C, BATCH = 4;  // lanes of a row, rows at a time, batches of them
    if (blockIdx.x == gridDim.x - 1) return check_starts(p.cu, p.seqs, p.tokens, p.c.status);
    const int lane = threadIdx.x % 32, ch = lane % C;
    const int64_t first_row = ((int64_t)blockIdx.x * (kReadThreads / 32) + threadIdx.x / 32) * kReadTokens;
    const int last = min(p.cu[p.seqs], p.tokens);
    if (first_row >= last) return;
    const int t0 = (int)first_row;
    int page = kNoRow, found[kReadTokens];
    int64_t pos = 0;
    find_seqs(p.cu, p.seqs, t0, found);
    if (lane < kReadTokens && t0 + lane < last) {
        const int t = t0 + lane;
        const int s = lane == 0 ? found[0] : lane == 1 ? found[1] : lane == 2 ? found[2] : found[3];
        const int start = p.cu[s];
        const int64_t f = p.first ? p.first[s] : 0;
        if (start < 0 || start > t || p.cu[s + 1] <= t || f < 0) {
            atomicOr(p.c.status, AMOE_KV_BAD_LENGTHS);
            page = -AMOE_KV_BAD_LENGTHS;  // a row of this call all the same: zeros
        } else {
            pos = f + (t - start);
            page = page_of(p.c, s, pos);
        }
    }
    __syncwarp();
    // row of a head's first page slot, in the pages: the head only adds a multiple of the page size
    const int64_t row0 = page >= 0 ? cache_row(p.c, page, 0, pos) : 0;
    const int items = kReadTokens * 2 * p.c.heads;
    for (int i0 = lane / C; i0 - lane / C < items; i0 += RPI * BATCH) {
        uint4 w[BATCH];
        uint32_t e[BATCH];
        // the copies of a batch are all on their way before the first is used
#pragma unroll
        for (int m = 0; m < BATCH; ++m) {
            const int i = i0 + m * RPI, tok = i % kReadTokens, hk = i / kReadTokens;
            const bool on = __shfl_sync(0xffffffffu, page, tok) >= 0 && i < items;
            const int64_t base = __shfl_sync(0xffffffffu, row0, tok);
            const bool is_v = hk >= p.c.heads;
            const int64_t row = base + ((int64_t)(is_v ? hk - p.c.heads : hk) << p.c.shift);
            w[m] = make_uint4(0, 0, 0, 0);
            e[m] = 127;
            if (on) {
                w[m] = *reinterpret_cast<const uint4 *>((is_v ? p.c.v : p.c.k) + row * (D * 16 / E) + ch * 16);
                if (CACHE == AMOE_KV_E4M3) e[m] = (is_v ? p.c.vs : p.c.ks)[row];
            }
        }
#pragma unroll
        for (int m = 0; m < BATCH; ++m) {
            const int i = i0 + m * RPI, tok = i % kReadTokens, hk = i / kReadTokens;
            if (__shfl_sync(0xffffffffu, page, tok) == kNoRow || i >= items) continue;
            const bool is_v = hk >= p.c.heads;
            const RowsDev &dst = is_v ? p.v : p.k;
            const int type = is_v ? p.v_type : p.k_type;
            char *y = dst.p + (int64_t)(t0 + tok) * dst.ts + (is_v ? hk - p.c.heads : hk) * dst.hs +
                      ch * E * elem_size(type);
            if constexpr (CACHE == AMOE_KV_E4M3) {
                float x[16];
                const float by = e8m0_to_float(e[m]);
                const uint32_t u[4] = {w[m].x, w[m].y, w[m].z, w[m].w};
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    uint32_t lo, hi;
                    e4m3x4_to_f16x2(u[n], lo, hi);
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&lo));
                    const float2 g = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
                    x[4 * n] = f.x * by, x[4 * n + 1] = f.y * by, x[4 * n + 2] = g.x * by, x[4 * n + 3] = g.y * by;
                }
                store8_any(y, type, *reinterpret_cast<const float(*)[8]>(x));
                store8_any(y + 8 * elem_size(type), type, *reinterpret_cast<const float(*)[8]>(x + 8));
            } else if (type == CACHE) {
                *reinterpret_cast<uint4 *>(y) = w[m];
            } else {
                float x[8];
                load8<CACHE>(reinterpret_cast<const char *>(&w[m]), x);
                store8_any(y, type, x);
            }
        }
    }
}

template <int D, int SRC>
cudaError_t launch_append(const AppendParams &p, int cache, cudaStream_t st) {
    // A CTA a token, and one for the starts: one warp, or four where the tokens alone do not fill the GPU.  8192 tokens of 64-wide f32 heads: 47.9 us with one warp to a token, 51 with two, 61 with four; 6000 of 128-wide
    // f16 ones with their read: 63.4, 68, 78.
    const int grid = p.tokens + 1, threads = p.tokens < 148 * 8 ? 32 * kAppendWarps : 32;
    if (cache == AMOE_GGUF_F16) append_kernel<D, SRC, AMOE_GGUF_F16><<<grid, threads, 0, st>>>(p);
    else if (cache == AMOE_GGUF_BF16) append_kernel<D, SRC, AMOE_GGUF_BF16><<<grid, threads, 0, st>>>(p);
    else append_kernel<D, SRC, AMOE_KV_E4M3><<<grid, threads, 0, st>>>(p);
    return cudaGetLastError();
}

template <int D>
cudaError_t launch_append_d(const AppendParams &p, int src, int cache, cudaStream_t st) {
    if (src == AMOE_GGUF_F32) return launch_append<D, AMOE_GGUF_F32>(p, cache, st);
    if (src == AMOE_GGUF_F16) return launch_append<D, AMOE_GGUF_F16>(p, cache, st);
    return launch_append<D, AMOE_GGUF_BF16>(p, cache, st);
}

int check_rope(int head_dim, double theta, const amoe_rope *out) {
    if (!out) return reject("out must not be NULL");
    if (head_dim <= 0 || head_dim % 2) return reject("rope head dimension must be positive and even");
    if (head_dim > 2 * AMOE_ROPE_MAX_HALF)
        return reject("rope head dimension above " + std::to_string(2 * AMOE_ROPE_MAX_HALF));
    if (!(theta > 0) || std::isinf(theta)) return reject("rope theta must be finite and positive");
    return AMOE_OK;
}

// The pair (not a whole one) that turns beta times within the original context.
double yarn_corner(int head_dim, double theta, double original, double beta) {
    const double pi = 3.14159265358979323846;
    return head_dim * std::log(original / (beta * 2.0 * pi)) / (2.0 * std::log(theta));
}

template <int D>
cudaError_t launch_read_d(const ReadParams &p, int cache, cudaStream_t st) {
    const int grid = (p.tokens - 1) / (kReadTokens * kReadThreads / 32) + 2;
    if (cache == AMOE_GGUF_F16) read_kernel<D, AMOE_GGUF_F16><<<grid, kReadThreads, 0, st>>>(p);
    else if (cache == AMOE_GGUF_BF16) read_kernel<D, AMOE_GGUF_BF16><<<grid, kReadThreads, 0, st>>>(p);
    else read_kernel<D, AMOE_KV_E4M3><<<grid, kReadThreads, 0, st>>>(p);
    return cudaGetLastError();
}

}  // namespace
}  // namespace attn
}  // namespace amoe

using namespace amoe;
using namespace amoe::attn;

extern "C" {

int amoe_rope_init(int32_t head_dim, double theta, int32_t yarn, amoe_rope *out) {
    if (int rc = check_rope(head_dim, theta, out)) return rc;
    *out = {};
    const int half = head_dim / 2;
    const double factor = 32.0, original = 4096.0;
    const double low = std::fmax(0.0, std::floor(yarn_corner(head_dim, theta, original, 32.0)));
    const double high = std::fmin(half - 1.0, std::ceil(yarn_corner(head_dim, theta, original, 1.0)));
    for (int i = 0; i < half; ++i) {
        out->freq[i] = std::pow(theta, -2.0 * i / head_dim);
        if (!yarn) continue;
        const double ramp = high == low ? 0.0 : std::fmax(0.0, std::fmin(1.0, (i - low) / (high - low)));
        out->freq[i] *= ramp + (1.0 - ramp) / factor;  // the reference's ends, not the published ones
    }
    out->concentration = yarn ? 1.0 + 0.1 * std::log(factor) : 1.0;
    out->head_dim = head_dim;
    return AMOE_OK;
}

int amoe_rope_init_yarn(int32_t head_dim, double theta, double factor, double original_context, double beta_fast,
                        double beta_slow, int32_t truncate, amoe_rope *out) {
    if (int rc = check_rope(head_dim, theta, out)) return rc;
    if (!(theta > 1)) return reject("yarn theta must be above 1");
    if (!(factor >= 1) || std::isinf(factor)) return reject("yarn factor must be finite and at least 1");
    if (!(original_context > 0) || std::isinf(original_context))
        return reject("yarn original_context must be finite and positive");
    if (!(beta_slow > 0) || !(beta_fast >= beta_slow) || std::isinf(beta_fast))
        return reject("yarn beta_fast must be finite and at least beta_slow, beta_slow positive");
    *out = {};
    double low = yarn_corner(head_dim, theta, original_context, beta_fast);
    double high = yarn_corner(head_dim, theta, original_context, beta_slow);
    if (truncate) low = std::floor(low), high = std::ceil(high);
    low = std::fmax(low, 0.0), high = std::fmin(high, head_dim - 1.0);
    for (int i = 0; i < head_dim / 2; ++i) {
        const double ramp = i <= low ? 0.0 : i >= high ? 1.0 : (i - low) / (high - low);
        out->freq[i] = std::pow(theta, -2.0 * i / head_dim) * (1.0 - ramp + ramp / factor);
    }
    out->concentration = 1.0 + 0.1 * std::log(factor);
    out->head_dim = head_dim;
    return AMOE_OK;
}

int amoe_kv_append(const amoe_kv_cache *cache, const amoe_kv_seqs *seqs, const int32_t *cu, const int32_t *past,
                   int32_t tokens, const amoe_rope *rope, const amoe_rows *q, const amoe_rows *k, const amoe_rows *v,
                   const amoe_rows *q_out, const amoe_rows *k_out, const amoe_rows *v_out, void *stream) {
    if (int rc = check_cache(cache, seqs)) return rc;
    if (!cu || !past) return reject("cu and past must not be NULL");
    if (tokens < 0) return reject("tokens must not be negative");
    if (tokens == INT_MAX) return reject("more than 2^31 - 2 tokens in one append call");  // a CTA each, and one more
    const int D = cache->head_dim, kv = cache->kv_heads;
    if (int rc = check_rows(k, "k", D, kv, tokens, -1)) return rc;
    if (int rc = check_rows(v, "v", D, kv, tokens, k->type)) return rc;
    if (q)
        if (int rc = check_rows(q, "q", D, 0, tokens, k->type)) return rc;
    if (q_out && !q) return reject("q_out without q");
    if (q_out)
        if (int rc = check_rows(q_out, "q_out", D, q->heads, tokens, -1)) return rc;
    if (k_out)
        if (int rc = check_rows(k_out, "k_out", D, kv, tokens, -1)) return rc;
    if (v_out)
        if (int rc = check_rows(v_out, "v_out", D, kv, tokens, -1)) return rc;
    if (rope && rope->head_dim != D) return reject("the rope's head_dim differs from the cache's");
    if (tokens == 0) return AMOE_OK;
    AppendParams p{};
    p.c = cache_dev(cache, seqs);
    p.q = rows_dev(q), p.k = rows_dev(k), p.v = rows_dev(v);
    p.q_out = rows_dev(q_out), p.k_out = rows_dev(k_out), p.v_out = rows_dev(v_out);
    p.cu = cu, p.past = past;
    p.tokens = tokens, p.seqs = seqs->seqs;
    p.q_heads = q && q_out ? q->heads : 0;  // a q that goes nowhere is not read
    p.q_out_type = q_out ? q_out->type : 0;
    p.k_out_type = k_out ? k_out->type : 0;
    p.v_out_type = v_out ? v_out->type : 0;
    if (rope) {
        for (int i = 0; i < D / 2; ++i) p.rope.freq[i] = rope->freq[i];
        p.rope.conc = rope->concentration;
        p.rope.on = 1;
    }
    DeviceScope scope;
    cudaError_t e = scope.enter(cache->device);
    if (e != cudaSuccess) return cuda_error(e, "cudaSetDevice");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    e = D == 64 ? launch_append_d<64>(p, k->type, cache->type, st) : launch_append_d<128>(p, k->type, cache->type, st);
    return e == cudaSuccess ? AMOE_OK : cuda_error(e, "append kernel");
}

int amoe_kv_read(const amoe_kv_cache *cache, const amoe_kv_seqs *seqs, const int32_t *cu, const int32_t *first,
                 int32_t tokens, const amoe_rows *k_out, const amoe_rows *v_out, void *stream) {
    if (int rc = check_cache(cache, seqs)) return rc;
    if (!cu) return reject("cu must not be NULL");
    if (tokens < 0) return reject("tokens must not be negative");
    if (int rc = check_rows(k_out, "k_out", cache->head_dim, cache->kv_heads, tokens, -1)) return rc;
    if (int rc = check_rows(v_out, "v_out", cache->head_dim, cache->kv_heads, tokens, -1)) return rc;
    if (tokens == 0) return AMOE_OK;
    ReadParams p{};
    p.c = cache_dev(cache, seqs);
    p.k = rows_dev(k_out), p.v = rows_dev(v_out);
    p.cu = cu, p.first = first;
    p.tokens = tokens, p.seqs = seqs->seqs;
    p.k_type = k_out->type, p.v_type = v_out->type;
    DeviceScope scope;
    cudaError_t e = scope.enter(cache->device);
    if (e != cudaSuccess) return cuda_error(e, "cudaSetDevice");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    e = cache->head_dim == 64 ? launch_read_d<64>(p, cache->type, st) : launch_read_d<128>(p, cache->type, st);
    return e == cudaSuccess ? AMOE_OK : cuda_error(e, "read kernel");
}

}  // extern "C"
