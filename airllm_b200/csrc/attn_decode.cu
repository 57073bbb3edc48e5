// attn_decode.cu -- attention of one new token a sequence over the paged cache
// (CausalAttentionWithConfig with one query, internal/backend/cpuref/attention.go:82-171).
//
// A step reads every visible key and value once and does a handful of products with each, so
// HBM bounds it, or the instructions that get E4M3 codes to the products.  What the kernel does about that:
//   - the query heads of one kv head share one read of its keys, as columns of mma.sync m16n8k16
//     products whose rows are keys (scores) and elements (values): eight heads fill a block.  CUDA cores could not
//     keep up: 8 heads x 2 products an element at 6.5 TB/s is two thirds of the f32 rate for 16-bit
//     caches and over it for E4M3;
//   - each warp walks its own tiles of 32 (16 for 128-wide 16-bit rows) keys through a private
//     ring of two cp.async stages, so no barrier stands in the loop; 12 to 20 warps an SM keep 100 to 200 KB
//     in flight, more than latency times bandwidth needs (deeper rings with fewer warps were slower: a
//     tile is a chain of dependent steps, and warps hide it).  Each copy carries its own length, so a
//     masked key, or one without a page, is staged as zeros: what lies in such slots, NaN included,
//     never reaches the products.  A tile that lies in one page is copied as one run; smaller pages
//     have each lane look up its key;
//   - a head's running maximum is lazy: it moves, and the sums are rescaled, when some weight has outgrown it by
//     2^8 (2^4 in f16, whose weights carry a factor: attn.cuh), which one vote a tile finds out;
//   - the keys of one (sequence, kv head) are split over the CTAs of a cluster of up to 8, whose
//     partial sums join through distributed shared memory: one launch.  A few long sequences
//     need more CTAs than clusters can place (clusters of 16 left SMs idle: 59 us instead of 50 for
//     131072 tokens of 8 f16 heads), so they write partial sums to the caller's workspace and
//     a second kernel, whose launch overlaps the first, joins them.  So do a few sequences of lengths that
//     may differ: the device shares the CTAs out by the lengths.  No atomics: the order of addition
//     does not depend on timing.
//
// E4M3 keys and values meet f16 operands (every code is an f16 value).  A key's scale multiplies
// its score.  A value's scale 2^e goes into the weight: w = exp2(t + e - m), t the score in
// log2 and m the running maximum of t + e, so that what a weight may lose is small beside the largest product
// whatever the scales are; the denominator sums exp2(t - n) with a maximum n of its own.
//
// Measured (B200): 131072 tokens, 8 kv heads, f16: 47.6 us in a graph, 5.6 TB/s, 0.86 of the copy bandwidth; 49.6 call after call.
// 48 sequences of 4096-8192 tokens, E4M3: 70 us, 4.3 TB/s, 0.65: the ALU pipe is 50 % busy (the codes'
// conversions) and sequences of unequal lengths leave SMs idle at the end.  E4M3 products (m16n8k32, queries
// and weights as two E4M3 terms each) took 89 us.
#include "attn.cuh"

#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

namespace amoe {
namespace attn {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kCluster = 8;
constexpr int kMaxWide = 256;  // CTAs that the join kernel takes: one for each of its threads

struct DecodeParams {
    CacheDev c;
    RowsDev q, out;
    const int32_t *kv_len;
    const float *sinks;
    float *work;  // partial sums of the CTAs, where they do not join in a cluster
    float scale_log2;
    int window, group, q_type;
    int split;  // CTAs to a (sequence, group of heads); where they join through work: to all sequences of a group of heads
    int seqs;
};

__device__ __forceinline__ uint32_t smem_addr(const void *p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// 16 bytes to shared memory; zeros when `live` is false (nothing is read then).
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// The first `bytes` (0..4) of an aligned word, the rest zeros.
__device__ __forceinline__ void copy4(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}

template <int TYPE>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (TYPE == AMOE_GGUF_F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 2^x to 2^-22, zero below the smallest normal.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// An 8 x 8 matrix of 16-bit elements, two of a row to a lane, transposed across the warp.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ float quad_max(float x) {
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
    return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}
// Over the eight lanes that hold the same pair of heads.
__device__ __forceinline__ float keys_max(float x) {
#pragma unroll
    for (int i = 4; i < 32; i <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, i));
    return x;
}
__device__ __forceinline__ float keys_sum(float x) {
#pragma unroll
    for (int i = 4; i < 32; i <<= 1) x += __shfl_xor_sync(0xffffffffu, x, i);
    return x;
}

// Sizes of one instantiation.  TYPE is the products' type: the cache's, or F16 for E4M3.
template <int D, int CACHE>
struct Tile {
    static constexpr bool kFp8 = CACHE == AMOE_KV_E4M3;
    static constexpr int kType = kFp8 ? AMOE_GGUF_F16 : CACHE;
    static constexpr float kShift = weight_shift(kType);        // log2 of the weights' factor
    static constexpr float kTop = kShift + weight_lazy(kType);  // and of the largest weight
    static constexpr int kRow = D * (kFp8 ? 1 : 2);             // bytes of a cache row
    static constexpr int kKeys = kRow == 256 ? 16 : 32;         // keys of a warp's tile
    static constexpr int kStage = 2 * kKeys * kRow;             // K then V
    static constexpr int kStages = 2;
    static constexpr int kCtas = kStage == 4096 ? 5 : 3;        // to an SM: what registers and shared memory allow
    static constexpr int kSide = kFp8 ? 256 : 0;                // two words of scales a key
    static constexpr int kWarpBytes = kStages * kStage + kStages * (kSide + 4);
    static constexpr int kSmem = kWarps * ((kWarpBytes + 127) / 128 * 128);
    // the join reuses the ring: per warp [16][D] sums, then m, n, l
    static constexpr int kPart = 16 * D + 3 * 16;               // floats
    static_assert((kWarps + 1) * kPart * 4 <= kSmem, "partial sums fit the ring");
};

// 16-byte chunk ch of row r of a staged tile: the order that leaves ldmatrix and the 16-byte
// loads of eight rows at one chunk without bank conflicts.
template <int ROW>
__device__ __forceinline__ uint32_t chunk_at(int r, int ch) {
    return r * ROW + ((ROW == 64 ? ch ^ ((r >> 1) & 3) : ch ^ (r & 7)) << 4);
}

// Four elements of an output row: a sums weights with the maximum top, sum with the maximum y.
__device__ __forceinline__ void store_row(const DecodeParams &p, int seq, int h, int col, float4 a, float sum,
                                          float top, float y) {
    // top -inf: nothing was seen, a is zero whatever the sink, or everything was NaN, and a is
    const float by = sum == 0.0f ? 0.0f : top == -INFINITY ? 1.0f / sum : exp2f(top - y) / sum;
    a.x *= by, a.y *= by, a.z *= by, a.w *= by;
    *reinterpret_cast<uint2 *>(p.out.p + seq * p.out.ts + (int64_t)h * p.out.hs + col * 8) =
        p.q_type == AMOE_GGUF_F16
            ? make_uint2(pack2<AMOE_GGUF_F16>(a.x, a.y), pack2<AMOE_GGUF_F16>(a.z, a.w))
            : make_uint2(pack2<AMOE_GGUF_BF16>(a.x, a.y), pack2<AMOE_GGUF_BF16>(a.z, a.w));
}

// Four elements of one output row out of `split` partial sums [16][D], m, n, l; part(w) is the w-th.
template <int D, class Part>
__device__ __forceinline__ void finish(const DecodeParams &p, int seq, int h, int i, int split, Part part) {
    const int r = i / (D / 4);
    const float sink = p.sinks ? p.sinks[h] * kLog2e : -INFINITY;
    float top = -INFINITY, ntop = sink;
    for (int w = 0; w < split; ++w) {
        const float *x = part(w);
        top = fmaxf(top, x[16 * D + r]);
        ntop = fmaxf(ntop, x[16 * D + 16 + r]);
    }
    const float z = top == -INFINITY ? 0.0f : top, y = ntop == -INFINITY ? 0.0f : ntop;
    float sum = exp2f(sink - y);
    float4 a = make_float4(0, 0, 0, 0);
    for (int w = 0; w < split; ++w) {
        const float *x = part(w);
        const float f = exp2f(x[16 * D + r] - z);
        const float4 v = *reinterpret_cast<const float4 *>(x + i * 4);
        a.x += f * v.x, a.y += f * v.y, a.z += f * v.z, a.w += f * v.w;
        sum += x[16 * D + 32 + r] * exp2f(x[16 * D + 16 + r] - y);
    }
    store_row(p, seq, h, i % (D / 4), a, sum, top, y);
}

// The tiles of `keys` keys that a sequence's query sees, and the first one's first key.
struct Seen {
    int from, end, base, tiles;
};
__device__ __forceinline__ Seen seen_of(const DecodeParams &p, int len, int keys) {
    Seen s;
    const int64_t cap = (int64_t)p.c.table_stride << p.c.shift;
    s.from = p.window > 0 && len > p.window ? len - p.window : 0;
    s.end = len < cap ? len : (int)cap;
    s.base = s.from / keys * keys;
    s.tiles = s.end > s.from ? (s.end - s.base - 1) / keys + 1 : 0;
    return s;
}

// CTAs first .. first + split - 1 of p.split take a sequence: one, and of the others a share like its tiles'.
struct Share {
    int seq, first, split;
};
// CTA x's share (seq < 0), or a sequence's.  Called by whole warps; split 0: the CTA has none.
__device__ __forceinline__ Share share_of(const DecodeParams &p, int keys, int x, int seq) {
    if (p.seqs == 1) return {0, 0, min(p.split, kMaxWide)};
    const int lane = threadIdx.x % 32;
    int64_t total = 0;
    for (int s = lane; s < p.seqs; s += 32) total += seen_of(p, p.kv_len[s], keys).tiles;
#pragma unroll
    for (int i = 16; i; i >>= 1) total += __shfl_xor_sync(0xffffffffu, total, i);
    int before = 0;
    for (int s0 = 0; s0 < p.seqs; s0 += 32) {
        const int s = s0 + lane;
        int n = 0;
        if (s < p.seqs)
            n = 1 + (int)min((int64_t)kMaxWide - 1,
                             seen_of(p, p.kv_len[s], keys).tiles * (int64_t)(p.split - p.seqs) / max(total, (int64_t)1));
        int upto = n;
#pragma unroll
        for (int i = 1; i < 32; i <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, i);
            if (lane >= i) upto += y;
        }
        const int first = before + upto - n;
        const uint32_t hit = __ballot_sync(0xffffffffu, s < p.seqs && (seq < 0 ? x >= first && x < first + n : s == seq));
        if (hit) {
            const int at = __ffs(hit) - 1;
            return {s0 + at, __shfl_sync(0xffffffffu, first, at), __shfl_sync(0xffffffffu, n, at)};
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return {0, 0, 0};
}

// Two blocks of heads over E4M3 spill 20 to 130 bytes a thread at these CTAs an SM.  One CTA fewer has none and is slower
// all the same: 12 heads to a kv head, 8 kv heads of 64, 48 sequences of 4096-8192 92.6 us (92.8 with fewer), 64 of 300
// 18.8 (23.0), one of 60000 29.5 (28.2); 4 kv heads of 128, the 48 108.9 (110.4); 16 heads, one of 60000 29.8 (32.1).
template <int D, int CACHE, int NB, bool WIDE>
__global__ void __launch_bounds__(kThreads, Tile<D, CACHE>::kCtas - (NB == 2 && Tile<D, CACHE>::kCtas > 3)) decode_attn_kernel(const __grid_constant__ DecodeParams p) {
    using T = Tile<D, CACHE>;
    constexpr int TYPE = T::kType, KEYS = T::kKeys, ROW = T::kRow, STAGES = T::kStages;
    constexpr int CPR = ROW / 16, MT = KEYS / 16;
    extern __shared__ __align__(128) char smem[];
    namespace cg = cooperative_groups;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, c = lane % 4;
    int split = p.split, rank = blockIdx.x, seq = blockIdx.z;
    if constexpr (WIDE) {
        cudaTriggerProgrammaticLaunchCompletion();
        const Share share = share_of(p, KEYS, rank, -1);
        if (share.split == 0) return;
        split = share.split, seq = share.seq, rank -= share.first;
        if (rank >= split) return;
    }
    const int kvh = blockIdx.y % p.c.heads, row0 = blockIdx.y / p.c.heads * 16;
    char *ring = smem + warp * ((T::kWarpBytes + 127) / 128 * 128);
    uint32_t *side = reinterpret_cast<uint32_t *>(ring + STAGES * T::kStage);  // [STAGES][2][32] scale words, then masks
    uint32_t *masks = side + STAGES * (T::kSide / 4);
    const uint32_t ring_a = smem_addr(ring);

    const int len = p.kv_len[seq];
    const Seen seen = seen_of(p, len, KEYS);
    const int from = seen.from, end = seen.end, base = seen.base, ntile = seen.tiles;
    if (threadIdx.x == 0 && rank == 0) {
        if (len < 0) atomicOr(p.c.status, AMOE_KV_BAD_LENGTHS);
        if (len > end) atomicOr(p.c.status, AMOE_KV_PAST_TABLE);
    }
    const int t0 = (int)((int64_t)ntile * rank / split) + warp, t1 = (int)((int64_t)ntile * (rank + 1) / split);

    // The queries of NB blocks of eight heads as the scores' B operand: lane's head g of a block.  qs: the factors of the
    // heads 2c and 2c + 1 whose scores the lane gets.
    uint32_t qb[NB][D / 16][2];
    float qs[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const int r = row0 + g + 8 * nb;
        const bool live = r < p.group;
        const char *src = p.q.p + seq * p.q.ts + (int64_t)(kvh * p.group + (live ? r : 0)) * p.q.hs;
        auto pair = [&](int d) -> uint32_t { return live ? *reinterpret_cast<const uint32_t *>(src + d * 2) : 0u; };
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            // E4M3: a thread's 16-byte chunk of a key holds four steps' operands of its column pair
            const int d = T::kFp8 ? (c * (D / 64) + ks / 4) * 16 + ks % 4 * 4 : ks * 16 + 2 * c;
            qb[nb][ks][0] = pair(d), qb[nb][ks][1] = pair(T::kFp8 ? d + 2 : d + 8);
        }
        float factor = p.scale_log2;
        if (T::kFp8 && p.q_type == AMOE_GGUF_BF16) {
            // bf16 queries as f16: the row's largest value brought to [1, 2) by a power of two, which
            // the score gets back; what f16 then loses is below 2^-25 of that value
            float big = 0.0f;
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&qb[nb][ks][i]));
                    big = fmaxf(big, fmaxf(fabsf(f.x), fabsf(f.y)));
                }
            big = quad_max(big);
            const int e = big > 0.0f ? min(max((int)(__float_as_uint(big) >> 23) - 127, -126), 126) : 0;
            const float by = __uint_as_float((uint32_t)(127 - e) << 23);
            factor *= __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&qb[nb][ks][i]));
                    qb[nb][ks][i] = pack2<AMOE_GGUF_F16>(f.x * by, f.y * by);
                }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) qs[nb][i] = __shfl_sync(0xffffffffu, factor, (2 * c + i) * 4);
    }

    // A tile lies in one page where pages hold whole tiles; otherwise each lane looks its key's page up.
    constexpr int LOG = KEYS == 32 ? 5 : 4;
    constexpr uint32_t FULL = KEYS == 32 ? 0xffffffffu : 0xffffu;
    const bool whole = p.c.shift >= LOG;
    const int32_t *table = p.c.table + (int64_t)seq * p.c.table_stride;
    // Page of tile t (of this lane's key), -1 where there is none.
    auto page_for = [&](int t) -> int {
        if (t >= t1) return -1;
        int pos = base + t * KEYS;
        if (!whole) {
            pos += lane % KEYS;
            if (pos < from || pos >= end) return -1;
        }
        const int page = table[pos >> p.c.shift];
        if (page >= 0 && page < p.c.pages) return page;
        atomicOr(p.c.status, AMOE_KV_BAD_PAGE);
        return -1;
    };
    uint32_t shifts = 0;  // E4M3: where in its word each staged key's scale stands, two bits a stage
    const uint32_t row_in = lane / CPR, ch_in = lane % CPR;
    auto issue = [&](int t, int stage, int page) {
        const int at = base + t * KEYS;
        const uint32_t dst = ring_a + stage * T::kStage;
        uint32_t live, row;  // this lane's key's row in the pages
        if (whole) {
            // the keys from `from` to `end` of this tile
            live = FULL;
            if (at < from) live &= FULL << (from - at);
            if ((uint32_t)at + KEYS > (uint32_t)end) live &= FULL >> ((uint32_t)at + KEYS - end);  // may pass 2^31
            if (page < 0) live = 0;
            const uint32_t first = page >= 0 ? (uint32_t)cache_row(p.c, page, kvh, at) : 0u;
            row = first + lane % KEYS;
            const char *k = p.c.k + (int64_t)first * ROW + lane * 16, *v = p.c.v + (int64_t)first * ROW + lane * 16;
            if (live == FULL) {
#pragma unroll
                for (int i = 0; i < KEYS * CPR / 32; ++i) {
                    const uint32_t to = dst + chunk_at<ROW>(i * (32 / CPR) + row_in, ch_in);
                    copy16(to, k + i * 512);
                    copy16(to + KEYS * ROW, v + i * 512);
                }
            } else {
#pragma unroll
                for (int i = 0; i < KEYS * CPR / 32; ++i) {
                    const int r = i * (32 / CPR) + row_in;
                    const uint32_t to = dst + chunk_at<ROW>(r, ch_in);
                    copy16(to, k + i * 512, live >> r & 1u);
                    copy16(to + KEYS * ROW, v + i * 512, live >> r & 1u);
                }
            }
        } else {
            row = page >= 0 ? (uint32_t)cache_row(p.c, page, kvh, at + lane % KEYS) : 0u;
            live = __ballot_sync(0xffffffffu, page >= 0) & FULL;
#pragma unroll
            for (int i = 0; i < KEYS * CPR / 32; ++i) {
                const int r = i * (32 / CPR) + row_in;
                const int64_t off = (int64_t)__shfl_sync(0xffffffffu, row, r) * ROW + ch_in * 16;
                const uint32_t to = dst + chunk_at<ROW>(r, ch_in);
                copy16(to, p.c.k + off, live >> r & 1u);
                copy16(to + KEYS * ROW, p.c.v + off, live >> r & 1u);
            }
        }
        if constexpr (T::kFp8) {
            const bool on = live >> lane & 1u;
            const int64_t word = on ? row & ~3u : 0u;
            const int64_t left = ((p.c.pages * p.c.heads) << p.c.shift) - word;
            const int n = on ? (left < 4 ? (int)left : 4) : 0;
            const uint32_t to = smem_addr(side + stage * 64 + lane);
            copy4(to, p.c.ks + word, n);
            copy4(to + 128, p.c.vs + word, n);
            shifts = shifts << 2 | (row & 3u);
        }
        if (lane == 0) masks[stage] = live;
    };

    // o: rows are elements, columns heads; m, n, l: of the lane's two heads of each block, l over its own keys.  m: the
    // maximum less kShift, which o (and l, but for E4M3) is relative to; n: the maximum that l is relative to for E4M3
    float o[D / 16][NB][4] = {}, m[NB][2], n[NB][2], l[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 2; ++i) m[nb][i] = n[nb][i] = -INFINITY, l[nb][i] = 0.0f;
    {
        int pages[STAGES - 1];
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) pages[i] = page_for(t0 + i * kWarps);
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) {
            if (t0 + i * kWarps < t1) issue(t0 + i * kWarps, i, pages[i]);
            copy_commit();
        }
    }
    int ahead = page_for(t0 + (STAGES - 1) * kWarps);
    int stage = 0, fill = STAGES - 1;
    for (int t = t0; t < t1; t += kWarps) {
        const int tn = t + (STAGES - 1) * kWarps;
        if (tn < t1) issue(tn, fill, ahead);
        copy_commit();
        ahead = page_for(tn + kWarps);
        copy_wait<STAGES - 1>();
        __syncwarp();
        const uint32_t mask = masks[stage];
        const uint32_t kt = ring_a + stage * T::kStage, vt = kt + KEYS * ROW;
        if constexpr (T::kFp8) {
            // this lane's key: 2^e of its K scale and e of its V scale, for the lanes that hold its scores.
            // back: how many stages were issued since this one, fewer than the ring holds at the end
            const int back = min(STAGES - 1, (t1 - 1 - t) / kWarps);
            const uint32_t sh = (shifts >> (2 * back) & 3u) * 8;
            uint32_t *sc = side + stage * 64;
            const uint32_t kb = sc[lane] >> sh & 0xffu, vb = sc[32 + lane] >> sh & 0xffu;
            const bool on = mask >> lane & 1u;
            __syncwarp();
            reinterpret_cast<float2 *>(sc)[lane] =
                make_float2(e8m0_to_float(kb), !on ? 0.0f : vb == 255u ? NAN : (float)(int)vb - 127.0f);
            __syncwarp();
        }

        // scores: rows are keys, columns heads
        float sc[MT][NB][4];
#pragma unroll
        for (int t16 = 0; t16 < MT; ++t16) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) sc[t16][nb][0] = sc[t16][nb][1] = sc[t16][nb][2] = sc[t16][nb][3] = 0.0f;
            if constexpr (T::kFp8) {
#pragma unroll
                for (int seg = 0; seg < D / 64; ++seg) {
                    uint32_t w[2][4];
#pragma unroll
                    for (int hi = 0; hi < 2; ++hi) {
                        const uint32_t a = kt + chunk_at<ROW>(t16 * 16 + hi * 8 + g, c * (D / 64) + seg);
                        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                                     : "=r"(w[hi][0]), "=r"(w[hi][1]), "=r"(w[hi][2]), "=r"(w[hi][3])
                                     : "r"(a)
                                     : "memory");
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t a[4];
                        e4m3x4_to_f16x2(w[0][i], a[0], a[2]);
                        e4m3x4_to_f16x2(w[1][i], a[1], a[3]);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb)
                            mma16<TYPE>(sc[t16][nb], a, qb[nb][seg * 4 + i][0], qb[nb][seg * 4 + i][1]);
                    }
                }
            } else {
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) {
                    uint32_t a[4];
                    ldm4(a, kt + chunk_at<ROW>(t16 * 16 + lane % 16, ks * 2 + lane / 16));
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) mma16<TYPE>(sc[t16][nb], a, qb[nb][ks][0], qb[nb][ks][1]);
                }
            }
        }
        // to log2; E4M3: with the keys' scales, the values' exponents beside
        float ev[MT][2];
        bool grown = false;
#pragma unroll
        for (int t16 = 0; t16 < MT; ++t16)
#pragma unroll
            for (int hi = 0; hi < 2; ++hi) {
                float by = 1.0f;
                ev[t16][hi] = 0.0f;
                if constexpr (T::kFp8) {
                    const float2 x = reinterpret_cast<const float2 *>(side + stage * 64)[t16 * 16 + hi * 8 + g];
                    by = x.x, ev[t16][hi] = x.y;
                }
                const bool on = mask >> (t16 * 16 + hi * 8 + g) & 1u;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float &x = sc[t16][nb][2 * hi + i];
                        x = on ? x * (T::kFp8 ? by * qs[nb][i] : qs[nb][i]) : -INFINITY;
                        if constexpr (T::kFp8) grown |= x - n[nb][i] > 8.0f;
                        grown |= x + ev[t16][hi] - m[nb][i] > T::kTop;
                    }
            }
        // The maxima are lazy: they move, and what hangs on them with them, when some weight outgrew
        // what it may (2^15 in f16, 2^8 in bf16 and in E4M3's denominator).
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float top = -INFINITY, ntop = -INFINITY;
#pragma unroll
                    for (int t16 = 0; t16 < MT; ++t16)
#pragma unroll
                        for (int hi = 0; hi < 2; ++hi) {
                            top = fmaxf(top, sc[t16][nb][2 * hi + i] + ev[t16][hi]);
                            ntop = fmaxf(ntop, sc[t16][nb][2 * hi + i]);
                        }
                    const float mm = fmaxf(m[nb][i], keys_max(top) - T::kShift), keep = ex2(m[nb][i] - (mm == -INFINITY ? 0.0f : mm));
#pragma unroll
                    for (int j = 0; j < D / 16; ++j) o[j][nb][i] *= keep, o[j][nb][2 + i] *= keep;
                    m[nb][i] = mm;
                    if constexpr (T::kFp8) {
                        const float nn = fmaxf(n[nb][i], keys_max(ntop));
                        l[nb][i] *= ex2(n[nb][i] - (nn == -INFINITY ? 0.0f : nn));
                        n[nb][i] = nn;
                    } else {
                        l[nb][i] *= keep;
                    }
                }
        }
        // the weights, transposed to the B operand of the values' products
        uint32_t pb[MT][NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            float z[2], y[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                z[i] = m[nb][i] == -INFINITY ? 0.0f : m[nb][i];
                y[i] = n[nb][i] == -INFINITY ? 0.0f : n[nb][i];
            }
#pragma unroll
            for (int t16 = 0; t16 < MT; ++t16)
#pragma unroll
                for (int hi = 0; hi < 2; ++hi) {
                    float w[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float x = sc[t16][nb][2 * hi + i];
                        w[i] = ex2(x + ev[t16][hi] - z[i]);
                        l[nb][i] += T::kFp8 ? ex2(x - y[i]) : w[i];
                    }
                    pb[t16][nb][hi] = transposed(pack2<TYPE>(w[0], w[1]));
                }
        }
        // values times weights: rows are elements, columns heads
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
            if constexpr (T::kFp8) {
                // a register holds two keys' codes of elements 2g and 2g + 1 of the chunk: element pairs become key pairs,
                // even elements the upper eight rows and odd ones the lower
                uint32_t b[4];
                ldm4t(b, vt + chunk_at<ROW>(lane, j));
#pragma unroll
                for (int t16 = 0; t16 < MT; ++t16) {
                    uint32_t a[4];
                    e4m3x4_to_f16x2(__byte_perm(b[2 * t16], 0, 0x3120), a[0], a[1]);
                    e4m3x4_to_f16x2(__byte_perm(b[2 * t16 + 1], 0, 0x3120), a[2], a[3]);
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) mma16<TYPE>(o[j][nb], a, pb[t16][nb][0], pb[t16][nb][1]);
                }
            } else {
#pragma unroll
                for (int t16 = 0; t16 < MT; ++t16) {
                    uint32_t a[4];
                    ldm4t(a, vt + chunk_at<ROW>(t16 * 16 + lane % 8 + lane / 16 * 8, j * 2 + lane / 8 % 2));
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) mma16<TYPE>(o[j][nb], a, pb[t16][nb][0], pb[t16][nb][1]);
                }
            }
        }
        __syncwarp();
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        fill = fill + 1 == STAGES ? 0 : fill + 1;
    }
    copy_wait<0>();
    __syncthreads();

    // join: the warps' sums in shared memory, then the cluster's
    float *part = reinterpret_cast<float *>(smem);
    {
        float *mine = part + (1 + warp) * T::kPart;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float sum = keys_sum(l[nb][i]);
                const int r = nb * 8 + 2 * c + i;
                if (g == 0) {
                    mine[16 * D + r] = m[nb][i];
                    mine[16 * D + 16 + r] = T::kFp8 ? n[nb][i] : m[nb][i];
                    mine[16 * D + 32 + r] = sum;
                }
#pragma unroll
                for (int j = 0; j < D / 16; ++j) {
                    float *x = mine + r * D + j * 16;
                    x[T::kFp8 ? 2 * g : g] = o[j][nb][i];
                    x[T::kFp8 ? 2 * g + 1 : g + 8] = o[j][nb][2 + i];
                }
            }
    }
    __syncthreads();
    constexpr int LIVE = 8 * NB;  // heads of the tile that the instantiation fills
    for (int i = threadIdx.x; i < LIVE * D / 4; i += kThreads) {
        const int r = i / (D / 4);
        float top = -INFINITY;
#pragma unroll
        for (int w = 1; w <= kWarps; ++w) top = fmaxf(top, part[w * T::kPart + 16 * D + r]);
        const float z = top == -INFINITY ? 0.0f : top;
        float4 a = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 1; w <= kWarps; ++w) {
            const float f = exp2f(part[w * T::kPart + 16 * D + r] - z);
            const float4 x = *reinterpret_cast<const float4 *>(part + w * T::kPart + i * 4);
            a.x += f * x.x, a.y += f * x.y, a.z += f * x.z, a.w += f * x.w;
        }
        *reinterpret_cast<float4 *>(part + i * 4) = a;
    }
    if (threadIdx.x < LIVE) {
        const int r = threadIdx.x;
        float top = -INFINITY, ntop = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 1; w <= kWarps; ++w) {
            top = fmaxf(top, part[w * T::kPart + 16 * D + r]);
            ntop = fmaxf(ntop, part[w * T::kPart + 16 * D + 16 + r]);
        }
        const float z = ntop == -INFINITY ? 0.0f : ntop;
#pragma unroll
        for (int w = 1; w <= kWarps; ++w)
            sum += part[w * T::kPart + 16 * D + 32 + r] * exp2f(part[w * T::kPart + 16 * D + 16 + r] - z);
        part[16 * D + r] = top, part[16 * D + 16 + r] = ntop, part[16 * D + 32 + r] = sum;
    }
    if constexpr (WIDE) {
        __syncthreads();
        float4 *dst = reinterpret_cast<float4 *>(
            p.work + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * T::kPart);
        for (int i = threadIdx.x; i < T::kPart / 4; i += kThreads)
            if (i < LIVE * D / 4 || i >= 4 * D) dst[i] = reinterpret_cast<const float4 *>(part)[i];
        return;
    }
    cg::cluster_group cluster = cg::this_cluster();
    if (split > 1) cluster.sync();
    else __syncthreads();
    // each CTA of the cluster finishes its share of the elements
    const int rows = min(LIVE, p.group - row0);
    for (int i = rank * kThreads + threadIdx.x; i < rows * (D / 4); i += split * kThreads)
        finish<D>(p, seq, kvh * p.group + row0 + i / (D / 4), i, split,
                  [&](int w) { return split > 1 ? cluster.map_shared_rank(part, w) : part; });
    if (split > 1) cluster.sync();  // no CTA leaves while others read its sums
}

// The join of the CTAs that did not share a cluster: a CTA takes one row.  Lanes take partial sums for
// the maxima and factors, then threads take (four elements, every so many-th partial sum): no
// chain of loads is longer than a few.
constexpr int kJoinThreads = 256;
template <int D, int CACHE>
__global__ void __launch_bounds__(kJoinThreads) decode_join_kernel(const __grid_constant__ DecodeParams p) {
    using T = Tile<D, CACHE>;
    constexpr int COLS = D / 4, LANES = kJoinThreads / COLS;
    __shared__ float factor[kMaxWide], red[2][kJoinThreads / 32], total[kJoinThreads / 32];
    __shared__ float4 acc[LANES][COLS];
    const int seq = blockIdx.z, kvh = blockIdx.y % p.c.heads, row0 = blockIdx.y / p.c.heads * 16, r = blockIdx.x;
    if (row0 + r >= p.group) return;
    const Share share = share_of(p, T::kKeys, 0, seq);
    const int split = share.split;
    cudaGridDependencySynchronize();  // launched while the partial sums are still being made
    const int h = kvh * p.group + row0 + r, tid = threadIdx.x;
    const float *work = p.work + ((int64_t)blockIdx.y * p.split + share.first) * T::kPart;
    const float sink = p.sinks ? p.sinks[h] * kLog2e : -INFINITY;
    float m = -INFINITY, n = -INFINITY, l = 0.0f;
    if (tid < split) {
        const float *x = work + (int64_t)tid * T::kPart + 16 * D + r;
        m = x[0], n = x[16], l = x[32];
    }
    auto block_max = [&](float v, float *slots) {
#pragma unroll
        for (int i = 16; i; i >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, i));
        if (tid % 32 == 0) slots[tid / 32] = v;
        __syncthreads();
        float top = slots[0];
#pragma unroll
        for (int i = 1; i < kJoinThreads / 32; ++i) top = fmaxf(top, slots[i]);
        return top;
    };
    const float top = block_max(m, red[0]), ntop = fmaxf(sink, block_max(n, red[1]));
    const float z = top == -INFINITY ? 0.0f : top, y = ntop == -INFINITY ? 0.0f : ntop;
    float sum = l * exp2f(n - y);
#pragma unroll
    for (int i = 16; i; i >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
    if (tid % 32 == 0) total[tid / 32] = sum;
    if (tid < split) factor[tid] = exp2f(m - z);
    __syncthreads();
    const int col = tid % COLS, lane = tid / COLS;
    float4 a = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (int w = lane; w < split; w += LANES) {
        const float f = factor[w];
        const float4 v = *reinterpret_cast<const float4 *>(work + (int64_t)w * T::kPart + r * D + col * 4);
        a.x += f * v.x, a.y += f * v.y, a.z += f * v.z, a.w += f * v.w;
    }
    acc[lane][col] = a;
    __syncthreads();
    if (tid >= COLS) return;
#pragma unroll
    for (int i = 1; i < LANES; ++i) {
        const float4 v = acc[i][col];
        a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
    }
    sum = exp2f(sink - y);
#pragma unroll
    for (int i = 0; i < kJoinThreads / 32; ++i) sum += total[i];
    store_row(p, seq, h, col, a, sum, top, y);
}

constexpr int kMaxDevices = 64;

template <int D, int CACHE, int NB, bool WIDE>
cudaError_t launch(const DecodeParams &p, int device, int units, int seqs, cudaStream_t st) {
    using T = Tile<D, CACHE>;
    auto *kernel = decode_attn_kernel<D, CACHE, NB, WIDE>;
    static std::atomic<bool> ready[kMaxDevices];
    if (!ready[device].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, T::kSmem);
        if (e != cudaSuccess) return e;
        ready[device].store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(p.split, units, WIDE ? 1 : seqs);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = T::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)p.split, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = WIDE ? 0 : 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    if (e != cudaSuccess || !WIDE) return e;
    cudaLaunchConfig_t join{};
    join.gridDim = dim3(8 * NB, units, seqs);
    join.blockDim = dim3(kJoinThreads);
    join.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    join.attrs = attr;
    join.numAttrs = 1;
    return cudaLaunchKernelEx(&join, decode_join_kernel<D, CACHE>, p);
}

// How a call is laid out: CTAs to a (sequence, group of query heads), and whether they join through
// the workspace.
struct Layout {
    int split;
    bool wide;
    int64_t bytes;
};

// Clusters (powers of two up to kCluster) while they fill the GPU: one launch.  Where even the largest leaves it half empty
// and the length allows more, or where the lengths may differ much and there are CTAs enough to share them out finely, as
// many CTAs as fit at once, joined by a second launch.  Cluster -> shared, 8 kv heads of 64: 7 sequences of 500-2000
// tokens and one of 60000, bf16, 58 -> 29 us, E4M3 60 -> 25; 8 of 10000-20000 46 -> 43 and 36 -> 32; 8 of 20000 62 -> 55 and
// 38 -> 38; 4 of 20000 29 -> 32 and 26 -> 24.  With fewer than four CTAs a sequence it loses: 32 of 8192, bf16, 87 -> 92,
// 48 of 4096-8192, E4M3, 71 -> 94; and so it does for short ones: 8 of 700, E4M3, 7.6 -> 9.3.
Layout layout(int64_t units, int64_t seqs, int64_t tokens, int row_bytes, int part_floats, int ctas) {
    const int keys = row_bytes == 256 ? 16 : 32;
    const int64_t tiles = (tokens - 1) / keys + 1, all = units * seqs;
    const int want = 6 * 148;
    Layout l{1, false, 0};
    while (l.split < kCluster && all * l.split < want && tiles > l.split * kWarps) l.split *= 2;
    const int64_t fit = std::min<int64_t>(ctas * 148 / units, kMaxWide * seqs);
    const int64_t s = std::min<int64_t>(fit, tiles * seqs / kWarps);
    const bool idle = l.split == kCluster && all * l.split < want / 2 && s > l.split * seqs;
    const bool shared = seqs > 1 && fit >= 4 * seqs && tokens >= 8192;
    if (idle || shared) l = {(int)s, true, units * s * part_floats * 4};
    return l;
}

template <int D, int CACHE>
Layout layout_for(int64_t units, int64_t seqs, int64_t tokens) {
    return layout(units, seqs, tokens, Tile<D, CACHE>::kRow, Tile<D, CACHE>::kPart, Tile<D, CACHE>::kCtas);
}

Layout layout_of(int D, int cache, int64_t units, int64_t seqs, int64_t tokens) {
    if (D == 64)
        return cache == AMOE_KV_E4M3 ? layout_for<64, AMOE_KV_E4M3>(units, seqs, tokens)
                                     : layout_for<64, AMOE_GGUF_F16>(units, seqs, tokens);
    return cache == AMOE_KV_E4M3 ? layout_for<128, AMOE_KV_E4M3>(units, seqs, tokens)
                                 : layout_for<128, AMOE_GGUF_F16>(units, seqs, tokens);
}

template <int D, int CACHE>
cudaError_t launch_rows(const DecodeParams &p, int device, int units, int seqs, bool wide, cudaStream_t st) {
    if (p.group > 8)
        return wide ? launch<D, CACHE, 2, true>(p, device, units, seqs, st)
                    : launch<D, CACHE, 2, false>(p, device, units, seqs, st);
    return wide ? launch<D, CACHE, 1, true>(p, device, units, seqs, st)
                : launch<D, CACHE, 1, false>(p, device, units, seqs, st);
}

template <int D>
cudaError_t launch_cache(const DecodeParams &p, int cache, int device, int units, int seqs, bool wide,
                         cudaStream_t st) {
    if (cache == AMOE_GGUF_F16) return launch_rows<D, AMOE_GGUF_F16>(p, device, units, seqs, wide, st);
    if (cache == AMOE_GGUF_BF16) return launch_rows<D, AMOE_GGUF_BF16>(p, device, units, seqs, wide, st);
    return launch_rows<D, AMOE_KV_E4M3>(p, device, units, seqs, wide, st);
}

// Keys that a row sees at most, as far as the caller says.
int64_t most_keys(const amoe_kv_cache *cache, const amoe_kv_seqs *seqs, int window, int max_len) {
    int64_t tokens = (int64_t)seqs->table_stride * cache->page_size;
    if (max_len > 0 && max_len < tokens) tokens = max_len;
    if (window > 0 && window < tokens) tokens = window;
    return tokens;
}

int64_t units_of(int q_heads, int kv_heads) { return (int64_t)kv_heads * ((q_heads / kv_heads + 15) / 16); }

}  // namespace
}  // namespace attn
}  // namespace amoe

using namespace amoe;
using namespace amoe::attn;

extern "C" {

int64_t amoe_attn_decode_workspace(const amoe_kv_cache *cache, const amoe_kv_seqs *seqs, int32_t q_heads,
                                   int32_t window, int32_t max_len) {
    if (int rc = check_cache(cache, seqs)) return rc;
    if (int rc = check_group(q_heads, cache->kv_heads)) return rc;
    if (window < 0 || max_len < 0) return reject("window and max_len must not be negative");
    return layout_of(cache->head_dim, cache->type, units_of(q_heads, cache->kv_heads), seqs->seqs,
                     most_keys(cache, seqs, window, max_len)).bytes;
}

int amoe_attn_decode(const amoe_kv_cache *cache, const amoe_kv_seqs *seqs, const amoe_attn *attn, const amoe_rows *q,
                     const amoe_rows *out, const int32_t *kv_len, int32_t max_len, void *workspace,
                     int64_t workspace_bytes, void *stream) {
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
    const int64_t units = units_of(q->heads, cache->kv_heads);
    if (units > 65535) return reject("more than 65535 groups of query heads in one decode call");
    if (cache->device < 0 || cache->device >= kMaxDevices) return reject("device ordinal out of range");
    DecodeParams p{};
    p.c = cache_dev(cache, seqs);
    p.q = rows_dev(q), p.out = rows_dev(out);
    p.kv_len = kv_len, p.sinks = attn->sinks;
    p.scale_log2 = attn_scale(attn, D) * kLog2e;
    p.window = attn->window, p.group = q->heads / cache->kv_heads, p.q_type = q->type;
    const Layout l =
        layout_of(D, cache->type, units, seqs->seqs, most_keys(cache, seqs, attn->window, max_len));
    if (l.wide && (!workspace || workspace_bytes < l.bytes))
        return reject("decode needs a workspace of " + std::to_string(l.bytes) + " bytes");
    if (l.wide && (reinterpret_cast<uintptr_t>(workspace) & 15)) return reject("workspace must be 16-byte aligned");
    p.split = l.split, p.seqs = seqs->seqs, p.work = static_cast<float *>(workspace);
    DeviceScope scope;
    cudaError_t e = scope.enter(cache->device);
    if (e != cudaSuccess) return cuda_error(e, "cudaSetDevice");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    e = D == 64 ? launch_cache<64>(p, cache->type, cache->device, (int)units, seqs->seqs, l.wide, st)
                : launch_cache<128>(p, cache->type, cache->device, (int)units, seqs->seqs, l.wide, st);
    return e == cudaSuccess ? AMOE_OK : cuda_error(e, "decode kernel");
}

}  // extern "C"
