// attn_prefill.cu -- causal attention of packed prompts with grouped heads, learned sinks
// and a sliding window (CausalAttentionWithConfig, internal/backend/cpuref/attention.go:82-171),
// on tcgen05 MMAs with the running maximum and sum of a softmax over key tiles.
//
//   s_j = scale q.k_j over the visible keys, m = max s_j,
//   out = sum exp(s_j - m) v_j / (sum exp(s_j - m) + exp(sink - m))
//
// One CTA takes 128 rows of one kv head: `group` query heads x 128 / group tokens, so that the
// keys it stages serve all of them and the diagonal wastes little.  Q, K and V arrive by TMA
// in 128-byte swizzled rows; S = Q K^T goes to TMEM; four warps (a thread a row) read it back, keep the
// row's maximum and sum, and write the weights, rounded to the inputs' type, to TMEM, where they are
// the A operand of O += P V.  V is staged as it lies in memory ([keys][d], the MN-major B operand).  S is read into
// registers at once, so the next tile's Q K^T runs under this tile's exponentials; and three CTAs share an
// SM (two of 128-wide heads: TMEM and shared memory allow no more), so that one's exponentials run while
// another waits for its scores or looks for their maximum.
//
// What bounds it.  64-wide heads: the exponentials, one a score on a pipe of 16 a clock an SM; 128 x 64 scores take 512
// clocks there and 256 on the tensor cores.  Measured in steady state: 600 clocks a tile; 8192 tokens of 64 heads over
// 8: 687 us in short runs, 800 TFLOP/s, 0.49 of the measured bf16 GEMM; 763 us and 720 TFLOP/s call after call, when
// the power cap lowers the clock (0.52 of the GEMM's sustained rate).  Two row tiles of one persistent CTA (0.93 ms: fewer warps
// to hide a tile's chain of waits), two threads a row (0.85 ms: the pair has to agree on its maximum) and P in S's
// own columns (0.80 ms: Q K^T waits for P V) were slower.  128-wide heads: the tensor cores and the operands they read
// from shared memory; 1500 tokens in three chunks behind 2600-2800 each: 90 to 95 us in a graph, 100 a call (730 TFLOP/s).
// Windows and short prompts: a CTA's start.
//
// A few queries behind many keys, or the last wave of a larger call, do not fill the GPU: the keys of those tiles are
// split over CTAs, and a second kernel joins the partial sums (`layout` below chooses, with what it measured).
//
// The maximum is lazy: O and the sum are rescaled only when a row's maximum has grown by more
// than 2^8 (2^4 in f16, whose weights carry a factor: attn.cuh) since the last time, which float32 sums hold without loss.
//
// A key that a row must not see has weight 0, but 0 times an infinity or NaN in its value is NaN.  Values behind the
// tile's last visible key are overwritten with zeros in shared memory.  Where a row's result still is not finite the CTA
// does its tiles once more, and the feeding warp now takes out what is not finite among the keys that only some of the
// rows see (at the diagonal and at the window's edge); the rows that see such a key add its value at the end, for with any weight
// above zero the sum is that infinity or NaN.  Finite inputs never go that way, others take about twice the time at most
// (4096 tokens 220 us, with one infinity 273, all NaN 486; looking through those keys at once cost windows 8 to 35 %).
#include "attn.cuh"
#include "tc_ptx.cuh"

#include <algorithm>
#include <atomic>

namespace amoe {
namespace attn {
namespace {

using bs::mbar_arrive;
using bs::mbar_expect_tx;
using bs::mbar_init;
using bs::smem_u32;
using bs::tc_fence_after;
using bs::tc_fence_before;

constexpr int kRows = 128;
constexpr int kStages = 2, kBars = 5 + 2 * kStages;
constexpr int kSoftWarps = 4, kFeedWarp = 4, kThreads = 160;

struct PrefillParams {
    RowsDev v, out;
    const int32_t *cu_q, *cu_k;
    const float *sinks;
    float scale_log2;
    int window, q_tokens, k_tokens, seqs, group, tile_tokens, kv_heads;
    int whole;    // row tiles (of all kv heads) that one CTA takes; those behind them have
    int split;    // so many CTAs to their keys
    float *work;  // split > 1: their partial sums, [tile][part][D + 2][kRows]: each row's O, m and l
};

template <int D>
struct Cfg {
    static constexpr int N = 64;                  // keys of a tile
    static constexpr int kHalves = D / 64;        // 128-byte column blocks of a row
    static constexpr int kQBytes = kRows * D * 2;
    static constexpr int kTileBytes = N * D * 2;
    static constexpr int kCtas = D == 64 ? 3 : 2;  // to an SM
    // Which of sixteen pairs of exponentials the FMA pipe computes: two.  8192 tokens of 64 heads: 733 us with
    // none, 704 with two, 713 with four; 128-wide heads, which products bound, gain nothing.
    static __device__ constexpr bool poly(int i) { return D == 64 && i % 8 == 7; }
    static constexpr int kSmem = 1024 + kQBytes + 2 * kStages * kTileBytes + 256;
    // TMEM columns: S and O in one allocation (powers of two), P in another where three CTAs share the SM
    static constexpr int kTmemCols = D == 64 ? 128 : 256, kTmemP = D == 64 ? 32 : 0;
    static constexpr int kS = 0, kO = N, kP = D == 64 ? 0 : N + D;
    static_assert(kO + D + (kTmemP ? 0 : N / 2) <= kTmemCols && kCtas * (kTmemCols + kTmemP) <= 512, "TMEM columns");
    static_assert(kCtas * (kSmem + 1024) <= 228 * 1024, "shared memory of an SM");
};

// What a CTA works on, found by one warp and shared.
struct Work {
    int tok0, tokens;    // first query row and how many of the tile's are the sequence's
    int at0;             // position of the first among its keys
    int k0, lo, hi;      // the sequence's first key row; the tile's visible keys [lo, hi), or this CTA's part of them
    int odd;             // values that are not finite were left out of the careful pass's products
    int dead;            // a bounded wait gave up
    int found;
};

// Waits for a phase, a second or so at most; at once when an earlier wait of the CTA gave up.
__device__ __forceinline__ bool wait_bar(uint64_t *bar, uint32_t parity, Work *w) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
    if (*reinterpret_cast<volatile int *>(&w->dead)) return false;
    return bs::mbar_wait(bar, parity, &w->dead, 1);
}

// The same for a whole warp, which stays together when a wait gives up.
__device__ __forceinline__ bool wait_warp(uint64_t *bar, uint32_t parity, Work *w) {
    return __all_sync(0xffffffffu, wait_bar(bar, parity, w));
}

__device__ __forceinline__ void tma_3d(void *dst, const CUtensorMap *tm, uint64_t *bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(tm)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

// Operand in 128-byte swizzled rows, eight-row groups 1024 bytes apart.  lbo: bytes between 64-column
// blocks, which only the MN-major operand of 128 columns has.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr, uint32_t lbo) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(1024u >> 4) << 32 |
           (uint64_t)1u << 46 | (uint64_t)2u << 61;
}

// kind::f16: f32 accumulators, both operands of TYPE, M = 128.
template <int TYPE>
__device__ __forceinline__ uint32_t idesc(int n, bool b_mn) {
    const uint32_t t = TYPE == AMOE_GGUF_F16 ? 0u : 1u;
    return 1u << 4 | t << 7 | t << 10 | (b_mn ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(kRows >> 4) << 24;
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool add) {
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
                 "l"(a), "l"(b), "r"(id), "r"((uint32_t)add)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, bool add) {
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
                 "r"(a), "l"(b), "r"(id), "r"((uint32_t)add)
                 : "memory");
}
// One lane of a converged warp.  The compiler knows what elect.sync picks to be one thread and keeps
// descriptors in uniform registers; behind `lane == 0` an MMA took 100 cycles to issue.
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(e));
    return e != 0;
}

__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}

// 16 columns of this warp's lanes.
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// 64 columns of this warp's lanes, waited for in the same statement.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float (&v)[64]) {
    uint32_t r[64];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,"
        "%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
          "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
          "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
          "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
          "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));  // volatile: a run of them stays a run
    return y;
}

// The larger, NaN where one is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Two float32 lanes in one instruction.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpair(uint64_t r) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(r));
    return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// 2^x of two values on the FMA pipe, to 2^-22.1: with n the integer next to x (read from the low bits of
// x + 1.5 * 2^23) and f = x - n in [-1/2, 1/2], 2^f by a polynomial of degree 5 fitted to the least relative error,
// and n added to its exponent.  Below -127 the result is a zero or the smallest subnormal, and so is it for NaN.
__device__ __forceinline__ float2 ex2_poly(float2 x) {
    x.x = fmaxf(x.x, -127.0f), x.y = fmaxf(x.y, -127.0f);
    const uint64_t v = pair(x.x, x.y), big = pair(12582912.0f, 12582912.0f);
    const uint64_t t = add2(v, big);
    const uint64_t f = fma2(add2(t, pair(-12582912.0f, -12582912.0f)), pair(-1.0f, -1.0f), v);
    uint64_t y = pair(0.001327647129073739f, 0.001327647129073739f);
    y = fma2(y, f, pair(0.009675540961325169f, 0.009675540961325169f));
    y = fma2(y, f, pair(0.05550713092088699f, 0.05550713092088699f));
    y = fma2(y, f, pair(0.24022120237350464f, 0.24022120237350464f));
    y = fma2(y, f, pair(0.6931469440460205f, 0.6931469440460205f));
    y = fma2(y, f, pair(1.0000001192092896f, 1.0000001192092896f));
    const float2 n = unpair(t), p = unpair(y);
    return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(n.x) << 23)),
                       __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(n.y) << 23)));
}

// One warp finds the sequence and rows of tile x: sequences in order, each one's last (longest) tile first; and of
// its keys the part-th part (-1: all).
template <int N>
__device__ __forceinline__ bool find_work(const PrefillParams &p, int x, int part, Work *w) {
    const int lane = threadIdx.x % 32;
    int before = 0;
    for (int s0 = 0; s0 < p.seqs; s0 += 32) {
        const int s = s0 + lane;
        int a = 0, b = 0, k0 = 0, k1 = 0, tiles = 0;
        if (s < p.seqs) {
            a = max(p.cu_q[s], 0), b = min(p.cu_q[s + 1], p.q_tokens);
            k0 = max(p.cu_k[s], 0), k1 = min(p.cu_k[s + 1], p.k_tokens);
            if (a < b) tiles = (b - a - 1) / p.tile_tokens + 1;
        }
        int upto = tiles;
#pragma unroll
        for (int i = 1; i < 32; i <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, i);
            if (lane >= i) upto += y;
        }
        const bool mine = tiles > 0 && x >= before + upto - tiles && x < before + upto;
        if (mine) {
            const int tile = before + upto - 1 - x;  // the last one first
            const int klen = max(k1 - k0, 0);
            w->tok0 = a + tile * p.tile_tokens;
            w->tokens = min(p.tile_tokens, b - w->tok0);
            w->at0 = klen - (b - w->tok0);
            w->k0 = k0;
            w->hi = max(w->at0 + w->tokens, 0);
            w->lo = p.window > 0 ? max(w->at0 - p.window + 1, 0) : 0;
            if (part >= 0 && w->hi > w->lo) {
                const int tiles = (w->hi - w->lo - 1) / N + 1;
                const int t0 = (int)((int64_t)tiles * part / p.split), t1 = (int)((int64_t)tiles * (part + 1) / p.split);
                w->hi = min(w->hi, w->lo + t1 * N);
                w->lo = min(w->lo + t0 * N, w->hi);
            }
            w->odd = w->dead = 0;
        }
        if (__any_sync(0xffffffffu, mine)) return true;
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}

// A sink's share of a denominator whose weights are relative to z (in log2).  It may pass float32's range, and the row is then 0;
// a sink of +inf leaves inf / inf.
__device__ __forceinline__ float sink_weight(float sink, float z) {
    return sink == INFINITY ? NAN : ex2(sink * kLog2e - z);
}

// Zeros in the place of a word's elements that are not finite; true where there was one.
template <int TYPE>
__device__ __forceinline__ bool drop_odd(uint32_t &w) {
    constexpr uint32_t EXP = TYPE == AMOE_GGUF_F16 ? 0x7c007c00u : 0x7f807f80u;
    constexpr uint32_t ONE = TYPE == AMOE_GGUF_F16 ? 0x04000400u : 0x00800080u;  // carries a full exponent into the sign's place
    const uint32_t odd = ((w & EXP) + ONE) >> 15 & 0x00010001u;
    w &= ~(odd * 0xffffu);
    return odd != 0;
}

// The keys that all of a tile's rows see: [from, to).
struct Shared {
    int from, to;
};
__device__ __forceinline__ Shared shared_keys(int window, int at0, int tokens) {
    return {window > 0 ? at0 + tokens - window : 0, at0 + 1};
}

// What drop_odd took out of 32 elements of a row that sees the keys [from, to).  v: the row and elements of key 0.
template <int TYPE>
__device__ __forceinline__ void add_odd(float (&o)[32], const char *v, int64_t step, int from, int to, Shared all) {
#pragma unroll 1
    for (int j = from; j < to; ++j) {
        if (j >= all.from && j < all.to) {
            j = all.to - 1;
            continue;
        }
        const char *row = v + j * step;
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
            float x[8];
            load8<TYPE>(row + i * 2, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[i + e] += isfinite(x[e]) ? 0.0f : x[e];
        }
    }
}

// Where a CTA's shared memory lies and which tile it has, of which part of the keys (-1: all).
struct Cta {
    uint8_t *sm;
    uint64_t *bars;
    uint32_t *tmem_slot;
    uint32_t tmem, tmem_p;  // S and O; P
    Work *work;
    int tile, part;
};
// The columns' addresses, once they are allocated.
template <int D>
__device__ __forceinline__ void find_tmem(Cta &c) {
    c.tmem = c.tmem_slot[0], c.tmem_p = Cfg<D>::kTmemP ? c.tmem_slot[1] : c.tmem + Cfg<D>::kP;
}
template <int D, bool SPLIT>
__device__ __forceinline__ Cta this_cta(const PrefillParams &p) {
    extern __shared__ __align__(1024) uint8_t sm_raw[];
    Cta c;
    c.sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(sm_raw) + 1023) & ~uintptr_t(1023));
    c.bars = reinterpret_cast<uint64_t *>(c.sm + Cfg<D>::kQBytes + 2 * kStages * Cfg<D>::kTileBytes);
    c.tmem_slot = reinterpret_cast<uint32_t *>(c.bars + kBars);
    c.work = reinterpret_cast<Work *>(c.tmem_slot + 2);
    c.tile = blockIdx.x, c.part = -1;
    if (SPLIT && c.tile >= p.whole) {
        c.part = (c.tile - p.whole) % p.split;
        c.tile = p.whole + (c.tile - p.whole) / p.split;
    }
    return c;
}

// Barriers: q_full, k_full[2], v_full[2], s_full, s_free, p_full, o_done.
__device__ __forceinline__ void init_bars(uint64_t *bars) {
    for (int i = 0; i < kBars; ++i) mbar_init(bars + i, i == kBars - 3 || i == kBars - 2 ? kSoftWarps : 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}

// The CTA's tiles from the first to the last.  SPLIT: those from p.whole on have their keys split over p.split CTAs.  CAREFUL: once
// more, with values that are not finite kept from rows that do not see them.  True where this thread's row has a sum
// that is not finite.
template <int D, int TYPE, bool SPLIT, bool CAREFUL>
__device__ __forceinline__ bool tile_pass(const PrefillParams &p, const CUtensorMap *tm_q, const CUtensorMap *tm_k,
                                          const CUtensorMap *tm_v, const Cta &cta) {
    using C = Cfg<D>;
    constexpr int N = C::N, HALVES = C::kHalves;
    uint8_t *q_s = cta.sm, *k_s = q_s + C::kQBytes, *v_s = k_s + kStages * C::kTileBytes;
    uint64_t *q_full = cta.bars, *k_full = q_full + 1, *v_full = k_full + kStages, *s_full = v_full + kStages;
    uint64_t *s_free = s_full + 1, *p_full = s_free + 1, *o_done = p_full + 1;
    Work *work = cta.work;
    const uint32_t tmem = cta.tmem, tmem_p = cta.tmem_p;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, tile = cta.tile, part = cta.part, kvh = tile % p.kv_heads;
    bool odd_row = false;
    const int tok0 = work->tok0, at0 = work->at0, lo = work->lo, hi = work->hi, k0 = work->k0;
    const int tiles = hi > lo ? (hi - lo - 1) / N + 1 : 0;
    // columns of the last tile that hold a visible key, in whole MMA steps
    const int last_cols = tiles > 0 ? (hi - lo - (tiles - 1) * N + 15) / 16 * 16 : 0;

    if (warp == kFeedWarp) {
        // Copies and products.  A stage needs no barrier of its own to be refilled: S of tile j read (s_free)
        // says that its Q K^T is done with K, and the weights of tile j written (p_full) that the
        // products of tile j - 1 are done with V.
        auto load = [&](uint8_t *ring, const CUtensorMap *tm, uint64_t *full, int j) {
            const int s = j % kStages;
            mbar_expect_tx(full + s, C::kTileBytes);
            for (int h = 0; h < HALVES; ++h)
                tma_3d(ring + s * C::kTileBytes + h * N * 128, tm, full + s, h * 64, kvh, k0 + lo + j * N);
        };
        if (lane == 0 && tiles > 0) {
            if (!CAREFUL) {
                mbar_expect_tx(q_full, p.tile_tokens * p.group * D * 2);
                for (int h = 0; h < HALVES; ++h) tma_3d(q_s + h * kRows * 128, tm_q, q_full, h * 64, kvh * p.group, tok0);
            }
            for (int j = 0; j < kStages && j < tiles; ++j) {
                load(k_s, tm_k, k_full, j);
                load(v_s, tm_v, v_full, j);
            }
        }
        __syncwarp();
        const uint64_t q_d = desc_sw128(smem_u32(q_s), 16), k_d = desc_sw128(smem_u32(k_s), 16);
        const uint64_t v_d = desc_sw128(smem_u32(v_s), N * 128);
        bool ok = tiles > 0 && (CAREFUL || wait_warp(q_full, 0, work));
        int scored = 0, weighed = 0;  // tiles whose products are issued
        auto scores = [&](int j) {  // S = Q K^T of tile j
            if (j >= tiles) return;
            const int s = j % kStages;
            ok = wait_warp(k_full + s, (uint32_t)(j / kStages) & 1u, work);
            if (ok && j > 0) ok = wait_warp(s_free, (uint32_t)(j - 1) & 1u, work);
            if (!ok) return;
            tc_fence_after();
            if (elect_one()) {
                const uint32_t id = idesc<TYPE>(j + 1 == tiles ? last_cols : N, false);
                const uint64_t kd = k_d + s * (C::kTileBytes / 16);
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
                    mma_ss(tmem + C::kS, q_d + i / 4 * (kRows * 8) + i % 4 * 2, kd + i / 4 * (N * 8) + i % 4 * 2, id, i > 0);
                mma_commit(s_full);
                if (j > 0 && j - 1 + kStages < tiles) load(k_s, tm_k, k_full, j - 1 + kStages);
            }
            __syncwarp();
            scored = j + 1;
        };
        auto weigh = [&](int t) {  // O += P V of tile t
            if (t < 0 || !ok) return;
            const int s = t % kStages;
            ok = wait_warp(v_full + s, (uint32_t)(t / kStages) & 1u, work);
            if (!ok) return;
            const int cols = t + 1 == tiles ? last_cols : N;
            const int seen = hi - lo - t * N;
            bool odd = false;
            if (CAREFUL) {  // keys [0, edge) and [diag, end) of the tile are not for all rows
                const int key = lo + t * N, end = min(seen, N);
                const Shared all = shared_keys(p.window, at0, work->tokens);
                const int edge = min(max(all.from - key, 0), end), diag = min(max(all.to - key, edge), end);
                for (int i = lane; i < (edge + end - diag) * 8 * HALVES; i += 32) {
                    const int r = i / (8 * HALVES), h = i / 8 % HALVES;
                    uint4 *at = reinterpret_cast<uint4 *>(v_s + s * C::kTileBytes + h * N * 128 +
                                                          (r < edge ? r : diag + r - edge) * 128 + i % 8 * 16);
                    uint4 w = *at;
                    bool here = drop_odd<TYPE>(w.x);
                    here |= drop_odd<TYPE>(w.y);
                    here |= drop_odd<TYPE>(w.z);
                    here |= drop_odd<TYPE>(w.w);
                    if (here) *at = w;
                    odd |= here;
                }
                odd = __any_sync(0xffffffffu, odd);
                if (odd) work->odd = 1;
            }
            if (seen < cols) {  // no value behind the last visible key reaches the products
                for (int i = lane; i < (cols - seen) * 8 * HALVES; i += 32) {
                    const int h = i / ((cols - seen) * 8), r = i / 8 % (cols - seen);
                    *reinterpret_cast<uint4 *>(v_s + s * C::kTileBytes + h * N * 128 + (seen + r) * 128 + i % 8 * 16) =
                        make_uint4(0, 0, 0, 0);
                }
            }
            if (odd || seen < cols) {
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
            ok = wait_warp(p_full, (uint32_t)t & 1u, work);
            if (!ok) return;
            tc_fence_after();
            if (elect_one()) {
                const uint32_t id = idesc<TYPE>(D, true);
                const uint64_t vd = v_d + s * (C::kTileBytes / 16);
#pragma unroll
                for (int i = 0; i < N / 16; ++i)
                    if (i * 16 < cols) mma_ts(tmem + C::kO, tmem_p + i * 8, vd + i * 128, id, t > 0 || i > 0);
                mma_commit(o_done);
                if (t > 0 && t - 1 + kStages < tiles) load(v_s, tm_v, v_full, t - 1 + kStages);
            }
            __syncwarp();
            weighed = t + 1;
        };
        for (int j = 0; ok && j <= tiles; ++j) {
            scores(j);
            weigh(j - 1);
        }
        // Whatever gave up, nothing of the CTA's is in flight when it ends (its successor's memory would get it): the products,
        // then the last copy to each stage, waited for without a look at work->dead, a second each at most.
        if (scored > 0) bs::mbar_wait(s_full, (uint32_t)(scored - 1) & 1u, &work->dead, 1);
        if (weighed > 0) bs::mbar_wait(o_done, (uint32_t)(weighed - 1) & 1u, &work->dead, 1);
        if (tiles > 0 && !CAREFUL) bs::mbar_wait(q_full, 0, &work->dead, 1);
        for (int s = 0; s < kStages; ++s) {
            const int k = last_fill(min(max(scored - 1, 0) + kStages, tiles), s, kStages);
            const int v = last_fill(min(max(weighed - 1, 0) + kStages, tiles), s, kStages);
            if (k >= 0) bs::mbar_wait(k_full + s, (uint32_t)(k / kStages) & 1u, &work->dead, 1);
            if (v >= 0) bs::mbar_wait(v_full + s, (uint32_t)(v / kStages) & 1u, &work->dead, 1);
        }
        __syncwarp();
        if (CAREFUL) asm volatile("bar.arrive 1, %0;" ::"n"(kThreads) : "memory");  // work->odd is as it stays
    } else {
        // a thread's row: token r / group of the tile, query head r % group of the kv head
        const int r = threadIdx.x, tok = r / p.group, head = kvh * p.group + r % p.group, at = at0 + tok;
        const uint32_t lanes = (uint32_t)(warp * 32) << 16;
        const uint64_t scale2 = pair(p.scale_log2, p.scale_log2);
        constexpr float SHIFT = weight_shift(TYPE);  // O and l carry the weights' factor
        float m = -INFINITY, l = 0.0f;
        bool ok = true;  // after a wait that gave up the warp goes on to the end on what is there, and writes NaN
        for (int j = 0; j < tiles; ++j) {
            ok &= wait_warp(s_full, (uint32_t)j & 1u, work);
            tc_fence_after();
            const int key = lo + j * N, cols = j + 1 == tiles ? last_cols : N;
            float s[N];
            tmem_ld64(tmem + lanes + C::kS, s);  // columns behind the tile's last are masked
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(s_free);
            if (key + N - 1 > at0) {  // some row's keys end in this tile
                const int last = at - key;
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (i > last) s[i] = -INFINITY;
            }
            if (p.window > 0 && key < (SPLIT ? at0 + p.tile_tokens : hi) - p.window) {  // some row's window begins in it
                const int first = at - p.window + 1 - key;
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (i < first) s[i] = -INFINITY;
            }
            float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // chains short enough to overlap
#pragma unroll
            for (int i = 0; i < N; ++i) tops[i % 4] = max_nan(tops[i % 4], s[i]);
            const float top = max_nan(max_nan(tops[0], tops[1]), max_nan(tops[2], tops[3]));
            l = top < INFINITY ? l : NAN;  // a score of NaN or +inf, which not every form of 2^x passes on
            bool waited = j == 0;  // P and O are free once the products of the tile before are done
            if (__any_sync(0xffffffffu, (top - m) * p.scale_log2 > weight_lazy(TYPE))) {
                const float mm = fmaxf(m, top);
                if (j > 0) {
                    ok &= wait_warp(o_done, (uint32_t)(j - 1) & 1u, work);
                    waited = true;
                    tc_fence_after();
                    const float keep = mm == -INFINITY ? 1.0f : ex2((m - mm) * p.scale_log2);
                    l *= keep;
#pragma unroll
                    for (int c = 0; c < D; c += 16) {
                        float o[16];
                        bs::tmem_ld16(tmem + lanes + C::kO + c, o);
                        uint32_t u[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) u[i] = __float_as_uint(o[i] * keep);
                        tmem_st16(tmem + lanes + C::kO + c, u);
                    }
                }
                m = mm;
            }
            const float off = m == -INFINITY ? 0.0f : m * p.scale_log2 - SHIFT;
            const uint64_t off2 = pair(-off, -off);
            uint64_t sums[2] = {0, 0};
#pragma unroll
            for (int c = 0; c < N; c += 32) {
                if (c >= cols) continue;
                uint32_t u[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float2 x = unpair(fma2(pair(s[c + 2 * i], s[c + 2 * i + 1]), scale2, off2));
                    const float2 e = C::poly(i) ? ex2_poly(x) : make_float2(ex2(x.x), ex2(x.y));
                    sums[i % 2] = add2(sums[i % 2], pair(e.x, e.y));
                    u[i] = pack2<TYPE>(e.x, e.y);
                }
                if (!waited) {
                    ok &= wait_warp(o_done, (uint32_t)(j - 1) & 1u, work);
                    waited = true;
                    tc_fence_after();
                }
                tmem_st16(tmem_p + lanes + c / 2, u);
            }
            const float2 sum = unpair(add2(sums[0], sums[1]));
            l += sum.x + sum.y;
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full);
        }
        if (tiles > 0) ok &= wait_warp(o_done, (uint32_t)(tiles - 1) & 1u, work);
        tc_fence_after();
        if (CAREFUL) asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
        const bool mine = tok < work->tokens && r < p.tile_tokens * p.group;
        float worst = 0.0f;  // 0, or NaN
        // 32 elements of the row's sums
        auto row_of = [&](int c, float (&o)[32]) {
            __syncwarp();
            if (tiles > 0) {
                bs::tmem_ld32(tmem + lanes + C::kO + c, o);
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = 0.0f;
            }
            if (CAREFUL && mine && work->odd)
                add_odd<TYPE>(o, p.v.p + k0 * p.v.ts + kvh * p.v.hs + c * 2, p.v.ts,
                              p.window > 0 ? max(lo, at - p.window + 1) : lo, min(at + 1, hi),
                              shared_keys(p.window, at0, work->tokens));
#pragma unroll
            for (int i = 0; i < 32; ++i) worst += o[i] * 0.0f;
        };
        if (SPLIT && part >= 0) {  // the row's sums over this part, for the kernel that joins them
            float *sums = p.work + (int64_t)((tile - p.whole) * p.split + part) * (D + 2) * kRows + r;
            if (mine) {
                sums[D * kRows] = m == -INFINITY ? -INFINITY : m * p.scale_log2 - SHIFT;
                sums[(D + 1) * kRows] = l;
            }
#pragma unroll
            for (int c = 0; c < D; c += 32) {
                float o[32];
                row_of(c, o);
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (mine) sums[(c + i) * kRows] = ok ? o[i] : NAN;
            }
        } else {
            const bool none = m == -INFINITY && !isnan(l);  // the row saw nothing
            if (p.sinks && mine) l += sink_weight(p.sinks[head], m == -INFINITY ? 0.0f : m * p.scale_log2 - SHIFT);
            const float by = !ok ? NAN : none ? 0.0f : 1.0f / l;
            char *dst = p.out.p + (int64_t)(tok0 + tok) * p.out.ts + (int64_t)head * p.out.hs;
#pragma unroll
            for (int c = 0; c < D; c += 32) {
                float o[32];
                row_of(c, o);
                if (mine) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        float x[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = o[i + e] * by;
                        store8<TYPE>(dst + (c + i) * 2, x);
                    }
                }
            }
        }
        odd_row = mine && worst != 0.0f;
    }
    return odd_row;
}

// Out of the kernel's line, so that it costs it no registers; what it can find again it is not given, which would go
// through local memory.
template <int D, int TYPE, bool SPLIT>
__device__ __noinline__ void careful_pass(const PrefillParams &p, const CUtensorMap *tm_q, const CUtensorMap *tm_k,
                                          const CUtensorMap *tm_v) {
    tc_fence_after();
    Cta cta = this_cta<D, SPLIT>(p);
    find_tmem<D>(cta);
    tile_pass<D, TYPE, SPLIT, true>(p, tm_q, tm_k, tm_v, cta);
}

// SPLIT: the keys of tiles from p.whole on are split over p.split CTAs (windowed calls of many tiles, which a CTA's start bounds, took 4 %
// longer where one kernel did both).
template <int D, int TYPE, bool SPLIT>
__global__ void __launch_bounds__(kThreads, Cfg<D>::kCtas)
    prefill_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                   const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PrefillParams p) {
    using C = Cfg<D>;
    Cta cta = this_cta<D, SPLIT>(p);
    Work *work = cta.work;
    uint32_t *tmem_slot = cta.tmem_slot;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    // the work is found while the TMEM columns, the barriers and the tensor maps are made ready
    if (warp == 0) {
        const bool f = find_work<C::N>(p, cta.tile / p.kv_heads, cta.part, work);
        if (lane == 0) work->found = f;
    } else if (warp == 1) {
        if (lane == 0) init_bars(cta.bars);
    } else if (warp == kFeedWarp) {
        if (lane == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_q) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_k) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_v) : "memory");
        }
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "n"(C::kTmemCols)
                     : "memory");
        if (C::kTmemP)
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot + 1)),
                         "n"(C::kTmemP ? C::kTmemP : 32)
                         : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    find_tmem<D>(cta);
    auto leave = [&]() {
        if (warp != kFeedWarp) return;
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(cta.tmem), "n"(C::kTmemCols));
        if (C::kTmemP)
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(cta.tmem_p),
                         "n"(C::kTmemP ? C::kTmemP : 32));
    };
    if (SPLIT) cudaTriggerProgrammaticLaunchCompletion();  // lets the join take the places that fall free
    if (!work->found) {
        leave();
        return;
    }
    bool odd = tile_pass<D, TYPE, SPLIT, false>(p, &tm_q, &tm_k, &tm_v, cta);
    tc_fence_before();
    odd = __syncthreads_or(odd);
    if (odd && !work->dead) {
        if (threadIdx.x == 0) {  // every phase of the barriers is over, and they begin anew
            for (int i = 0; i < kBars; ++i)
                asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(smem_u32(cta.bars + i)) : "memory");
            init_bars(cta.bars);
        }
        __syncthreads();
        careful_pass<D, TYPE, SPLIT>(p, &tm_q, &tm_k, &tm_v);
        tc_fence_before();
        __syncthreads();
    }
    leave();
}

// The join of the parts' sums.  A CTA takes 32 rows of a tile, a lane a row, a warp eight of the row's elements: sums are
// read along the rows, as they were written, and a thread's loads do not wait for one another: two CTAs an SM are asked for
// so that the compiler takes registers for them (16 queries behind 32768 keys 41 us with 40 registers, 34 with 63).
constexpr int kJoinBlocks = kRows / 32, kJoinParts = 4;
template <int D, int TYPE>
__global__ void __launch_bounds__(D * 4, 2) prefill_join_kernel(const __grid_constant__ PrefillParams p) {
    __shared__ Work work;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int tile = p.whole + blockIdx.x / kJoinBlocks, kvh = tile % p.kv_heads;
    if (warp == 0) {
        const bool f = find_work<Cfg<D>::N>(p, tile / p.kv_heads, -1, &work);
        if (lane == 0) work.found = f;
    }
    __syncthreads();
    // Launched while the partial sums are still being made.  CTAs without work wait as well: what follows on the stream waits
    // for this grid only, which must not end before the other.
    cudaGridDependencySynchronize();
    if (!work.found) return;
    const int r = blockIdx.x % kJoinBlocks * 32 + lane, tok = r / p.group, head = kvh * p.group + r % p.group;
    if (r >= work.tokens * p.group) return;
    const int64_t step = (D + 2) * kRows;
    const float *sums = p.work + (tile - p.whole) * p.split * step + r;
    float top = -INFINITY;
#pragma unroll 8
    for (int i = 0; i < p.split; ++i) top = fmaxf(top, sums[i * step + D * kRows]);
    const float z = top == -INFINITY ? 0.0f : top;
    float l = 0.0f, o[8] = {};
    for (int i0 = 0; i0 < p.split; i0 += kJoinParts) {
        // the loads of some parts are all on their way before the first is used; no branch, behind which they would sink
        float by[kJoinParts], x[kJoinParts][9];
#pragma unroll
        for (int i = 0; i < kJoinParts; ++i) {
            const bool on = i0 + i < p.split;
            const float *part = sums + (on ? i0 + i : 0) * step;
            by[i] = part[D * kRows], x[i][8] = part[(D + 1) * kRows];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[i][e] = part[(warp * 8 + e) * kRows];
            by[i] = on ? ex2(by[i] - z) : 0.0f;
#pragma unroll
            for (int e = 0; e < 9; ++e) x[i][e] = on ? x[i][e] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < kJoinParts; ++i) {
            l += by[i] * x[i][8];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] += by[i] * x[i][e];
        }
    }
    const bool none = top == -INFINITY && !isnan(l);
    if (p.sinks) l += sink_weight(p.sinks[head], z);
    const float by = none ? 0.0f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] *= by;
    store8<TYPE>(p.out.p + (int64_t)(work.tok0 + tok) * p.out.ts + (int64_t)head * p.out.hs + warp * 16, o);
}

// [tokens][heads][D] rows as a 3-D map with boxes of 64 elements x heads x tokens.
bool encode_rows(CUtensorMap *tm, const amoe_rows *r, int D, int tokens, int box_heads, int box_tokens) {
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)r->heads, (cuuint64_t)(tokens > 0 ? tokens : 1)};
    // the stride of a dimension of one is never used, but has to be a valid one
    const cuuint64_t strides[2] = {(cuuint64_t)(r->heads > 1 ? r->head_stride * 2 : D * 2),
                                   (cuuint64_t)(tokens > 1 ? r->token_stride * 2 : D * 2)};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens}, es[3] = {1, 1, 1};
    return bs::encode_fn()(tm, r->type == AMOE_GGUF_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                        : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                           3, r->data, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int kMaxDevices = 64;
constexpr int kSms = 148;
constexpr int kMaxTokens = 1 << 30;  // row indexes and positions stay far inside 32 bits

template <int D, int TYPE>
cudaError_t launch(const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v, const PrefillParams &p, int device,
                   dim3 grid, cudaStream_t st) {
    auto *kernel = p.split > 1 ? prefill_kernel<D, TYPE, true> : prefill_kernel<D, TYPE, false>;
    static std::atomic<bool> done[2][kMaxDevices];
    std::atomic<bool> *ready = done[p.split > 1];
    if (!ready[device].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kSmem);
        if (e != cudaSuccess) return e;
        ready[device].store(true, std::memory_order_release);
    }
    kernel<<<grid, kThreads, Cfg<D>::kSmem, st>>>(q, k, v, p);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || p.split == 1) return e;
    cudaLaunchConfig_t join{};
    join.gridDim = dim3((grid.x - p.whole) / p.split * kJoinBlocks);
    join.blockDim = dim3(D * 4);
    join.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    join.attrs = attr;
    join.numAttrs = 1;
    return cudaLaunchKernelEx(&join, prefill_join_kernel<D, TYPE>, p);
}

// How a call is laid out: row tiles of all kv heads, how many of them one CTA takes, CTAs to the keys of each of the
// others, and the workspace of more than one.
struct Layout {
    int64_t tiles, whole;
    int split;
    int64_t bytes;
};

// The tiles behind the last whole wave of CTAs (all, where they fill none) leave SMs idle, and their keys are then
// split.  The split is the one of the least expected time: a CTA takes 1 us for 64 keys however many share its SM, and
// 4 us to start and end; the join takes 3 us, 1/4 us a part that its threads walk, and the partial sums' way through
// L2 15 ns (64-wide heads) or 30 ns a CTA.  Measured, one CTA a tile -> split (64/8 heads of 64): 16 queries behind
// 2048 keys 29 -> 12 us in 8 parts (14.4 in 16), behind 32768 460 -> 34 us in 32; 512 behind 8192 129 -> 122 us in 3;
// 128 behind none 6.0 us, in 2 parts 8.9.  32/8 heads of 128: 64 behind 8192 134 -> 26 us; 300 behind 3000 55 -> 32 us
// in 3 (39 in 4); 1500 behind 8000 (296 whole tiles, 80 split) 256 -> 206 us in 3 (216 in 4; all tiles in 3: 233); 1400
// behind none 27.5 us, its last tiles in 2 parts 33.
constexpr int kMaxSplit = 32;
Layout layout(int head_dim, int window, int64_t q_tokens, int64_t k_tokens, int64_t seqs, int q_heads, int kv_heads) {
    const int tile_tokens = kRows / (q_heads / kv_heads);
    // every sequence's last tile may hold a single token
    const int64_t tiles = (q_tokens + std::min(seqs, q_tokens) * (tile_tokens - 1)) / tile_tokens * kv_heads;
    const int64_t slots = kSms * (head_dim == 64 ? Cfg<64>::kCtas : Cfg<128>::kCtas);
    const int64_t whole = tiles / slots * slots, rest = tiles - whole;
    Layout l{tiles, tiles, 1, 0};
    if (rest == 0) return l;  // whole waves (or no rows): nothing to split
    // The host knows no sequence's own length and takes them as equal.  A sequence's first tokens come last and
    // see the fewest keys.
    const int64_t most = window > 0 ? (int64_t)window + tile_tokens : INT_MAX, keys = k_tokens / seqs;
    const int64_t before = std::max<int64_t>(keys - q_tokens / seqs, 0);
    const int64_t steps = (std::min(keys, most) + 63) / 64;
    const int64_t last = (std::min({keys, most, before + (rest + kv_heads - 1) / kv_heads * tile_tokens}) + 63) / 64;
    const float full = (float)(whole / slots * (steps + 4));
    float best = 0.95f * (full + last + 4);  // a split has to gain something
    // no more than four waves of parts: the partial sums (34 or 67 KB a CTA) stay in L2
    for (int64_t s = 2; s <= kMaxSplit && s <= last && rest * s <= 4 * slots; ++s) {
        const float us = full + (rest * s + slots - 1) / slots * ((last + s - 1) / s + 4) + 3.0f + 0.25f * s +
                         (head_dim == 64 ? 0.015f : 0.03f) * (rest * s);
        if (us < best) best = us, l.whole = whole, l.split = (int)s;
    }
    if (l.split > 1) l.bytes = rest * l.split * kRows * (head_dim + 2) * 4;
    return l;
}

}  // namespace
}  // namespace attn
}  // namespace amoe

using namespace amoe;
using namespace amoe::attn;

extern "C" {

int64_t amoe_attn_prefill_workspace(int32_t head_dim, int32_t window, int32_t q_heads, int32_t kv_heads,
                                    int32_t q_tokens, int32_t k_tokens, int32_t seqs) {
    if (int rc = check_head_dim(head_dim)) return rc;
    if (int rc = check_group(q_heads, kv_heads)) return rc;
    if (window < 0 || q_tokens < 0 || k_tokens < 0 || seqs < 1)
        return reject("window, q_tokens and k_tokens must not be negative, seqs must be positive");
    return layout(head_dim, window, q_tokens, k_tokens, seqs, q_heads, kv_heads).bytes;
}

int amoe_attn_prefill(int32_t device, int32_t head_dim, const amoe_attn *attn, const amoe_rows *q, const amoe_rows *k,
                      const amoe_rows *v, const amoe_rows *out, int32_t q_tokens, int32_t k_tokens,
                      const int32_t *cu_q, const int32_t *cu_k, int32_t seqs, void *workspace,
                      int64_t workspace_bytes, void *stream) {
    if (int rc = check_attn(attn)) return rc;
    if (int rc = check_head_dim(head_dim)) return rc;
    if (q_tokens < 0 || k_tokens < 0) return reject("q_tokens and k_tokens must not be negative");
    if (q_tokens > kMaxTokens || k_tokens > kMaxTokens) return reject("more than 2^30 rows in one prefill call");
    if (int rc = check_rows(q, "q", head_dim, 0, q_tokens, -1)) return rc;
    if (q->type != AMOE_GGUF_F16 && q->type != AMOE_GGUF_BF16) return reject("prefill takes F16 or BF16 rows");
    if (int rc = check_rows(k, "k", head_dim, 0, k_tokens, q->type)) return rc;
    if (int rc = check_rows(v, "v", head_dim, k->heads, k_tokens, q->type)) return rc;
    if (int rc = check_rows(out, "out", head_dim, q->heads, q_tokens, q->type)) return rc;
    if (int rc = check_group(q->heads, k->heads)) return rc;
    if (!cu_q || !cu_k) return reject("cu_q and cu_k must not be NULL");
    if (seqs < 1) return reject("seqs must be positive");
    if (device < 0 || device >= kMaxDevices) return reject("device ordinal out of range");
    if (q_tokens == 0) return AMOE_OK;
    PrefillParams p{};
    p.v = rows_dev(v), p.out = rows_dev(out);
    p.cu_q = cu_q, p.cu_k = cu_k;
    p.sinks = attn->sinks;
    p.scale_log2 = attn_scale(attn, head_dim) * kLog2e;
    // a window as long as the keys hides none
    p.window = attn->window < k_tokens ? attn->window : 0, p.q_tokens = q_tokens, p.k_tokens = k_tokens, p.seqs = seqs;
    p.group = q->heads / k->heads;
    p.tile_tokens = kRows / p.group;
    p.kv_heads = k->heads;
    const Layout l = layout(head_dim, attn->window, q_tokens, k_tokens, seqs, q->heads, k->heads);
    if (l.tiles > INT_MAX / 2) return reject("too many query rows");
    if (l.split > 1 && (!workspace || workspace_bytes < l.bytes))
        return reject("prefill needs a workspace of " + std::to_string(l.bytes) + " bytes");
    if (l.split > 1 && (reinterpret_cast<uintptr_t>(workspace) & 15))
        return reject("workspace must be 16-byte aligned");
    p.whole = (int)l.whole, p.split = l.split, p.work = static_cast<float *>(workspace);
    DeviceScope scope;
    cudaError_t e = scope.enter(device);
    if (e != cudaSuccess) return cuda_error(e, "cudaSetDevice");
    if (!bs::get_encode()) {
        set_thread_error("cuTensorMapEncodeTiled is not available");
        return AMOE_ERR_CUDA;
    }
    const int n = head_dim == 64 ? Cfg<64>::N : Cfg<128>::N;
    CUtensorMap tq, tk, tv;
    if (!encode_rows(&tq, q, head_dim, q_tokens, p.group, p.tile_tokens) ||
        !encode_rows(&tk, k, head_dim, k_tokens, 1, n) || !encode_rows(&tv, v, head_dim, k_tokens, 1, n))
        return reject("prefill: strides of q, k or v that a tensor map cannot take");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // kv heads first, then a sequence's tiles from the longest down; a split tile's parts before those
    const dim3 grid((unsigned)(l.whole + (l.tiles - l.whole) * l.split));
    if (head_dim == 64)
        e = q->type == AMOE_GGUF_F16 ? launch<64, AMOE_GGUF_F16>(tq, tk, tv, p, device, grid, st)
                                     : launch<64, AMOE_GGUF_BF16>(tq, tk, tv, p, device, grid, st);
    else
        e = q->type == AMOE_GGUF_F16 ? launch<128, AMOE_GGUF_F16>(tq, tk, tv, p, device, grid, st)
                                     : launch<128, AMOE_GGUF_BF16>(tq, tk, tv, p, device, grid, st);
    return e == cudaSuccess ? AMOE_OK : cuda_error(e, "prefill kernel");
}

}  // extern "C"
