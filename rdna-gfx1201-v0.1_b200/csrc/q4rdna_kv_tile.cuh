// Attention over the 8-bit cache, many columns per sequence: prompts and pieces of
// prompts (q4rdna_kv_attention), on the 5th-generation tensor cores.
//
// A task (q4rdna_kv_split.cuh) is 256 columns as two tiles of 128 rows; its pieces are
// steps of 128 tokens.  Bound by the tensor cores and the exponentials alike: a step
// takes 2 x (128 x 128 x D) x 2 products (2048 cycles at D = 128) and 2 x 128 x 128
// exponentials (2048 cycles at 16 a cycle).
//   * One persistent CTA per SM, 16 warps (128 registers; a 17th would leave 96):
//       warps 0-3, 4-7   softmax of tile 0 and tile 1, one row per thread;
//       warps 8-14       read the cache's 8-bit tiles, write K and V as f16;
//       warp 15          one thread issues the products.
//   * S = Q K^T: tcgen05.mma kind::f16, M = 128, N = 128, f32 in tensor memory; Q and
//     the codes of K (exact in f16) in shared memory, K-major with 128-byte swizzle.
//   * O += P V: P in f16 as the A operand in tensor memory, over the first half of S's
//     columns; V as it lies (dims contiguous: the MN-major B operand), 128-byte
//     swizzle.  O stays in tensor memory over a task.
//   * While one tile's softmax runs, the other tile's products do.
//   * Scales: a block's key scale multiplies its 16 columns of S, the logarithm of its
//     value scale joins the exponent, p = 2^(s + log2 sv - R); the sum of the weights
//     themselves takes each block's sum times 1 / sv.  R, per row, moves only when the
//     weights would leave f16's range (the row's O is then rescaled by its own thread),
//     and p carries 2^7.
//   * Tensor memory (512 columns): S0 S1 O0 O1, 128 each.
//   * P rounded to f16 (2^-12) and O in the tensor core's running sum, which truncates (2^-17 over a task): for 16-bit
//     rows only, whose own rounding is 2^-9 or 2^-12; against 64 bits a prompt of 1900 in f16 is off by 2.7e-4
//     (2.1e-4 with weights in f32, the rest is the output's rounding), bf16 by 1.67e-3 (1.66e-3).
// Measured (device time with the join): 2048 tokens behind 8191 others, 32 query and 8 kv
// heads of 128, e4m3, bf16 426 us, 0.44 of the products' time at 1650 TFLOP/s; three
// prompts of up to 1900, 16 and 4 heads of 64, window 1000, f16 89 us.  Work left out in turn, when the first took 460 us: 354 without
// the loading warps' conversion, 308 without the exponentials too, 300 with the products
// and the waits alone.  So no unit is full: what bounds it are the waits between the
// roles, the softmax's latency (about 3000 cycles a tile and step) above all.
// Every wait is bounded (about a second, %globaltimer): on expiry the role sets bit 4
// of the fault word and takes no more waits, copies or products; the issuing thread
// still waits (bounded) for its products before the tensor memory is freed.
#pragma once

#include <climits>

#include "q4rdna_kv_split.cuh"

namespace q4kv {

constexpr int kTileWarps = 16, kTileLoadWarps = 7, kTileMmaWarp = 15;
constexpr int kTileThreads = 32 * kTileWarps;
constexpr int kTileRows = 128, kTileTokens = 128, kTileCols = 256, kTileShift = 7;
constexpr int kTileLoaders = 32 * kTileLoadWarps;
constexpr int kTileAhead = 7;  // pieces of a loading thread in flight: what shared memory holds
constexpr unsigned kFaultTile = 16u;
constexpr uint64_t kTileWaitNs = 1000000000ull;

template <int D>
struct TileSmem {
    static constexpr int PANEL = kTileTokens * 128;       // 128 rows of 64 f16, swizzled
    static constexpr int STAGE = PANEL * (D / 64);        // a K or V stage, or a tile's Q
    uint8_t q[2][STAGE];
    uint8_t k[2][STAGE];
    uint8_t v[2][STAGE];
    uint8_t ring[kTileAhead * kTileLoaders * 16];  // pieces of the loading threads on their way
    float4 scale[4][8];  // per block of a step: key scale, log2 and inverse of the value scale; .w of the first and the
                         // second: the largest and smallest inverse of the step
    float qscale[2][kTileRows];
    float turn[4][kTileRows], sum[kTileRows * 4], ref[kTileRows * 4];  // f32 rows: O's factor, sum and reference (rings of 4 steps)
    uint64_t bar[28];
    ShareSmem<kTileWarps> share;
    uint32_t tmem;
};

static_assert(sizeof(TileSmem<128>) <= 232448, "shared memory of the tile kernels");

// ------------------------------------------------------------ PTX

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __noinline__ bool bar_wait_slow(uint32_t bar, uint32_t parity) {
    uint64_t t0, t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
    for (uint32_t n = 1;; ++n) {
        if (bar_try(bar, parity)) return true;
        if ((n & 63u) == 0) {
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
            if (t - t0 > kTileWaitNs) return false;
        }
    }
}
// Whether three phases are there, asked for at once (one barrier's answer takes about 100 cycles)
__device__ __forceinline__ bool bar_try3(uint32_t b0, uint32_t p0, uint32_t b1, uint32_t p1, uint32_t b2, uint32_t p2) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p, q, r;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        " mbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4;\n mbarrier.try_wait.parity.shared::cta.b64 r, [%5], %6;\n"
        " and.pred p, p, q;\n and.pred p, p, r;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(b0), "r"(p0), "r"(b1), "r"(p1), "r"(b2), "r"(p2)
        : "memory");
    return ok != 0;
}
// Waits for the phase of the given parity; `ok` false: not any more
__device__ __forceinline__ void bar_wait(uint32_t bar, uint32_t parity, bool &ok) {
    if (ok && !bar_try(bar, parity)) {
        ok = bar_wait_slow(bar, parity);
        if (!ok) atomicOr(&g_kv_fault, kFaultTile);
    }
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Shared-memory operand, 128-byte swizzle: stride 1024 between groups of 8 rows;
// `lead` between panels of 64 elements (MN-major only)
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((lead >> 4) & 0x3FFFu) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(add)
        : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];\n"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(addr));
}
// Waits for the loads; the registers are named, so that nothing that reads them comes first
__device__ __forceinline__ void tmem_arrived(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]),
                   "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]),
                   "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]),
                   "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]),
                   "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31]));
}
__device__ __forceinline__ void tmem_arrived(uint32_t (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]),
                   "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]),
                   "+r"(v[14]), "+r"(v[15]));
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
        "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(v[0]),
        "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]),
        "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
        "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(addr)
        : "memory");
}

// Byte of element (row, chunk of 8) of a swizzled operand of 64-element panels
__device__ __forceinline__ uint32_t swizzled(int row, int chunk) {
    return (uint32_t)((chunk >> 3) * (kTileTokens * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

// ------------------------------------------------------------ softmax

struct RowState {
    float R, l;    // reference of the exponents, sum of the weights
    float scale;   // of the row's scores
    int lo, hi;    // tokens that the row sees: [lo, hi]
};

// Where a softmax warp works and what it waits for
struct RowPlace {
    uint32_t s_at, o_at;                // tensor memory of the warp's rows
    uint32_t s_full, p_full, sc_full;   // mbarriers (sc_full: the first of four)
    uint32_t steps, it, parity;         // of the task; steps before it, of the CTA and (parity of S) of the tile
    int tok0, all_lo, all_hi;           // first token of the task; tokens that all rows of the warp see
};

// A step's weights without the logarithms of the value scales.  The sums by blocks lose those of a block whose values
// are 2^100 times smaller than the ones that set the reference: they fall below f32's numbers before 1 / sv brings
// them back (the products may lose them, the sum must not).
__device__ __noinline__ float weights_alone(float by, float ref, int lo, int hi, const float4 *scale, uint32_t s_at, int tok0) {
    float add = 0.0f;
#pragma unroll 1
    for (int b = 0; b < 8; ++b) {
        uint32_t v[16];
        tmem_load16(s_at + 16 * b, v);
        tmem_arrived(v);
        const float4 g = scale[b];
        const float a = g.x * by;
        const int tok = tok0 + 16 * b;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            sum += tok + i < lo || tok + i > hi ? 0.0f : ex2(fmaf(__uint_as_float(v[i]), a, -ref));
        if (g.y != -INFINITY) add += sum;  // (a page outside the cache)
    }
    return add;
}

// One step of one row: S to P in one pass over S with the reference as it stands: p is
// right for any reference, as long as it stays in f16's range, and no weight is above
// the sum of its block.  Where a sum is above 2^15 (or the row has seen nothing yet) the
// step's largest exponent is looked for, becomes the reference, and the pass is made
// again; P goes to tensor memory (over S) only when it is right.  `alone`: once more, with
// the sum of weights_alone.
// Tokens that a row of the warp does not see lie outside [all_lo, all_hi]; only the
// blocks there pay for the mask.
template <int D>
__device__ __forceinline__ void softmax_step(RowState &r, const float4 *scale, uint32_t s_at, uint32_t o_at, int tok0,
                                             int all_lo, int all_hi, bool first) {
    uint32_t p[64];
    float add, exact = 0.0f;
    bool look = first, alone = false;
#pragma unroll 1
    while (true) {
        if (look) {
            uint32_t v[32];
            float t = -INFINITY;  // the largest exponent
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
                tmem_load32(s_at + 32 * c, v);
                tmem_arrived(v);
                const int tok = tok0 + 32 * c;
                if (tok < all_lo || tok + 31 > all_hi) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (tok + i < r.lo || tok + i > r.hi) v[i] = 0xff800000u;  // -inf
                }
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const float4 f = scale[2 * c + b];
                    float m = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 16; ++i) m = fmaxf(m, __uint_as_float(v[16 * b + i]));
                    // a block without a visible token has m = -inf, which a scale of 0 would turn into NaN
                    if (m != -INFINITY) t = fmaxf(t, fmaf(m, f.x * r.scale, f.y));
                }
            }
            const float f = t > r.R ? ex2(r.R - t) : 1.0f;  // 0 for the first: R = -inf
            if (t > r.R) {
                r.l = shrunk(r.l, r.R - t);
                r.R = t;
            }
            if (!first) {
                // the products of the step before have ended (they come before this S), the next ones wait for this P
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    tmem_load32(o_at + c, v);
                    tmem_arrived(v);
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
                    tmem_store32(o_at + c, v);
                }
            }
            if (alone) exact = weights_alone(r.scale, (r.R == -INFINITY ? 0.0f : r.R) - 7.0f, r.lo, r.hi, scale, s_at, tok0);
        }
        const float ref = (r.R == -INFINITY ? 0.0f : r.R) - 7.0f;
        uint32_t v[2][16];
        float e[2][16];
        tmem_load16(s_at, v[0]);
        add = 0.0f;
        float most = 0.0f;
        // the weights of a block in flight while the block before it is summed and packed
#pragma unroll
        for (int b = 0; b < 9; ++b) {
            if (b < 8) {
                tmem_arrived(v[b & 1]);
                if (b < 7) tmem_load16(s_at + 16 * (b + 1), v[(b + 1) & 1]);
                const float4 g = scale[b];
                const float a = g.x * r.scale, d = g.y - ref;
                const F2 a2 = pack2(a, a), d2 = pack2(d, d);
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const float2 x =
                        both(fma2(pack2(__uint_as_float(v[b & 1][i]), __uint_as_float(v[b & 1][i + 1])), a2, d2));
                    e[b & 1][i] = x.x;
                    e[b & 1][i + 1] = x.y;
                }
                const int tok = tok0 + 16 * b;
                if (tok < all_lo || tok + 15 > all_hi) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (tok + i < r.lo || tok + i > r.hi) e[b & 1][i] = -INFINITY;
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) e[b & 1][i] = ex2(e[b & 1][i]);
            }
            if (b > 0) {
                const float(&y)[16] = e[(b - 1) & 1];
                F2 sum[2] = {pack2(y[0], y[1]), pack2(y[2], y[3])};
#pragma unroll
                for (int i = 4; i < 16; i += 4) {
                    sum[0] = add2(sum[0], pack2(y[i], y[i + 1]));
                    sum[1] = add2(sum[1], pack2(y[i + 2], y[i + 3]));
                }
#pragma unroll
                for (int i = 0; i < 16; i += 2) p[8 * (b - 1) + i / 2] = pack_half(y[i], y[i + 1]);
                const float2 two = both(add2(sum[0], sum[1]));
                const float one = two.x + two.y;
                most = fmaxf(most, one);
                // a block without a visible token takes nothing from its scale, be it NaN
                if (one != 0.0f) add = fmaf(one, scale[b - 1].z, add);
            }
        }
        if (alone) {
            add = exact;
            break;
        }
        // The largest weight that may have fallen below 2^-126 in a block, against the sum
        alone = __any_sync(0xffffffffu, r.R != -INFINITY && scale[0].w * 0x1p-92f > r.l + add);
        if (look && !alone) break;  // every exponent is now at most the reference
        look = alone || __any_sync(0xffffffffu, most > 32768.0f || r.R == -INFINITY);
        if (!look) break;
    }
    r.l += add;
    tmem_store32(s_at, *reinterpret_cast<uint32_t(*)[32]>(p));
    tmem_store32(s_at + 32, *reinterpret_cast<uint32_t(*)[32]>(p + 32));
    tmem_wait_store();
}

// The steps of a task for a warp's 32 rows.  Not inlined: the state of the walk over
// the tasks would take the registers that S needs.
template <int D>
__device__ __noinline__ bool softmax_rows(RowState &row, const RowPlace &at, const float4 (*scale)[8], bool ok) {
    RowState r = row;
    const RowPlace a = at;
#pragma unroll 1
    for (uint32_t j = 0; j < a.steps; ++j) {
        const uint32_t n = a.it + j;
        bar_wait(a.s_full, (a.parity + j) & 1, ok);
        bar_wait(a.sc_full + 8 * (n & 3), (n >> 2) & 1, ok);  // at most one phase ahead once S is there
        fence_after();
        const int tok0 = a.tok0 + (int)j * kTileTokens;
        softmax_step<D>(r, scale[n & 3], a.s_at, a.o_at, tok0, a.all_lo, a.all_hi, j == 0);
        fence_before();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) bar_arrive(a.p_full);
    }
    row = r;
    return ok;
}

// ------------------------------------------------------------ loading

struct LoadPlace {
    uint8_t *k, *v;                              // two stages each
    uint8_t *ring;
    float4 (*scale)[8];
    uint32_t k_full, k_empty, v_full, v_empty, sc_full;
    uint32_t steps, it;
    int begin, s, h, lo, hi, len;                // first step; sequence, head, its visible 16-token blocks and length
};

// K and V of a task's steps, from 8-bit tiles to f16 operands (the loading warps).  A
// thread's pieces are 16 codes of a token, N of K and then N of V in every step; they
// come through a ring of its own in shared memory, kTileAhead pieces ahead (HBM takes
// about 1500 cycles to answer, a step's conversion 2500).  8 lanes of a store are 4
// pieces of 2 tokens: all banks once.
template <int D, int FMT>
__device__ __noinline__ bool load_steps(const AttnArgs &A, const LoadPlace &place, bool ok) {
    const LoadPlace P = place;
    const int u = threadIdx.x - 32 * (kTileMmaWarp - kTileLoadWarps), lane = threadIdx.x & 31;
    constexpr int PIECES = D / 16;
    constexpr int STEP = kTileLoaders / PIECES;         // tokens from piece to piece of a thread: 28 or 56
    constexpr int N = (kTileTokens + STEP - 1) / STEP;  // pieces of a thread, K or V of a step
    constexpr int STAGE = TileSmem<D>::STAGE;
    constexpr int SLOT = kTileLoaders * 16;
    const int ch = D == 128 ? (lane & 3) | (lane >> 1 & 4) : lane & 3;
    const int tk = D == 128 ? 4 * (u >> 5) + (lane >> 2 & 1) + (lane >> 3 & 2) : u >> 2;
    const uint32_t to = swizzled(tk, 2 * ch);
    const uint32_t from = kHeader + (tk & 3) * D + 16 * ch;
    const uint32_t ring = smem_u32(P.ring) + 16 * u;
    const uint8_t *const ring_at = P.ring + 16 * u;
    // lane i < 8: the tile of block i of steps j, j + 1 and j + 2, or 0: zeros
    unsigned long long tile0 = 0, tile1 = 0, tile2 = 0;
    auto find = [&](int j) -> unsigned long long {
        const int blk = (P.begin + j) * 8 + (lane & 7);
        return j < (int)P.steps && blk >= P.lo && blk < P.hi ? (unsigned long long)tile_of(A.c, A.b, P.s, P.h, blk) : 0ull;
    };
    // Piece i of half z of step j + ahead.  A row that holds no token yet may hold NaN, which
    // a weight of 0 would keep: zeros there, too.
    int put_slot = 0, get_slot = 0;
    auto issue = [&](int j, int ahead, int z, int i) {
        const int t = tk + i * STEP;
        const unsigned long long p =
            __shfl_sync(0xffffffffu, ahead == 0 ? tile0 : ahead == 1 ? tile1 : tile2, (t >> 4) & 7);
        const bool there = p != 0 && t + (P.begin + j + ahead) * kTileTokens < P.len && (i + 1 < N || t < kTileTokens);
        const unsigned long long src =
            there ? p + from + (z * kBlock + (t & 15) - (tk & 3)) * D : (unsigned long long)A.c.tiles;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ring + put_slot), "l"(src), "r"(there ? 16 : 0)
                     : "memory");
        asm volatile("cp.async.commit_group;" ::: "memory");
        put_slot = put_slot == (kTileAhead - 1) * SLOT ? 0 : put_slot + SLOT;
    };
    auto take = [&]() -> uint4 {
        asm volatile("cp.async.wait_group %0;" ::"n"(kTileAhead - 2) : "memory");
        const uint4 r = *reinterpret_cast<const uint4 *>(ring_at + get_slot);
        get_slot = get_slot == (kTileAhead - 1) * SLOT ? 0 : get_slot + SLOT;
        return r;
    };
    auto put = [&](uint8_t *stage, int i, const uint4 &r) {
        const uint32_t wd[4] = {r.x, r.y, r.z, r.w};
        uint32_t h[8];
#pragma unroll
        for (int z = 0; z < 4; ++z) {
            const uint32_t y = FMT == Q4RDNA_KV_INT8 ? wd[z] ^ 0x80808080u : wd[z];
            h[2 * z] = pair_of<FMT, 0>(y);
            h[2 * z + 1] = pair_of<FMT, 2>(y);
        }
        if (i + 1 < N || tk + i * STEP < kTileTokens) {
            // the swizzle of token tk + i STEP: STEP is a multiple of 4
            const uint32_t at = (to ^ ((i * STEP & 4) << 4)) + i * STEP * 128;
            *reinterpret_cast<uint4 *>(stage + at) = make_uint4(h[0], h[1], h[2], h[3]);
            *reinterpret_cast<uint4 *>(stage + (at ^ 16)) = make_uint4(h[4], h[5], h[6], h[7]);
        }
    };
    tile0 = find(0);
    tile1 = find(1);
    float2 head = u < 8 && tile0 != 0 ? *reinterpret_cast<const float2 *>(tile0) : make_float2(0.0f, 0.0f);
#pragma unroll
    for (int a = 0; a < kTileAhead; ++a) issue(0, a / (2 * N), a / N % 2, a % N);
#pragma unroll 1
    for (uint32_t j = 0; j < P.steps; ++j) {
        const uint32_t n = P.it + j, stage = n & 1, parity = ((n >> 1) & 1) ^ 1;
        tile2 = find(j + 2);
        const float2 next_head = u < 8 && tile1 != 0 ? *reinterpret_cast<const float2 *>(tile1) : make_float2(0.0f, 0.0f);
        uint4 r = take();
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            bar_wait((z == 0 ? P.k_empty : P.v_empty) + 8 * stage, parity, ok);
            uint8_t *const to_stage = (z == 0 ? P.k : P.v) + stage * STAGE;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                constexpr int A0 = kTileAhead;
                const int a = z * N + i + A0;
                const uint4 now = r;
                if (z == 0 || i + 1 < N) r = take();
                put(to_stage, i, now);
                issue(j, a / (2 * N), a / N % 2, a % N);  // into the slot that `now` came from
            }
            fence_async();
            __syncwarp();
            if (lane == 0) bar_arrive((z == 0 ? P.k_full : P.v_full) + 8 * stage);
            if (z == 0 && u < 32) {
                const float sv = head.y <= kTinyScale ? kTinyScale : head.y;  // NaN stays
                const float inv = tile0 != 0 ? 1.0f / sv : 0.0f;
                float ends = u == 1 ? -INFINITY : 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {  // lane 0 the largest, lane 1 the smallest, negative
                    const float x = __shfl_sync(0xffffffffu, inv, i);
                    if (x > 0.0f) ends = fmaxf(ends, u == 1 ? -x : x);
                }
                if (u == 1) ends = -ends;
                // a block on a page outside the cache takes no weight, as if it were masked
                if (u < 8)
                    P.scale[n & 3][u] = tile0 != 0 ? make_float4(head.x, log2f(sv), inv, ends)
                                                   : make_float4(0.0f, -INFINITY, 0.0f, ends);
                __syncwarp();
                if (lane == 0) bar_arrive(P.sc_full + 8 * (n & 3));
            }
        }
        tile0 = tile1;
        tile1 = tile2;
        head = next_head;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    return ok;
}

// ------------------------------------------------------------ products

__device__ __forceinline__ bool elected() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
}

// Barriers of the CTA: K and V stage full / empty, scales (ring of 4), and per tile Q
// written, S computed, P written, O complete
struct Bars {
    uint32_t at;
    __device__ __forceinline__ uint32_t k_full(int i) const { return at + 8u * i; }
    __device__ __forceinline__ uint32_t k_empty(int i) const { return at + 8u * (2 + i); }
    __device__ __forceinline__ uint32_t v_full(int i) const { return at + 8u * (4 + i); }
    __device__ __forceinline__ uint32_t v_empty(int i) const { return at + 8u * (6 + i); }
    __device__ __forceinline__ uint32_t sc_full(int i) const { return at + 8u * (8 + i); }
    __device__ __forceinline__ uint32_t q_full(int x) const { return at + 8u * (12 + x); }
    __device__ __forceinline__ uint32_t s_full(int x) const { return at + 8u * (14 + x); }
    __device__ __forceinline__ uint32_t p_full(int x) const { return at + 8u * (16 + x); }
    __device__ __forceinline__ uint32_t o_full(int x) const { return at + 8u * (18 + x); }
    __device__ __forceinline__ uint32_t drained() const { return at + 8u * 20; }
    // f32 rows: the step's O read, and O's factor written (ring of 4)
    __device__ __forceinline__ uint32_t o_free() const { return at + 8u * 21; }
    __device__ __forceinline__ uint32_t turned(int i) const { return at + 8u * (22 + i); }
};

// Tensor memory and barriers at the kernel's begin and end
template <int D>
__device__ __forceinline__ uint32_t tile_enter(TileSmem<D> &sm, Bars bar) {
    if ((threadIdx.x >> 5) == kTileMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            bar_init(bar.k_full(i), kTileLoadWarps);
            bar_init(bar.v_full(i), kTileLoadWarps);
            bar_init(bar.k_empty(i), 1);
            bar_init(bar.v_empty(i), 1);
            bar_init(bar.q_full(i), 4);
            bar_init(bar.s_full(i), 1);
            bar_init(bar.p_full(i), 4);
            bar_init(bar.o_full(i), 1);
        }
        for (int i = 0; i < 4; ++i) {
            bar_init(bar.sc_full(i), 1);
            bar_init(bar.turned(i), 4);
        }
        bar_init(bar.o_free(), 4);
        bar_init(bar.drained(), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    return sm.tmem;
}
__device__ __forceinline__ void tile_leave(uint32_t tmem, Bars bar) {
    const bool mine = (threadIdx.x >> 5) == kTileMmaWarp;
    if (mine) {  // no product may still run when the tensor memory goes
        bool last = true;
        if (elected()) commit(bar.drained());
        __syncwarp();
        bar_wait(bar.drained(), 0, last);
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (mine) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// The loading warps' part of a task
template <int D, int FMT>
__device__ __forceinline__ bool load_task(const AttnArgs &A, TileSmem<D> &sm, Bars bar, const Walk &W, int nc, int steps,
                                          uint32_t it, bool ok) {
    // 16-token blocks that a column of the task sees
    const Span sp = span_of(W.q, W.col0, nc, A.group, A.window, 4);
    LoadPlace p;
    p.k = sm.k[0];
    p.v = sm.v[0];
    p.ring = sm.ring;
    p.scale = sm.scale;
    p.k_full = bar.k_full(0);
    p.k_empty = bar.k_empty(0);
    p.v_full = bar.v_full(0);
    p.v_empty = bar.v_empty(0);
    p.sc_full = bar.sc_full(0);
    p.steps = steps;
    p.it = it;
    p.begin = W.begin;
    p.s = W.s;
    p.h = W.h;
    p.lo = sp.lo;
    p.hi = sp.hi;
    p.len = W.q.L;
    return load_steps<D, FMT>(A, p, ok);
}

// The products of a task's steps.  Order: S0 S1 of the first step, then per step and
// tile O += P V and the next step's S.  st, tt: steps and tasks of either tile so far.
template <int D>
__device__ __forceinline__ void issue_steps(TileSmem<D> &sm, uint32_t tmem, Bars bar, int steps, uint32_t it, int tiles,
                                            const uint32_t (&st)[2], const uint32_t (&tt)[2], bool &ok) {
    using Smem = TileSmem<D>;
    // f16 operands, f32 sums, M = 128; S: both K-major, N = 128; O: B MN-major, N = D
    constexpr uint32_t S_DESC = (1u << 4) | ((uint32_t)(128 >> 3) << 17) | (8u << 24);
    constexpr uint32_t O_DESC = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | (8u << 24);
    const uint64_t q0 = operand(smem_u32(sm.q[0]), 16), k0 = operand(smem_u32(sm.k[0]), 16);
    const uint64_t v0 = operand(smem_u32(sm.v[0]), Smem::PANEL);
    auto scores = [&](int x, uint32_t stage) {
        const uint64_t a = q0 + x * (Smem::STAGE >> 4), b = k0 + stage * (Smem::STAGE >> 4);
        if (elected()) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                const uint32_t off = ((i >> 2) * Smem::PANEL + (i & 3) * 32) >> 4;
                mma_ss(tmem + 128 * x, a + off, b + off, S_DESC, i > 0);
            }
            commit(bar.s_full(x));
        }
        __syncwarp();
    };
    auto release = [&](uint32_t which) {
        if (elected()) commit(which);
        __syncwarp();
    };
    for (int x = 0; x < tiles; ++x) bar_wait(bar.q_full(x), tt[x] & 1, ok);
    bar_wait(bar.k_full(it & 1), (it >> 1) & 1, ok);
    fence_after();
    if (ok) {
        for (int x = 0; x < tiles; ++x) scores(x, it & 1);
        release(bar.k_empty(it & 1));
    }
#pragma unroll 1
    for (int j = 0; j < steps; ++j) {
        const uint32_t n = it + j;
        const bool more = j + 1 < steps;
        const uint32_t kb = more ? bar.k_full((n + 1) & 1) : bar.v_full(n & 1), kp = more ? ((n + 1) >> 1) & 1 : (n >> 1) & 1;
        if (!bar_try3(kb, kp, bar.v_full(n & 1), (n >> 1) & 1, bar.p_full(0), (st[0] + j) & 1)) {
            bar_wait(kb, kp, ok);
            bar_wait(bar.v_full(n & 1), (n >> 1) & 1, ok);
            bar_wait(bar.p_full(0), (st[0] + j) & 1, ok);
        }
        const uint64_t b = v0 + (n & 1) * (Smem::STAGE >> 4);
#pragma unroll 1
        for (int x = 0; x < tiles; ++x) {
            if (x == 1) bar_wait(bar.p_full(1), (st[1] + j) & 1, ok);
            fence_after();
            if (!ok) continue;
            if (elected()) {
#pragma unroll
                for (int i = 0; i < kTileTokens / 16; ++i)
                    mma_ts(tmem + 256 + 128 * x, tmem + 128 * x + 8 * i, b + i * (2048 >> 4), O_DESC, j > 0 || i > 0);
                if (!more) commit(bar.o_full(x));
            }
            __syncwarp();
            if (more) scores(x, (n + 1) & 1);
        }
        if (ok) {
            release(bar.v_empty(n & 1));
            if (more) release(bar.k_empty((n + 1) & 1));
        }
    }
}

template <int D, int FMT>
__global__ void __launch_bounds__(kTileThreads, 1) kv_tile_kernel(const __grid_constant__ AttnArgs A) {
    using Smem = TileSmem<D>;
    extern __shared__ __align__(1024) uint8_t tile_smem[];
    Smem &sm = *reinterpret_cast<Smem *>(tile_smem);
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Bars bar{smem_u32(sm.bar)};

    // Tensor memory is taken between the two: behind every kernel of the stream before this one, which may still
    // want some of its own (this CTA would hold it and wait for that kernel), and before every one after it
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t tmem = tile_enter<D>(sm, bar);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    const Share found = find_share<kTileWarps>(A, kTileCols, kTileShift, sm.share);
    bool ok = true, open = false;
    if (found.left > 0) {
        Walk W(A, kTileCols, kTileShift, found);
        uint32_t it = 0;   // steps so far: stage it % 2
        uint32_t st[2] = {0, 0}, tt[2] = {0, 0};  // steps of either tile, and tasks with steps
        while (W.next()) {
            const Seq &sq = W.q;
            const int steps = max(0, W.end - W.begin);
            const int rows = W.cols - W.col0;            // columns of the task, 256 at most count
            const int tiles = rows > kTileRows ? 2 : 1;
            const int first = sq.L - sq.n;               // token of the sequence's first row
            if (w < 8) {
                // ------------------------------------------------ softmax
                const int x = w >> 2;
                const int rt = threadIdx.x & 127;  // row of the tile = TMEM lane
                if (x < tiles) {
                    if (steps > 0) {
                        // Q: each thread its row, scaled by a power of two to f16
                        const int t = (W.col0 + kTileRows * x + rt) / A.group, hq = W.col0 + kTileRows * x + rt - t * A.group;
                        const bool there = W.col0 + kTileRows * x + rt < W.cols;
                        const uint4 *from = reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(A.q) +
                                                                            (size_t)(sq.a + t) * A.qs +
                                                                            ((size_t)W.h * A.group + hq) * D);
                        uint4 y[D / 8];
#pragma unroll
                        for (int i = 0; i < D / 8; ++i) y[i] = there ? from[i] : make_uint4(0, 0, 0, 0);
                        uint32_t mx = 0;  // the largest |q|, in its own type's bits
#pragma unroll
                        for (int i = 0; i < D / 8; ++i) {
                            const uint32_t u[4] = {y[i].x, y[i].y, y[i].z, y[i].w};
#pragma unroll
                            for (int z = 0; z < 4; ++z) mx = max(mx, max(u[z] & 0x7fffu, u[z] >> 16 & 0x7fffu));
                        }
                        float f = 1.0f;  // f16 stays as it is
                        if (A.type == Q4RDNA_BF16) {
                            int e = 140 - (int)(mx >> 7);  // the largest |q| to [2^13, 2^14)
                            e = mx == 0 || mx >= 0x7f80u ? 0 : min(e, kMostExponent);
                            f = __int_as_float((127 + e) << 23);
#pragma unroll
                            for (int i = 0; i < D / 8; ++i) {
                                uint32_t u[4] = {y[i].x, y[i].y, y[i].z, y[i].w};
#pragma unroll
                                for (int z = 0; z < 4; ++z)
                                    u[z] = pack_half(__uint_as_float(u[z] << 16) * f, __uint_as_float(u[z] & 0xffff0000u) * f);
                                y[i] = make_uint4(u[0], u[1], u[2], u[3]);
                            }
                            f = __int_as_float((127 - e) << 23);
                        }
#pragma unroll
                        for (int i = 0; i < D / 8; ++i) *reinterpret_cast<uint4 *>(sm.q[x] + swizzled(rt, i)) = y[i];
                        sm.qscale[x][rt] = A.scale * f;
                        fence_async();
                        __syncwarp();
                        if (lane == 0) bar_arrive(bar.q_full(x));
                    }
                    RowState r;
                    const int col = W.col0 + kTileRows * x + rt;
                    const bool there = col < W.cols;
                    r.R = -INFINITY;
                    r.l = 0.0f;
                    r.scale = steps > 0 ? sm.qscale[x][rt] : 0.0f;  // written by this warp
                    r.hi = there ? first + col / A.group : INT_MAX;  // (a padded row is computed and never read)
                    r.lo = there && A.window > 0 ? max(0, r.hi - A.window + 1) : 0;
                    const uint32_t lanes = (uint32_t)(32 * (w & 3)) << 16;
                    const uint32_t o_at = tmem + lanes + 256 + 128 * x;
                    if (steps > 0) {
                        RowPlace at;
                        at.s_at = tmem + lanes + 128 * x;
                        at.o_at = o_at;
                        at.s_full = bar.s_full(x);
                        at.p_full = bar.p_full(x);
                        at.sc_full = bar.sc_full(0);
                        at.steps = steps;
                        at.it = it;
                        at.parity = st[x];
                        at.tok0 = W.begin * kTileTokens;
                        at.all_lo = __reduce_max_sync(0xffffffffu, r.lo);
                        at.all_hi = __reduce_min_sync(0xffffffffu, r.hi);
                        ok = softmax_rows<D>(r, at, sm.scale, ok);
                        st[x] += steps;
                    }
                    // the result
                    if (steps > 0) bar_wait(bar.o_full(x), tt[x] & 1, ok);
                    if (steps > 0) ++tt[x];
                    fence_after();
                    const bool whole = W.whole();
                    const float inv = r.l == 0.0f ? 0.0f : 1.0f / r.l;
                    float *part = W.part(D);
                    const int j = kTileRows * x + rt;
                    const int tok = there ? col / A.group : 0;
                    const size_t at = (size_t)(sq.a + tok) * A.os + ((size_t)W.h * A.group + (there ? col - tok * A.group : 0)) * D;
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        uint32_t v[32];
                        if (steps > 0) {
                            tmem_load32(o_at + c, v);
                            tmem_arrived(v);
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = 0;
                        }
                        if (there) {
#pragma unroll
                            for (int i = 0; i < 32; i += 8) {
                                float y[8];
#pragma unroll
                                for (int z = 0; z < 8; ++z) y[z] = __uint_as_float(v[i + z]) * (whole ? inv : 1.0f);
                                if (whole) store_row<8>(A.out, at + c + i, A.type, y);
                                else store_row<8>(part, (size_t)j * D + c + i, Q4RDNA_F32, y);
                            }
                        }
                    }
                    if (there && !whole) {
                        part[kTileCols * D + j] = r.R;
                        part[kTileCols * D + kTileCols + j] = r.l;
                    }
                    fence_before();
                }
            } else if (w < kTileMmaWarp) {
                // ------------------------------------------------ loading
                if (steps > 0) {
                    ok = load_task<D, FMT>(A, sm, bar, W, kTileCols, steps, it, ok);
                }
            } else {
                // ------------------------------------------------ products
                // The whole warp walks and waits; one elected lane issues, so that operands
                // stay in uniform registers.
                if (steps > 0) {
                    issue_steps<D>(sm, tmem, bar, steps, it, tiles, st, tt, ok);
                    for (int x = 0; x < tiles; ++x) {
                        ++tt[x];
                        st[x] += steps;
                    }
                }
            }
            it += steps;
            if (W.open()) {
                open = true;
                if (threadIdx.x == 0) W.note();
            }
        }
    }
    if (threadIdx.x == 0 && !open) A.rec[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
    tile_leave(tmem, bar);
}

// ------------------------------------------------------------ f32 rows
//
// The same for f32 rows, in the same precision as the kernel for few columns: q and p as
// two f16 terms each (22 bits), and O summed in f32 by a warpgroup of its own, because
// the tensor core's running sum truncates (measured: 1 + 1.9 * 2^-24 stays 1), which over
// a task's products would cost 2^-17.  A task is 128 columns, one tile; Q's two terms
// take the two Q buffers, S two buffers in turn (the next step's S is made under this
// step's softmax), then the step's O and the task's O.  Warps 4-7 add one to the other.
// 1024 tokens behind 1024 others, 32 and 8 heads of 128: 143 us (bf16 rows 97 us).

constexpr int kTile32Cols = 128;

// Columns 32 c .. of S become the step's weights: 16 columns of first terms, 16 of second ones
template <int D>
__device__ __noinline__ bool softmax32_rows(const RowState &row, TileSmem<D> &sm, Bars bar, uint32_t tmem, int steps,
                                            uint32_t it, int tok0, bool ok) {
    RowState r = row;
    const int rt = threadIdx.x;
    const uint32_t lanes = (uint32_t)(threadIdx.x & 96) << 16;
    const int all_lo = __reduce_max_sync(0xffffffffu, r.lo), all_hi = __reduce_min_sync(0xffffffffu, r.hi);
#pragma unroll 1
    for (int j = 0; j < steps; ++j, tok0 += kTileTokens) {
        const uint32_t n = it + j;
        bar_wait(bar.s_full(n & 1), (n >> 1) & 1, ok);
        bar_wait(bar.sc_full(n & 3), (n >> 2) & 1, ok);  // at most one phase ahead once S is there
        fence_after();
        const uint32_t s_at = tmem + lanes + 128 * (n & 1);
        const float4 *const scale = sm.scale[n & 3];
        uint32_t v[32];
        auto hide = [&](int tok) {
            if (tok < all_lo || tok + 31 > all_hi) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (tok + i < r.lo || tok + i > r.hi) v[i] = 0xff800000u;  // -inf
            }
        };
        float t = -INFINITY;  // the largest exponent
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
            tmem_load32(s_at + 32 * c, v);
            tmem_arrived(v);
            hide(tok0 + 32 * c);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const float4 f = scale[2 * c + b];
                float m = -INFINITY;
#pragma unroll
                for (int i = 0; i < 16; ++i) m = fmaxf(m, __uint_as_float(v[16 * b + i]));
                // a block without a visible token has m = -inf, which a scale of 0 would turn into NaN
                if (m != -INFINITY) t = fmaxf(t, fmaf(m, f.x * r.scale, f.y));
            }
        }
        float f = 1.0f;
        if (t > r.R + 8.0f) {  // also the first: R = -inf
            f = ex2(r.R - t);
            r.l = shrunk(r.l, r.R - t);
            r.R = t;
        }
        const float ref = (r.R == -INFINITY ? 0.0f : r.R) - 7.0f;
        // the largest weight that may fall below 2^-126 in a block, against what the sum holds at least (2^7 / sv of its
        // first reference)
        const bool alone = __any_sync(0xffffffffu, scale[0].w * 0x1p-92f > (r.l > 0.0f ? r.l : 128.0f * scale[1].w));
        float exact = 0.0f;
        if (alone) exact = r.l + weights_alone(r.scale, ref, r.lo, r.hi, scale, s_at, tok0);
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
            uint32_t p[32];
            tmem_load32(s_at + 32 * c, v);
            tmem_arrived(v);
            const int tok = tok0 + 32 * c;
            const bool part = tok < all_lo || tok + 31 > all_hi;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const float4 g = scale[2 * c + b];
                const float a = g.x * r.scale, d = g.y - ref;
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    float e[2];
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        float x = fmaf(__uint_as_float(v[16 * b + i + z]), a, d);
                        const int at = tok + 16 * b + i + z;
                        if (part && (at < r.lo || at > r.hi)) x = -INFINITY;
                        e[z] = ex2(x);
                    }
                    sum += e[0] + e[1];
                    const uint32_t hi = pack_half(e[0], e[1]);
                    const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
                    p[8 * b + i / 2] = hi;
                    p[16 + 8 * b + i / 2] = pack_half(e[0] - h.x, e[1] - h.y);
                }
                // a block without a visible token takes nothing from its scale, be it NaN
                if (sum != 0.0f) r.l = fmaf(sum, g.z, r.l);
            }
            tmem_store32(s_at + 32 * c, p);
        }
        if (alone) r.l = exact;
        tmem_wait_store();
        fence_before();
        sm.turn[n & 3][rt] = f;
        if (j + 1 == steps) {
            sm.sum[128 * (n & 3) + rt] = r.l;
            sm.ref[128 * (n & 3) + rt] = r.R;
        }
        __syncwarp();
        if ((threadIdx.x & 31) == 0) {
            bar_arrive(bar.p_full(0));
            bar_arrive(bar.turned(n & 3));
        }
    }
    return ok;
}

// O = O * f + the step's O; after the last step to the output
template <int D>
__device__ __noinline__ bool add32_rows(const AttnArgs &A, const Walk &W, TileSmem<D> &sm, Bars bar, uint32_t tmem, int steps,
                                        uint32_t it, bool ok) {
    const int rt = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)(threadIdx.x & 96) << 16;
    const uint32_t step_at = tmem + lanes + 256, o_at = tmem + lanes + 384;
    const bool whole = W.whole();
    const int col = W.col0 + rt;
    const bool there = col < W.cols;
    const int tok = there ? col / A.group : 0;
    float *const part = W.part(D);
    const size_t at = (size_t)(W.q.a + tok) * A.os + ((size_t)W.h * A.group + (there ? col - tok * A.group : 0)) * D;
    for (int j = 0; j < max(steps, 1); ++j) {
        const uint32_t n = it + j;
        float f = 1.0f, l = 0.0f, R = -INFINITY;
        const bool last = j + 1 >= steps;
        if (steps > 0) {
            bar_wait(bar.o_full(0), n & 1, ok);
            bar_wait(bar.turned(n & 3), (n >> 2) & 1, ok);  // at most one phase ahead once the step's O is there
            fence_after();
            f = sm.turn[n & 3][rt];
            if (last) {
                l = sm.sum[128 * (n & 3) + rt];
                R = sm.ref[128 * (n & 3) + rt];
            }
        }
        const float inv = !whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
            uint32_t v[32], u[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = u[i] = 0;
            if (steps > 0) {
                tmem_load32(step_at + c, v);
                if (j > 0) tmem_load32(o_at + c, u);
                tmem_arrived(v);
                tmem_arrived(u);
            }
            if (j > 0) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    v[i] = __float_as_uint(fmaf(__uint_as_float(u[i]), f, __uint_as_float(v[i])));
            }
            if (!last) {
                tmem_store32(o_at + c, v);
            } else if (there) {
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    float y[8];
#pragma unroll
                    for (int z = 0; z < 8; ++z) y[z] = __uint_as_float(v[i + z]) * inv;
                    if (whole) store_row<8>(A.out, at + c + i, A.type, y);
                    else store_row<8>(part, (size_t)rt * D + c + i, Q4RDNA_F32, y);
                }
            }
        }
        if (last && there && !whole) {
            part[kTile32Cols * D + rt] = R;
            part[kTile32Cols * D + kTile32Cols + rt] = l;
        }
        if (steps > 0) {
            tmem_wait_store();
            fence_before();
            __syncwarp();
            if ((threadIdx.x & 31) == 0) bar_arrive(bar.o_free());
        }
    }
    return ok;
}

template <int D>
__device__ __forceinline__ void issue32_steps(TileSmem<D> &sm, uint32_t tmem, Bars bar, int steps, uint32_t it, uint32_t task,
                                              bool &ok) {
    using Smem = TileSmem<D>;
    constexpr uint32_t S_DESC = (1u << 4) | ((uint32_t)(128 >> 3) << 17) | (8u << 24);
    constexpr uint32_t O_DESC = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | (8u << 24);
    const uint64_t q0 = operand(smem_u32(sm.q[0]), 16), k0 = operand(smem_u32(sm.k[0]), 16);
    const uint64_t v0 = operand(smem_u32(sm.v[0]), Smem::PANEL);
    auto scores = [&](uint32_t n) {
        const uint64_t b = k0 + (n & 1) * (Smem::STAGE >> 4);
        if (elected()) {
#pragma unroll
            for (int x = 1; x >= 0; --x)  // the second, small terms first: their sum's rounding is small too
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    const uint32_t off = ((i >> 2) * Smem::PANEL + (i & 3) * 32) >> 4;
                    mma_ss(tmem + 128 * (n & 1), q0 + x * (Smem::STAGE >> 4) + off, b + off, S_DESC, x == 0 || i > 0);
                }
            commit(bar.s_full(n & 1));
            commit(bar.k_empty(n & 1));
        }
        __syncwarp();
    };
    bar_wait(bar.q_full(0), task & 1, ok);
    bar_wait(bar.k_full(it & 1), (it >> 1) & 1, ok);
    fence_after();
    if (ok) scores(it);
#pragma unroll 1
    for (int j = 0; j < steps; ++j) {
        const uint32_t n = it + j;
        if (j + 1 < steps) {
            // S of the next step goes where the step before this one had its P, whose products were issued earlier
            bar_wait(bar.k_full((n + 1) & 1), ((n + 1) >> 1) & 1, ok);
            fence_after();
            if (ok) scores(n + 1);
        }
        if (!bar_try3(bar.p_full(0), n & 1, bar.v_full(n & 1), (n >> 1) & 1, bar.o_free(), (n & 1) ^ 1)) {
            bar_wait(bar.v_full(n & 1), (n >> 1) & 1, ok);
            bar_wait(bar.o_free(), (n & 1) ^ 1, ok);
            bar_wait(bar.p_full(0), n & 1, ok);
        }
        fence_after();
        if (!ok) continue;
        const uint64_t b = v0 + (n & 1) * (Smem::STAGE >> 4);
        if (elected()) {
#pragma unroll
            for (int x = 1; x >= 0; --x)
#pragma unroll
                for (int i = 0; i < kTileTokens / 16; ++i)
                    mma_ts(tmem + 256, tmem + 128 * (n & 1) + 32 * (i >> 1) + 8 * (i & 1) + 16 * x, b + i * (2048 >> 4), O_DESC,
                           x == 0 || i > 0);
            commit(bar.o_full(0));
            commit(bar.v_empty(n & 1));
        }
        __syncwarp();
    }
}

template <int D, int FMT>
__global__ void __launch_bounds__(kTileThreads, 1) kv_tile32_kernel(const __grid_constant__ AttnArgs A) {
    using Smem = TileSmem<D>;
    extern __shared__ __align__(1024) uint8_t tile_smem[];
    Smem &sm = *reinterpret_cast<Smem *>(tile_smem);
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Bars bar{smem_u32(sm.bar)};
    // Tensor memory is taken between the two: behind every kernel of the stream before this one, which may still
    // want some of its own (this CTA would hold it and wait for that kernel), and before every one after it
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t tmem = tile_enter<D>(sm, bar);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    const Share found = find_share<kTileWarps>(A, kTile32Cols, kTileShift, sm.share);
    bool ok = true, open = false;
    if (found.left > 0) {
        Walk W(A, kTile32Cols, kTileShift, found);
        uint32_t it = 0, task = 0;  // steps and tasks with steps so far
        while (W.next()) {
            const Seq &sq = W.q;
            const int steps = max(0, W.end - W.begin);
            if (w < 4) {
                if (steps > 0) {
                    // Q: each thread its row, scaled by a power of two, in two f16 terms
                    const int rt = threadIdx.x, col = W.col0 + rt, tok = col / A.group;
                    const bool there = col < W.cols;
                    const float4 *from = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(A.q) +
                                                                          (size_t)(sq.a + (there ? tok : 0)) * A.qs +
                                                                          ((size_t)W.h * A.group + (there ? col - tok * A.group : 0)) * D);
                    uint32_t mx = 0;
#pragma unroll 8
                    for (int i = 0; i < D / 4; ++i) {
                        const float4 y = from[i];
                        mx = max(max(mx, max(__float_as_uint(y.x) & 0x7fffffffu, __float_as_uint(y.y) & 0x7fffffffu)),
                                 max(__float_as_uint(y.z) & 0x7fffffffu, __float_as_uint(y.w) & 0x7fffffffu));
                    }
                    int e = 140 - (int)(mx >> 23);  // the largest |q| to [2^13, 2^14)
                    e = mx == 0 || mx >= 0x7f800000u ? 0 : min(e, kMostExponent);
                    const float f = there ? __int_as_float((127 + e) << 23) : 0.0f;
#pragma unroll 4
                    for (int i = 0; i < D / 8; ++i) {
                        const float4 a = from[2 * i], b = from[2 * i + 1];
                        const float y[8] = {a.x * f, a.y * f, a.z * f, a.w * f, b.x * f, b.y * f, b.z * f, b.w * f};
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int z = 0; z < 4; ++z) {
                            hi[z] = pack_half(y[2 * z], y[2 * z + 1]);
                            const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&hi[z]));
                            lo[z] = pack_half(y[2 * z] - h.x, y[2 * z + 1] - h.y);
                        }
                        *reinterpret_cast<uint4 *>(sm.q[0] + swizzled(rt, i)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        *reinterpret_cast<uint4 *>(sm.q[1] + swizzled(rt, i)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                    fence_async();
                    __syncwarp();
                    if (lane == 0) bar_arrive(bar.q_full(0));
                    RowState r;
                    r.R = -INFINITY;
                    r.l = 0.0f;
                    r.scale = A.scale * __int_as_float((127 - e) << 23);
                    r.hi = there ? sq.L - sq.n + tok : INT_MAX;  // (a padded row is computed and never read)
                    r.lo = there && A.window > 0 ? max(0, r.hi - A.window + 1) : 0;
                    ok = softmax32_rows<D>(r, sm, bar, tmem, steps, it, W.begin * kTileTokens, ok);
                }
            } else if (w < 8) {
                ok = add32_rows<D>(A, W, sm, bar, tmem, steps, it, ok);
            } else if (w < kTileMmaWarp) {
                if (steps > 0) ok = load_task<D, FMT>(A, sm, bar, W, kTile32Cols, steps, it, ok);
            } else if (steps > 0) {
                issue32_steps<D>(sm, tmem, bar, steps, it, task, ok);
            }
            it += steps;
            if (steps > 0) ++task;
            if (W.open()) {
                open = true;
                if (threadIdx.x == 0) W.note();
            }
        }
    }
    if (threadIdx.x == 0 && !open) A.rec[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
    tile_leave(tmem, bar);
}

}  // namespace q4kv
