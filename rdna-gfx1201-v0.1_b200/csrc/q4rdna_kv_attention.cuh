// Attention over the 8-bit cache, few columns per sequence (q4rdna_kv_attention): a task
// (q4rdna_kv_split.cuh) is NC = 8 NT columns, its pieces the 16-token blocks.
// HBM-bound: every block is read once per task, 2 D + 1/2 bytes per token and head.
//
//   * A CTA's 8 warps take its blocks in turn and meet in shared memory at the end
//     of a task's blocks.
//   * Scores on the tensor cores: S^T = K q^T as mma.m16n8k16 with f16 operands and
//     f32 sums, A = 16 tokens x 16 dims of codes (exact in f16), B = 16 dims x 8
//     columns.  q is scaled per column by a power of two and, for f32 rows, taken as
//     two f16 terms (22 bits); 16-bit rows are exact in one.  The block's key scale
//     multiplies the sums.
//   * O^T = V^T p^T likewise: A = 16 dims x 16 tokens, one block's sum from zero,
//     then O = fma(value scale, sum, O) in f32 (the tensor core's own running sum
//     truncates; started anew for each block it never runs long).  p = 2^(s - m) in
//     f16, two terms for f32 rows; m moves only when a score outgrows it by 2^8, and
//     p carries a factor 2^7, so neither the largest nor the small weights leave
//     f16's range.  One term for 16-bit rows: 2^-12 of a weight, below their own rounding
//     (bf16 128 x 4093: off by 1.67e-3 against 64 bits, 1.66e-3 with weights in f32).
//   * Codes go straight from global memory to the fragments: any order of the dims
//     (of K and q alike), of the tokens (of K's rows and V's columns alike) and of
//     the output dims is as good as another, so the order is chosen such that a lane
//     loads 16 bytes at a time: K, dims 16 c .. 16 c + 15 of tokens t0 and t0 + 2; V,
//     dims D/8 g .. of tokens 4 c .. 4 c + 3 (lane = 4 g + c).
//
// Measured (8 kv heads of 128, device time with the join): 128 sequences of up to 4093
// tokens, 64 query heads, e4m3, bf16 141 us, 0.63 of the bytes' time at 6543 GB/s; 32
// query heads, int8, f32: 16 sequences of up to 8191 46 us and one of 65521 39 us, 0.52 and
// 0.53, one of 517 12 us.  About 17 us of a call are fixed: the table of shares, the
// latency of the first loads, the meeting of the warps, the join.  Sums by int8 products
// (codes as they are, q in digits) took 164 us where this took 157 (64 of 8191).
#pragma once

#include "q4rdna_kv_split.cuh"

namespace q4kv {

constexpr int kAttnWarps = 8;
constexpr int kAttnThreads = 32 * kAttnWarps;
constexpr float kBoost = 7.0f;  // p carries 2^7
constexpr float kStep = 8.0f;   // m moves when a score outgrows it by more

// ------------------------------------------------------------ fragments

// Ordinary loads: the kernel is resident while the append before it in the stream writes these tiles, and the
// read-only path promises data that nobody writes as long as the kernel lives (griddepcontrol.wait makes the
// writes visible to ordinary loads; the times are the same)
__device__ __forceinline__ uint4 ld_stream(const uint8_t *p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 ld_stream2(const uint8_t *p) {
    uint2 v;
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}

// (a, b): code number I of the words a and b (two tokens, one dim)
template <int FMT>
__device__ __forceinline__ void pairs_of(uint32_t a, uint32_t b, uint32_t (&r)[4]) {
    if constexpr (FMT == Q4RDNA_KV_INT8) {
        const uint32_t lo = __byte_perm(a, b, 0x5140), hi = __byte_perm(a, b, 0x7362);
        r[0] = sub_1152(__byte_perm(lo, 0x64646464u, 0x4140));
        r[1] = sub_1152(__byte_perm(lo, 0x64646464u, 0x4342));
        r[2] = sub_1152(__byte_perm(hi, 0x64646464u, 0x4140));
        r[3] = sub_1152(__byte_perm(hi, 0x64646464u, 0x4342));
    } else {
        const uint32_t lo = __byte_perm(a, b, 0x5140), hi = __byte_perm(a, b, 0x7362);
        r[0] = e4m3_pair<false>(lo);
        r[1] = e4m3_pair<true>(lo);
        r[2] = e4m3_pair<false>(hi);
        r[3] = e4m3_pair<true>(hi);
    }
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
// ------------------------------------------------------------ the kernel

template <int D, int NT>
struct AttnSmem {
    static constexpr int NC = 8 * NT;
    static constexpr int QROW = D + 8;  // halves of a q row: 16 bytes more, so that the rows' fragments fall into different banks
    static constexpr int OROW = D + 4;
    __half q[2][NC][QROW];
    float qscale[NC];
    float o[kAttnWarps][NC][OROW];
    float m[kAttnWarps][NC], l[kAttnWarps][NC];
    ShareSmem<kAttnWarps> share;
};

template <int D, int FMT, int NT, int TERMS>
__global__ void __launch_bounds__(kAttnThreads, D == 64 || (NT == 1 && D == 128) ? 2 : 1)
kv_attention_kernel(const __grid_constant__ AttnArgs A) {
    using Smem = AttnSmem<D, NT>;
    constexpr int NC = Smem::NC, KW = D / 64;  // KW: 16-byte loads of a K row per lane
    constexpr int VB = D / 8;                  // bytes of a V row per lane
    constexpr int MT = D / 16;                 // M tiles of the output
    extern __shared__ __align__(16) uint8_t smem_raw[];
    Smem &sm = *reinterpret_cast<Smem *>(smem_raw);
    const Batch &B = A.b;
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const Share found = find_share<kAttnWarps>(A, NC, 4, sm.share);
    if (found.left == 0) {
        if (threadIdx.x == 0) A.rec[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
        return;
    }
    bool open = false;  // the share ends inside a task that began in it
    const int t0 = 4 * (g >> 1) + (g & 1);  // K rows g and g + 8 of the fragments: tokens t0 and t0 + 2
    Walk W(A, NC, 4, found);

    uint4 kr[2][KW];
    uint32_t vr[4][VB / 4];
    float2 sc = make_float2(0.0f, 0.0f);
    auto load_k = [&](const uint8_t *tile) {
#pragma unroll
        for (int i = 0; i < KW; ++i) {
            kr[0][i] = ld_stream(tile + kHeader + t0 * D + 16 * c + 64 * i);
            kr[1][i] = ld_stream(tile + kHeader + (t0 + 2) * D + 16 * c + 64 * i);
        }
    };
    auto load_v = [&](const uint8_t *tile) {
        const uint8_t *p = tile + kHeader + (kBlock + 4 * c) * D + VB * g;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if constexpr (VB == 8) {
                const uint2 x = ld_stream2(p + t * D);
                vr[t][0] = x.x; vr[t][1] = x.y;
            } else {
#pragma unroll
                for (int i = 0; i < VB / 16; ++i) {
                    const uint4 x = ld_stream(p + t * D + 16 * i);
                    vr[t][4 * i] = x.x; vr[t][4 * i + 1] = x.y; vr[t][4 * i + 2] = x.z; vr[t][4 * i + 3] = x.w;
                }
            }
        }
    };
    // This warp's blocks are b, b + kAttnWarps, ...; lane i holds the page of the i-th of 32,
    // so that the loop waits for no page table
    int b = 0, at = 0, pages = 0;
    const uint8_t *tile = nullptr;
    auto fetch_pages = [&]() {
        const int blk = b + kAttnWarps * lane;
        pages = blk < W.end ? B.table[(size_t)W.s * B.stride + (blk >> A.c.nbl)] : 0;
        at = 0;
    };
    // the next block of this warp, from b on, whose page lies in the cache
    auto next_tile = [&]() -> const uint8_t * {
        for (; b < W.end; b += kAttnWarps, ++at) {
            if (at == 32) fetch_pages();
            const int page = __shfl_sync(0xffffffffu, pages, at);
            if ((unsigned)page < (unsigned)A.c.pages) {
                const size_t t = (((size_t)page * A.c.hk + W.h) << A.c.nbl) + (b & ((1 << A.c.nbl) - 1));
                return A.c.tiles + t * A.c.tile_bytes;
            }
            if (lane == 0) atomicOr(&g_kv_fault, kFaultBatch);
        }
        return nullptr;
    };
    // a task's first block on its way
    auto enter = [&]() {
        b = W.begin + w;
        fetch_pages();
        tile = next_tile();
        if (tile != nullptr) {
            load_k(tile);
            load_v(tile);
            sc = *reinterpret_cast<const float2 *>(tile);
        }
    };
    bool more = W.next();
    if (more) enter();
    while (more) {
        const Seq sq = W.q;
        const int cols = W.cols, h = W.h, col0 = W.col0;
        const int first = sq.L - sq.n;  // token of the sequence's first row

        // ---- q of the columns, scaled to f16
        __syncthreads();  // the last task's join has read shared memory
        for (int j = w; j < NC; j += kAttnWarps) {
            const int col = col0 + j;
            float x[D / 32];
            uint32_t mx = 0;
            if (col < cols) {
                const int i = col / A.group;
                load_row<D / 32>(A.q, (size_t)(sq.a + i) * A.qs +
                                          ((size_t)h * A.group + (col - i * A.group)) * D + lane * (D / 32),
                                 A.type, x);
            }
#pragma unroll
            for (int t = 0; t < D / 32; ++t) {
                if (col >= cols) x[t] = 0.0f;
                mx = max(mx, __float_as_uint(x[t]) & 0x7fffffffu);
            }
            mx = __reduce_max_sync(0xffffffffu, mx);
            // the largest |q| to [2^13, 2^14)
            int e = 140 - (int)(mx >> 23);
            e = mx == 0 || mx >= 0x7f800000u ? 0 : min(e, kMostExponent);
            const float f = __int_as_float((127 + e) << 23);
#pragma unroll
            for (int t = 0; t < D / 32; t += 2) {
                const float a = x[t] * f, b = x[t + 1] * f;
                const uint32_t hi = pack_half(a, b);
                *reinterpret_cast<uint32_t *>(&sm.q[0][j][lane * (D / 32) + t]) = hi;
                if constexpr (TERMS == 2) {
                    const float2 r = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
                    *reinterpret_cast<uint32_t *>(&sm.q[1][j][lane * (D / 32) + t]) = pack_half(a - r.x, b - r.y);
                }
            }
            if (lane == 0)
                sm.qscale[j] = A.scale * __int_as_float((127 - e) << 23);
        }
        __syncthreads();

        // ---- this warp's blocks
        float o[NT][MT][4], m[NT][2], l[NT][2], cs[NT][2];
        int plo[NT][2], phi[NT][2];  // tokens that the lane's columns see
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int z = 0; z < 4; ++z) o[n][i][z] = 0.0f;
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                m[n][z] = -INFINITY;
                l[n][z] = 0.0f;
                const int col = col0 + 8 * n + 2 * c + z;
                cs[n][z] = sm.qscale[8 * n + 2 * c + z];
                phi[n][z] = col < cols ? first + col / A.group : -1;
                plo[n][z] = A.window > 0 ? phi[n][z] - A.window + 1 : 0;
            }
        }
        // blocks that every column sees whole need no mask (padded columns are all zero and never read)
        const int last = first + min(sq.n - 1, (col0 + NC - 1) / A.group);
        const int full_hi = (first + col0 / A.group + 1) >> 4;  // first block that is not whole below
        const int full_lo = A.window > 0 ? (max(0, last - A.window + 1) + 15) >> 4 : 0;

        while (tile != nullptr) {
            const int cur = b;
            b += kAttnWarps;
            ++at;
            const uint8_t *next = next_tile();
            // its registers are free only as this block's are used up; until then it comes to L2 (128 x 4093: 143 -> 140
            // us; the block after it too: 148)
            if (next != nullptr)
                for (int i = lane * 128; i < kHeader + 2 * kBlock * D; i += 32 * 128)
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(next + i) : "memory");

            // scores
            float sa[NT][TERMS][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int t = 0; t < TERMS; ++t)
#pragma unroll
                    for (int z = 0; z < 4; ++z) sa[n][t][z] = 0.0f;
#pragma unroll
            for (int i = 0; i < KW; ++i) {
                const uint32_t r0[4] = {kr[0][i].x, kr[0][i].y, kr[0][i].z, kr[0][i].w};
                const uint32_t r1[4] = {kr[1][i].x, kr[1][i].y, kr[1][i].z, kr[1][i].w};
                uint32_t qf[NT][TERMS][8];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int t = 0; t < TERMS; ++t) {
                        const uint4 *p = reinterpret_cast<const uint4 *>(&sm.q[t][8 * n + g][64 * i + 16 * c]);
                        const uint4 x = p[0], y = p[1];
                        qf[n][t][0] = x.x; qf[n][t][1] = x.y; qf[n][t][2] = x.z; qf[n][t][3] = x.w;
                        qf[n][t][4] = y.x; qf[n][t][5] = y.y; qf[n][t][6] = y.z; qf[n][t][7] = y.w;
                    }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const uint32_t x0 = FMT == Q4RDNA_KV_INT8 ? r0[u] ^ 0x80808080u : r0[u];
                    const uint32_t x1 = FMT == Q4RDNA_KV_INT8 ? r1[u] ^ 0x80808080u : r1[u];
                    const uint32_t a0 = pair_of<FMT, 0>(x0), a2 = pair_of<FMT, 2>(x0);
                    const uint32_t a1 = pair_of<FMT, 0>(x1), a3 = pair_of<FMT, 2>(x1);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int t = 0; t < TERMS; ++t)
                            mma_f16(sa[n][t], a0, a1, a2, a3, qf[n][t][2 * u], qf[n][t][2 * u + 1]);
                }
            }
            const float2 scale = sc;
            if (next != nullptr) {
                load_k(next);
                sc = *reinterpret_cast<const float2 *>(next);
            }

            // softmax weights; lane: tokens t0, t0 + 2 of columns 2 c, 2 c + 1
            const bool whole = cur >= full_lo && cur < full_hi;
            uint32_t pf[NT][TERMS][2];
            float sv[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float x[4];
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    x[z] = sa[n][0][z];
                    if constexpr (TERMS == 2) x[z] += sa[n][1][z];
                    x[z] *= scale.x * cs[n][z & 1];
                }
                sv[n][0] = sv[n][1] = scale.y;
                if (!whole) {
                    if (FMT == Q4RDNA_KV_E4M3 && n == 0) {
                        // rows of the tile that hold no token yet may hold NaN, which a weight of 0 would keep
#pragma unroll
                        for (int t = 0; t < 4; ++t)
                            if (cur * kBlock + 4 * c + t > last)
#pragma unroll
                                for (int i = 0; i < VB / 4; ++i) vr[t][i] = 0;
                    }
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        const int tok = cur * kBlock + t0 + (z & 2);
                        if (tok > phi[n][z & 1] || tok < plo[n][z & 1]) x[z] = -INFINITY;
                    }
#pragma unroll
                    for (int z = 0; z < 2; ++z)  // a column that sees nothing here takes nothing from the tile's scale
                        if (cur * kBlock > phi[n][z] || cur * kBlock + kBlock - 1 < plo[n][z]) sv[n][z] = 0.0f;
                }
                float f[2];
                bool moved = false;
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    float y = fmaxf(x[z], x[z + 2]);
                    y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 4));
                    y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 8));
                    y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 16));
                    f[z] = 1.0f;
                    if (y > m[n][z] + kStep) {  // also the first score: m = -inf
                        f[z] = ex2(m[n][z] - y);
                        m[n][z] = y;
                        moved = true;
                    }
                }
                if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int z = 0; z < 4; ++z) o[n][i][z] *= f[z & 1];
                    l[n][0] *= f[0];
                    l[n][1] *= f[1];
                }
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    const float ref = m[n][z & 1];
                    x[z] = ex2(x[z] - (ref == -INFINITY ? 0.0f : ref) + kBoost);
                    l[n][z & 1] += x[z];
                }
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    const uint32_t hi = pack_half(x[2 * z], x[2 * z + 1]);
                    pf[n][0][z] = transpose8(hi);
                    if constexpr (TERMS == 2) {
                        const float2 r = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
                        pf[n][1][z] = transpose8(pack_half(x[2 * z] - r.x, x[2 * z + 1] - r.y));
                    }
                }
            }

            // values
#pragma unroll
            for (int u = 0; u < VB / 4; ++u) {
                uint32_t lo[4], hi[4];
                if constexpr (FMT == Q4RDNA_KV_INT8) {
                    pairs_of<FMT>(vr[0][u] ^ 0x80808080u, vr[1][u] ^ 0x80808080u, lo);
                    pairs_of<FMT>(vr[2][u] ^ 0x80808080u, vr[3][u] ^ 0x80808080u, hi);
                } else {
                    pairs_of<FMT>(vr[0][u], vr[1][u], lo);
                    pairs_of<FMT>(vr[2][u], vr[3][u], hi);
                }
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int t = 0; t < TERMS; ++t)
                            mma_f16(acc, lo[2 * v], lo[2 * v + 1], hi[2 * v], hi[2 * v + 1], pf[n][t][0], pf[n][t][1]);
#pragma unroll
                        for (int z = 0; z < 4; ++z)
                            o[n][2 * u + v][z] = fmaf(sv[n][z & 1], acc[z], o[n][2 * u + v][z]);
                    }
            }
            if (next != nullptr) load_v(next);
            tile = next;
        }

        // ---- the warps meet
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                const int j = 8 * n + 2 * c + z;
                float x = l[n][z];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                if (g == 0) {
                    sm.m[w][j] = m[n][z];
                    sm.l[w][j] = x;
                }
#pragma unroll
                for (int i = 0; i < MT; ++i)  // M tile i: dims VB g + 2 i (rows g) and + 1 (rows g + 8)
                    *reinterpret_cast<float2 *>(&sm.o[w][j][VB * g + 2 * i]) =
                        make_float2(o[n][i][z], o[n][i][z + 2]);
            }
        const bool whole_task = W.whole();
        float *part = W.part(D);
        if (W.open()) {
            open = true;
            if (threadIdx.x == 0) W.note();
        }
        more = W.next();
        if (more) enter();  // while this task's results meet
        __syncthreads();
        for (int e = threadIdx.x; e < NC * (D / 4); e += kAttnThreads) {
            const int j = e / (D / 4), d = 4 * (e % (D / 4));
            const int col = col0 + j;
            if (col >= cols) continue;
            float M = -INFINITY, L = 0.0f, f[kAttnWarps];
#pragma unroll
            for (int i = 0; i < kAttnWarps; ++i) M = fmaxf(M, sm.m[i][j]);
            float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < kAttnWarps; ++i) {
                // a warp that saw nothing has l = 0 and o = 0, or NaN, which goes through
                f[i] = sm.m[i][j] == -INFINITY ? 1.0f : ex2(sm.m[i][j] - M);
                L = fmaf(f[i], sm.l[i][j], L);
                const float4 y = *reinterpret_cast<const float4 *>(&sm.o[i][j][d]);
                x[0] = fmaf(f[i], y.x, x[0]);
                x[1] = fmaf(f[i], y.y, x[1]);
                x[2] = fmaf(f[i], y.z, x[2]);
                x[3] = fmaf(f[i], y.w, x[3]);
            }
            if (whole_task) {
                const float r = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
                for (int z = 0; z < 4; ++z) x[z] *= r;
                const int i = col / A.group;
                store_row<4>(A.out, (size_t)(sq.a + i) * A.os + ((size_t)h * A.group + (col - i * A.group)) * D + d,
                             A.type, x);
            } else {
                *reinterpret_cast<float4 *>(part + j * D + d) = make_float4(x[0], x[1], x[2], x[3]);
                if (d == 0) {
                    part[NC * D + j] = M;
                    part[NC * D + NC + j] = L;
                }
            }
        }
    }
    if (threadIdx.x == 0 && !open) A.rec[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
}

}  // namespace q4kv
