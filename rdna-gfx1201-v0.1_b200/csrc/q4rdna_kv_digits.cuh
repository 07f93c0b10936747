// Attention over an int8 cache, at most four columns per task: decode with up to four
// query heads per kv head (q4rdna_kv_attention), in exact integer arithmetic on the int8
// tensor cores.  HBM-bound; the kernel for any columns (q4rdna_kv_attention.cuh) spends
// 490 instructions per 16-token block, 200 of them on turning codes into f16, and reaches
// half of the bandwidth.  Here the codes are operands as they lie.
//
//   * q of a column is scaled by a power of two and rounded to 31 bits, X = four balanced
//     base-256 digits; the 16 rows of an mma.m16n8k32 are 4 columns x 4 digits (rows g and
//     g + 8 of a lane: digits 2 (g & 1) and 2 (g & 1) + 1 of column g / 2).  S = sum of
//     digit sums times 256^d: exact up to q's rounding, 2^-31 of the column's largest.
//   * p = 2^(s - m) times the block's value scale over `vref` likewise becomes 31 bits,
//     2^27 for 1, and four digits; O's rows are digit sums, in int32 without rounding over
//     all of a warp's blocks.  They go to f32 sums in shared memory when m or vref has to
//     move (a score outgrows m by 2^3, or a value scale vref: rare), after 2^16 tokens, and at the end.
//   * Per 32 tokens: S = 4 tiles of 8 tokens x D / 32 products, O = D / 8 tiles x 1.  The
//     order of the tokens in S's columns is such that a lane's weights are just those that
//     it needs as O's A operand; values take a 4 x 4 byte transpose (8 byte permutes for
//     16 codes).
//   * A lane's own bytes come through a ring of its own in shared memory (cp.async, two
//     pairs of blocks), so that no registers wait for HBM and no barrier is needed.
#pragma once

#include "q4rdna_kv_split.cuh"

namespace q4kv {

constexpr int kDigWarps = 6, kDigThreads = 32 * kDigWarps, kDigCols = 4;
constexpr uint32_t kDigMagic = 0x4B400000u;  // 1.5 * 2^23: an int32 sum on it reads back as f32 by a subtraction
constexpr float kDigMagicF = 12582912.0f;
constexpr float kDigAhead = 1.0f, kDigStep = 3.0f;  // m above the scores that set it; scores above m
constexpr float kDigOne = 0x1p27f;                   // the integer of a weight of 1: 2^30 with a score kDigStep above m

template <int D>
struct DigSmem {
    static constexpr int BLOCK = 32 * D;  // codes of a tile
    uint8_t ring[kDigWarps][4][BLOCK];
    float o[kDigWarps][kDigCols][D + 4];
    uint32_t q[kDigCols][D];  // X's digits, one word per element
    float qscale[kDigCols];
    float m[kDigWarps][kDigCols], l[kDigWarps][kDigCols];
    ShareSmem<kDigWarps> share;
};

__device__ __forceinline__ void mma_s8(uint32_t (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                       const uint32_t (&c)[4]) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}
// X as four balanced base-256 digits, one per byte
__device__ __forceinline__ uint32_t digits_of(int x) { return ((uint32_t)x + 0x00808080u) ^ 0x00808080u; }

// The digit sums join the warp's f32 sums of the four columns: o = (o + sums * unit) * f,
// f per column (this lane's column g / 2)
template <int D>
__device__ __forceinline__ void flush_sums(int (&acc)[D / 8][4], float (*o)[D + 4], float unit, float f) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const float low = (g & 1) ? unit * 65536.0f : unit;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
        float v[2];
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            v[z] = fmaf((float)acc[j][z + 2], 256.0f, (float)acc[j][z]) * low;
            v[z] += __shfl_xor_sync(0xffffffffu, v[z], 4);
            acc[j][z] = acc[j][z + 2] = 0;
        }
        // columns 2 c, 2 c + 1 of tile j are dims (D / 8) (2 c) + j and (D / 8) (2 c + 1) + j; one for either lane of the pair
        float *const at = &o[g >> 1][(D / 8) * (2 * c + (g & 1)) + j];
        *at = (*at + ((g & 1) ? v[1] : v[0])) * f;
    }
    __syncwarp();
}

template <int D>
__global__ void __launch_bounds__(kDigThreads, 2) kv_digits_kernel(const __grid_constant__ AttnArgs A) {
    using Smem = DigSmem<D>;
    constexpr int NC = kDigCols;
    constexpr int CH = D / 64;   // 16-byte pieces of a K row per lane
    constexpr int KS = D / 32;   // k-steps of S
    constexpr int VB = D / 8;    // bytes of a V row per lane
    extern __shared__ __align__(16) uint8_t smem_raw[];
    Smem &sm = *reinterpret_cast<Smem *>(smem_raw);
    const Batch &B = A.b;
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const long long left = find_share<kDigWarps>(A, NC, 4, sm.share);
    if (left == 0) {
        if (threadIdx.x == 0) A.rec[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
        return;
    }
    bool open = false;  // the share ends inside a task that began in it
    const uint32_t magic[4] = {kDigMagic, kDigMagic, kDigMagic, kDigMagic};
    // byte selectors of this lane's two digits, from two words' same bytes
    const uint32_t sel0 = (g & 1) ? 0x0062u : 0x0040u, sel1 = (g & 1) ? 0x0073u : 0x0051u;
    uint8_t *const ring = sm.ring[w][0];
    const uint32_t ring_at = smem_u32(ring);
    Walk W(A, NC, 4, left, sm.share);
    while (W.next()) {
        const Seq &sq = W.q;
        const int s = W.s, cols = W.cols, h = W.h, col0 = W.col0, b0 = W.begin, b1 = W.end;
        const int first = sq.L - sq.n;  // token of the sequence's first row

        // ---- q of this warp's column and the pages of its first 16 pairs, on their way together
        constexpr int N = D / 32;
        float qx[N];
#pragma unroll
        for (int t = 0; t < N; ++t) qx[t] = 0.0f;
        if (w < NC && col0 + w < cols) {
            const int i = (col0 + w) / A.group;
            load_row<N>(A.q, (size_t)(sq.a + i) * A.qs + ((size_t)h * A.group + (col0 + w - i * A.group)) * D + lane * N, A.type, qx);
        }
        // this warp's pairs are blocks p, p + 1, then 2 kDigWarps further; lane i: the page of the
        // pair i / 2 of 16
        int p = b0 + 2 * w;
        auto pages_from = [&](int at) {
            const int blk = at + 2 * kDigWarps * (lane >> 1) + (lane & 1);
            return blk < b1 ? B.table[(size_t)s * B.stride + (blk >> A.c.nbl)] : -2;
        };
        int pages = pages_from(p);
        // tile of block blk, the k-th of the 32 that `pages` covers; null: nothing there to read
        auto tile_at = [&](int blk, int k) -> const uint8_t * {
            const int page = __shfl_sync(0xffffffffu, pages, k);
            if ((unsigned)page >= (unsigned)A.c.pages) {
                if (blk < b1 && lane == 0) atomicOr(&g_kv_fault, kFaultBatch);
                return nullptr;
            }
            const size_t t = (((size_t)page * A.c.hk + h) << A.c.nbl) + (blk & ((1 << A.c.nbl) - 1));
            return A.c.tiles + t * A.c.tile_bytes;
        };
        // ---- the ring
        auto issue = [&](const uint8_t *tile, int stage) {
            if (tile != nullptr) {
                const uint32_t to = ring_at + stage * Smem::BLOCK + 16 * lane;
                // K: tokens 4 (g / 2) + g % 2 and 2 further (columns g of S's two tiles of the block)
                const uint8_t *kp = tile + kHeader + (4 * (g >> 1) + (g & 1)) * D + 16 * c;
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    copy16(to + (2 * i) * 512, kp + 64 * i);
                    copy16(to + (2 * i + 1) * 512, kp + 2 * D + 64 * i);
                }
                // V: tokens 4 c .. 4 c + 3, VB dims at VB g
                const uint8_t *vp = tile + kHeader + (kBlock + 4 * c) * D + VB * g;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    if constexpr (VB == 16) copy16(to + 16 * D + t * 512, vp + t * D);
                    else copy8(ring_at + stage * Smem::BLOCK + 16 * D + t * 256 + 8 * lane, vp + t * D);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        auto scales_of = [&](const uint8_t *tile) {
            return tile != nullptr ? __ldg(reinterpret_cast<const float2 *>(tile)) : make_float2(0.0f, 0.0f);
        };
        const uint8_t *t0 = tile_at(p, 0), *t1 = tile_at(p + 1, 1);
        const uint8_t *u0 = tile_at(p + 2 * kDigWarps, 2), *u1 = tile_at(p + 2 * kDigWarps + 1, 3);
        issue(t0, 0);
        issue(t1, 1);
        issue(u0, 2);
        issue(u1, 3);
        float2 sc0 = scales_of(t0), sc1 = scales_of(t1);

        // ---- q in digits
        __syncthreads();  // the last task's join has read shared memory
        if (w < NC) {
            uint32_t mx = 0;
#pragma unroll
            for (int t = 0; t < N; ++t) mx = max(mx, __float_as_uint(qx[t]) & 0x7fffffffu);
            mx = __reduce_max_sync(0xffffffffu, mx);
            // the largest |q| to [2^29, 2^30); a column that is not finite gets a scale that is NaN
            const int e = mx == 0 || mx >= 0x7f800000u ? 0 : min(120, 156 - (int)(mx >> 23));
            const float f = __int_as_float((127 + e) << 23);
#pragma unroll
            for (int t = 0; t < N; ++t) sm.q[w][lane * N + t] = digits_of(__float2int_rn(qx[t] * f));
            if (lane == 0) sm.qscale[w] = mx >= 0x7f800000u ? __int_as_float(0x7fffffff) : A.scale * __int_as_float((127 - e) << 23);
        }
        for (int i = lane; i < NC * (D + 4); i += 32) sm.o[w][0][i] = 0.0f;
        __syncthreads();

        // A operand of S: element e of the row's column for k-step 2 i + z and half y: dims 64 i + 16 c + 8 z + 4 y ..
        uint32_t qa[KS][4];
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int z = 0; z < 2; ++z)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const uint4 d = *reinterpret_cast<const uint4 *>(&sm.q[g >> 1][64 * i + 16 * c + 8 * z + 4 * y]);
                    qa[2 * i + z][2 * y] = __byte_perm(__byte_perm(d.x, d.y, sel0), __byte_perm(d.z, d.w, sel0), 0x5410);
                    qa[2 * i + z][2 * y + 1] = __byte_perm(__byte_perm(d.x, d.y, sel1), __byte_perm(d.z, d.w, sel1), 0x5410);
                }
        const int col = col0 + (g >> 1);  // this lane's column
        const float qs = sm.qscale[g >> 1] * ((g & 1) ? 65536.0f : 1.0f);
        const int phi = col < cols ? first + col / A.group : -1;  // tokens that it sees
        const int plo = A.window > 0 ? phi - A.window + 1 : 0;
        // blocks [full_lo, full_hi) are seen whole by every column (padded columns are never read)
        const int last = first + min(sq.n - 1, (col0 + NC - 1) / A.group);
        const int full_hi = (first + col0 / A.group + 1) >> 4;
        const int full_lo = A.window > 0 ? (max(0, last - A.window + 1) + 15) >> 4 : 0;

        int acc[D / 8][4];
#pragma unroll
        for (int j = 0; j < D / 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0;
        float m = -INFINITY, l = 0.0f, vref = 0x1p-100f;
        int held = 0;  // pairs in acc
        int half = 0;  // pair of the ring in work
        int k = 2;     // pair of `pages` after the next one
        for (; p < b1; p += 2 * kDigWarps, half ^= 1, ++k) {
            const int pn = p + 4 * kDigWarps;
            if (k == 16) {
                pages = pages_from(pn);
                k = 0;
            }
            const uint8_t *const n0 = tile_at(pn, 2 * k), *const n1 = tile_at(pn + 1, 2 * k + 1);
            const float2 sn0 = scales_of(u0), sn1 = scales_of(u1);
            asm volatile("cp.async.wait_group 2;" ::: "memory");
            const uint8_t *const st = ring + 2 * half * Smem::BLOCK;

            // scores: tile j of 8 tokens, this lane's columns 2 c and 2 c + 1: tokens 16 (j / 2) + 4 c + 2 (j % 2) + z of the pair
            float x[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t d[4];
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    const uint4 k = *reinterpret_cast<const uint4 *>(st + (j >> 1) * Smem::BLOCK + (2 * i + (j & 1)) * 512 + 16 * lane);
                    if (i == 0) mma_s8(d, qa[0], k.x, k.y, magic);
                    else mma_s8(d, qa[2 * i], k.x, k.y, d);
                    mma_s8(d, qa[2 * i + 1], k.z, k.w, d);
                }
                const float sc = (j < 2 ? sc0.x : sc1.x) * qs;
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    const float v = fmaf(__uint_as_float(d[z + 2]) - kDigMagicF, 256.0f, __uint_as_float(d[z]) - kDigMagicF) * sc;
                    x[2 * j + z] = v + __shfl_xor_sync(0xffffffffu, v, 4);
                }
            }
            if (!(p >= full_lo && p + 1 < full_hi && t0 != nullptr && t1 != nullptr)) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int tok = (p + (i >> 2)) * kBlock + 4 * c + 2 * (i >> 1 & 1) + (i & 1);
                    if ((i < 4 ? t0 : t1) == nullptr || tok > phi || tok < plo) x[i] = -INFINITY;
                }
            }
            float t = x[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) t = fmaxf(t, x[i]);
            const float vs = fmaxf(t0 != nullptr ? sc0.y : 0.0f, t1 != nullptr ? sc1.y : 0.0f);
            if (__any_sync(0xffffffffu, t > m + kDigStep) || vs > vref || held == 2048) {
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
                float f = 1.0f;
                const float unit = vref * (1.0f / kDigOne);
                if (t > m + kDigStep) {  // also the first score: m = -inf
                    f = m == -INFINITY ? 0.0f : ex2(m - (t + kDigAhead));
                    m = t + kDigAhead;
                    l *= f;
                }
                if (held > 0) flush_sums<D>(acc, sm.o[w], unit, f);
                held = 0;
                if (vs > vref) vref = __int_as_float((min(253, (__float_as_int(vs) >> 23) + 1)) << 23);  // a power of two above vs
            }
            ++held;
            const float ref = m == -INFINITY ? 0.0f : m;
            const float vi = kDigOne / vref;
            const float f0 = sc0.y * vi, f1 = sc1.y * vi;
            uint32_t y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float e = ex2(x[i] - ref);
                l += e;
                y[i] = digits_of(__float2int_rn(e * (i < 4 ? f0 : f1)));
            }
            if (!(sc0.y >= 0.0f && sc1.y >= 0.0f)) {  // a scale that is NaN makes its rows NaN
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (!((i < 4 ? sc0.y : sc1.y) >= 0.0f) && x[i] != -INFINITY) l = __int_as_float(0x7fffffff);
            }
            uint32_t pa[4];
            pa[0] = __byte_perm(__byte_perm(y[0], y[1], sel0), __byte_perm(y[2], y[3], sel0), 0x5410);
            pa[1] = __byte_perm(__byte_perm(y[0], y[1], sel1), __byte_perm(y[2], y[3], sel1), 0x5410);
            pa[2] = __byte_perm(__byte_perm(y[4], y[5], sel0), __byte_perm(y[6], y[7], sel0), 0x5410);
            pa[3] = __byte_perm(__byte_perm(y[4], y[5], sel1), __byte_perm(y[6], y[7], sel1), 0x5410);

            // values: four tokens' words to four dims' words
            uint32_t vw[2][4][VB / 4];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint8_t *const at = st + b * Smem::BLOCK + 16 * D;
                    if constexpr (VB == 16) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(at + k * 512 + 16 * lane);
                        vw[b][k][0] = v.x; vw[b][k][1] = v.y; vw[b][k][2] = v.z; vw[b][k][3] = v.w;
                    } else {
                        const uint2 v = *reinterpret_cast<const uint2 *>(at + k * 256 + 8 * lane);
                        vw[b][k][0] = v.x; vw[b][k][1] = v.y;
                    }
                }
#pragma unroll
            for (int u = 0; u < VB / 4; ++u) {
                uint32_t r[2][4];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const uint32_t a0 = __byte_perm(vw[b][0][u], vw[b][1][u], 0x5140), a1 = __byte_perm(vw[b][2][u], vw[b][3][u], 0x5140);
                    const uint32_t a2 = __byte_perm(vw[b][0][u], vw[b][1][u], 0x7362), a3 = __byte_perm(vw[b][2][u], vw[b][3][u], 0x7362);
                    r[b][0] = __byte_perm(a0, a1, 0x5410);
                    r[b][1] = __byte_perm(a0, a1, 0x7632);
                    r[b][2] = __byte_perm(a2, a3, 0x5410);
                    r[b][3] = __byte_perm(a2, a3, 0x7632);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t(&d)[4] = reinterpret_cast<uint32_t(&)[4]>(acc[4 * u + k]);
                    mma_s8(d, pa, r[0][k], r[1][k], d);
                }
            }
            // the pair's slots are free: the pair after the next one
            issue(n0, 2 * half);
            issue(n1, 2 * half + 1);
            t0 = u0; t1 = u1; u0 = n0; u1 = n1;
            sc0 = sn0; sc1 = sn1;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");

        // ---- the warps meet
        flush_sums<D>(acc, sm.o[w], vref * (1.0f / kDigOne), 1.0f);
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (c == 0 && (g & 1) == 0) {
            sm.m[w][g >> 1] = m;
            sm.l[w][g >> 1] = l;
        }
        __syncthreads();
        const bool whole = W.whole();
        float *part = W.part(D);
        for (int e = threadIdx.x; e < NC * (D / 4); e += kDigThreads) {
            const int j = e / (D / 4), d = 4 * (e % (D / 4));
            const int cj = col0 + j;
            if (cj >= cols) continue;
            float M = -INFINITY, L = 0.0f;
#pragma unroll
            for (int i = 0; i < kDigWarps; ++i) M = fmaxf(M, sm.m[i][j]);
            float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < kDigWarps; ++i) {
                // a warp that saw nothing has l = 0 and o = 0, or NaN, which goes through
                const float f = sm.m[i][j] == -INFINITY ? 1.0f : ex2(sm.m[i][j] - M);
                L = fmaf(f, sm.l[i][j], L);
                const float4 y = *reinterpret_cast<const float4 *>(&sm.o[i][j][d]);
                x[0] = fmaf(f, y.x, x[0]);
                x[1] = fmaf(f, y.y, x[1]);
                x[2] = fmaf(f, y.z, x[2]);
                x[3] = fmaf(f, y.w, x[3]);
            }
            if (whole) {
                const float r = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
                for (int z = 0; z < 4; ++z) x[z] *= r;
                const int i = cj / A.group;
                store_row<4>(A.out, (size_t)(sq.a + i) * A.os + ((size_t)h * A.group + (cj - i * A.group)) * D + d, A.type, x);
            } else {
                *reinterpret_cast<float4 *>(part + j * D + d) = make_float4(x[0], x[1], x[2], x[3]);
                if (d == 0) {
                    part[NC * D + j] = M;
                    part[NC * D + NC + j] = L;
                }
            }
        }
        if (W.open()) {
            open = true;
            if (threadIdx.x == 0) W.note();
        }
    }
    if (threadIdx.x == 0 && !open) A.rec[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
}

}  // namespace q4kv
