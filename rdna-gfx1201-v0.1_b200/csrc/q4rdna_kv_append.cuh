// Append of keys and values to the 8-bit cache: per-head RMSNorm, rotation,
// block scales and codes in one pass (q4rdna_kv_append).
//
// HBM-bound for prompts (every element is read once, q written once, the codes
// written), bound by the chain of its loads for single tokens.  One CTA owns one
// 16-token block of one sequence and the heads blockIdx.y, + gridDim.y, ...
//   * D / 16 lanes hold a row (token, head), 8 elements of either half each (Place), so
//     a rotation in halves of the whole row finds both elements of a pair in one lane,
//     as the interleaved one does, and the norm's sum takes 3 shuffles for 4 rows
//     (D = 128).  One row per warp with 4 elements a lane took 190 instructions a row
//     and 160 us for 8192 tokens of 32 + 8 + 8 heads in bf16 (now 46 us, 4.0 TB/s).
//   * The CTA's D threads are 16 such groups: `tp` tokens x 16 / tp heads at a time,
//     tp the block's new tokens rounded up to a power of two, so a single token's
//     heads run side by side.
//   * Cosines and sines are made once per CTA, in shared memory and the lanes' order:
//     position * inv_freq and the reduction to a turn in f64 (an f32
//     product is off by 0.06 rad at position 10^6), then sincospif of the f32 rest
//     and what its rounding lost (2^-24 of the angle) to first order.
//   * A lane's rows come through a ring in shared memory, 6 (f32: 4) ahead, from before
//     the cosines on.
//   * Keys and values stay in registers between the maximum and the codes.  A code is
//     round(x / s) with 1 / s as a sum of two f32 numbers, so that a quotient half-way
//     between two codes (frequent with 16-bit inputs) is met exactly.
#pragma once

#include "q4rdna_kv.cuh"

namespace q4kv {

struct AppendArgs {
    Cache c;
    Batch b;
    const void *k, *v, *q;
    void *q_out;
    int64_t ks, vs, qs, qos;
    const float *inv_freq, *q_norm, *k_norm;
    const int32_t *positions;
    int heads, rot;
    float eps;
};

// How the rotation's pairs lie: in halves of the whole row, side by side, or in halves of a part of it
enum { kTurnHalves = 0, kTurnPairs = 1, kTurnPart = 2 };

// First unit of sequence s: sequences take at most (n + 15) / 16 + 1 blocks, and
// floor((a + n) / 16) - floor(a / 16) + 2 is never less.
__device__ __forceinline__ int append_unit(const Batch &b, int s) {
    return b.q_start == nullptr ? s : (b.q_start[s] >> 4) + 2 * s;
}

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Which elements of a row a lane holds: 8 of either half, as 16-byte pieces that
// lie side by side over the lanes (16-bit types: 8 elements at 8 l; f32: 4 at 4 l
// of either quarter; 32 bytes per lane would fetch every 32-byte sector twice)
template <int D, int TYPE>
struct Place {
    static constexpr bool WIDE = TYPE == Q4RDNA_F32;
    // element i (0..7) of the lane's half z
    static __device__ __forceinline__ int at(int l, int z, int i) {
        return z * (D / 2) + (WIDE ? (i >> 2) * (D / 4) + 4 * l + (i & 3) : 8 * l + i);
    }
    // of element e: the lane, and 8 z + i
    static __device__ __forceinline__ int lane(int e) { return WIDE ? e % (D / 4) / 4 : e % (D / 2) / 8; }
    static __device__ __forceinline__ int slot(int e) {
        return e / (D / 2) * 8 + (WIDE ? e % (D / 2) / (D / 4) * 4 + e % 4 : e % 8);
    }
};

// A lane's 16 elements of a row on their way: 16-byte pieces, copied asynchronously to
// slots of the lane's own, which only it reads (its own wait is all it needs)
template <int D, int TYPE>
struct Ring {
    static constexpr int N = TYPE == Q4RDNA_F32 ? 2 : 1;      // pieces of 8 elements
    static constexpr int DEPTH = TYPE == Q4RDNA_F32 ? 4 : 6;  // rows of a lane in flight
    static constexpr int ROW = 2 * N * D * 16;                // a row of every lane
    static constexpr int BYTES = DEPTH * ROW;
    uint8_t *base;  // the lane's slots
    int put = 0, get = 0;

    __device__ __forceinline__ explicit Ring(uint8_t *smem) : base(smem + 16 * threadIdx.x) {}
    // p: the row's bytes from the lane's first on; null: no copy
    __device__ __forceinline__ void issue(const uint8_t *p) {
        if (p != nullptr) {
            const uint32_t to = smem_u32(base) + put;
#pragma unroll
            for (int i = 0; i < 2 * N; ++i) copy16(to + i * D * 16, p + i * D);  // D / 2 (f32: D / 4) elements on
        }
        put = put == (DEPTH - 1) * ROW ? 0 : put + ROW;
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    // elements 2 i and 2 i + 1 in x[i]; zeros where nothing was copied
    __device__ __forceinline__ void take(bool on, F2 (&x)[8]) {
        asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
        const uint8_t *const from = base + get;
        get = get == (DEPTH - 1) * ROW ? 0 : get + ROW;
#pragma unroll
        for (int i = 0; i < 2 * N; ++i) {
            const uint4 r = on ? *reinterpret_cast<const uint4 *>(from + i * D * 16) : make_uint4(0, 0, 0, 0);
            const uint32_t w[4] = {r.x, r.y, r.z, r.w};
            if constexpr (TYPE == Q4RDNA_F32) {
                x[2 * i] = pack2(__uint_as_float(w[0]), __uint_as_float(w[1]));
                x[2 * i + 1] = pack2(__uint_as_float(w[2]), __uint_as_float(w[3]));
            } else {
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    if constexpr (TYPE == Q4RDNA_BF16) {
                        x[4 * i + t] = pack2(__uint_as_float(w[t] << 16), __uint_as_float(w[t] & 0xffff0000u));
                    } else {
                        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[t]));
                        x[4 * i + t] = pack2(f.x, f.y);
                    }
                }
            }
        }
    }
};

// A sum or maximum over the LPR lanes of a group
template <int LPR>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
template <int LPR>
__device__ __forceinline__ float group_max(float x) {
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) x = max_nan(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}

// 16 numbers to codes, x / s = x * hi + x * lo
template <int FMT>
__device__ __forceinline__ void codes_of(const F2 (&x)[8], float hi, float lo, uint2 (&c)[2]) {
    const F2 h = pack2(hi, hi), l = pack2(lo, lo), magic = pack2(12582912.0f, 12582912.0f);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const F2 y0 = fma2(x[2 * i], h, mul2(x[2 * i], l)), y1 = fma2(x[2 * i + 1], h, mul2(x[2 * i + 1], l));
        if constexpr (FMT == Q4RDNA_KV_INT8) {
            // 1.5 * 2^23 + y: the code in the lowest byte, to nearest even; |y| is at most 127 and a rounding
            const float2 a = both(add2(y0, magic)), b = both(add2(y1, magic));
            w[i] = __byte_perm(__byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040),
                               __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040), 0x5410);
        } else {
            w[i] = __byte_perm(__nv_cvt_float2_to_fp8x2(both(y0), __NV_SATFINITE, __NV_E4M3),
                               __nv_cvt_float2_to_fp8x2(both(y1), __NV_SATFINITE, __NV_E4M3), 0x5410);
        }
    }
    c[0] = make_uint2(w[0], w[1]);
    c[1] = make_uint2(w[2], w[3]);
}

template <int D, int TYPE, int FMT, int TURN>
__global__ void __launch_bounds__(D, 640 / D) kv_append_kernel(const __grid_constant__ AppendArgs A) {
    constexpr int LPR = D / 16;  // lanes of a row
    using P = Place<D, TYPE>;
    // cosines and sines in the lanes' order: [token][i][lane] two cosines, two sines of the
    // lane's pairs 2 i and 2 i + 1 (16 bytes more per token, so that tokens differ in banks)
    __shared__ __align__(16) float cs[kBlock][4 * LPR + 1][4];
    __shared__ __align__(16) float nw[2][4][LPR][4];  // norm weights of k and q in the lanes' order
    __shared__ float part[2][2][16];   // maxima of the groups: keys, values
    extern __shared__ __align__(16) uint8_t slots[];
    Ring<D, TYPE> ring(slots);
    // rows of a rotation whose pairs do not meet in a lane
    float(*const line)[D + 1] = reinterpret_cast<float(*)[D + 1]>(slots + Ring<D, TYPE>::BYTES);
    const Batch &B = A.b;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int s = blockIdx.x;
    if (B.q_start != nullptr) {  // the last sequence whose first unit is not behind this one
        int lo = 0, hi = B.S - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (append_unit(B, mid) <= (int)blockIdx.x) lo = mid; else hi = mid - 1;
        }
        s = lo;
    }
    const int j = (int)blockIdx.x - append_unit(B, s);
    const Seq q = load_seq(B, s);
    const int first = q.L - q.n;       // may be negative: padded rows, not stored
    const int blk = (first >> 4) + j;  // rounds down
    const int lo = max(first, blk * kBlock), cnt = min(q.L, (blk + 1) * kBlock) - lo;
    if (j < 0 || cnt <= 0) return;
    const int r0 = lo - blk * kBlock;     // the tile's first new row
    const int row0 = q.a + (lo - first);  // its row of q, k, v
    const int half = A.rot >> 1;

    const int gid = threadIdx.x / LPR, l = threadIdx.x % LPR;
    const int tpl = cnt > 8 ? 4 : cnt > 4 ? 3 : cnt > 2 ? 2 : cnt > 1 ? 1 : 0;  // tp = 2^tpl token places
    const int tok = gid & ((1 << tpl) - 1), hp = 16 >> tpl;                     // heads side by side
    const bool on = tok < cnt;
    const int step = hp * (int)gridDim.y;  // heads from pass to pass
    const int h0 = (int)blockIdx.y + (int)gridDim.y * (gid >> tpl);
    const size_t row = (size_t)(row0 + (on ? tok : 0));

    // the lane's rows in order: k and v of each pass over the kv heads, then q
    const int kvp = blk >= 0 && A.c.hk > (int)blockIdx.y ? (A.c.hk - (int)blockIdx.y + step - 1) / step : 0;
    const int qp = A.heads > (int)blockIdx.y ? (A.heads - (int)blockIdx.y + step - 1) / step : 0;
    constexpr int E = TYPE == Q4RDNA_F32 ? 4 : 2;
    const size_t col = (size_t)h0 * D * E + 16 * l, over = (size_t)step * D * E;
    const uint8_t *kn = reinterpret_cast<const uint8_t *>(A.k) + row * A.ks * E + col;
    const uint8_t *vn = reinterpret_cast<const uint8_t *>(A.v) + row * A.vs * E + col;
    const uint8_t *qn = reinterpret_cast<const uint8_t *>(A.q) + row * A.qs * E + col;
    // this lane's rows that are there: passes over kv and q heads
    int kleft = kvp > 0 && on && h0 < A.c.hk ? (A.c.hk - h0 + step - 1) / step : 0;
    int qleft = on && h0 < A.heads ? (A.heads - h0 + step - 1) / step : 0;
    int next = -2 * kvp;  // below 0: k and v in turn
    auto issue = [&]() {
        const uint8_t *p = nullptr;
        if (next >= 0) {
            if (qleft > 0) {
                p = qn;
                qn += over;
                --qleft;
            }
        } else if (next & 1) {
            if (kleft > 0) p = vn;
            vn += over;
            --kleft;
        } else {
            if (kleft > 0) p = kn;
            kn += over;
        }
        ++next;
        ring.issue(p);
    };
    // a tile and its scales (0 where this call begins it: what it held does not count)
    uint8_t *tile = nullptr;
    float2 old = make_float2(0.0f, 0.0f);
    auto enter = [&](int h) {
        tile = tile_of(A.c, B, s, h < A.c.hk ? h : 0, blk);
        if (r0 > 0 && tile != nullptr) old = *reinterpret_cast<const float2 *>(tile);
    };
#pragma unroll 1
    for (int i = 0; i < ring.DEPTH; ++i) issue();
    if (kvp > 0) enter(h0);
    for (int i = threadIdx.x; i < cnt * (D / 2) && half > 0; i += D) {
        const int t = i / (D / 2), p = i % (D / 2);
        float sn = 0.0f, c = 1.0f;
        if (p < half) {
            const int pos = A.positions != nullptr ? A.positions[row0 + t] : lo + t;
            const double a = (double)pos * (double)A.inv_freq[p] * 0.3183098861837907;  // in half turns
            const double turn = a - 2.0 * rint(0.5 * a);
            const float f = (float)turn, d = 3.14159265f * (float)(turn - f);  // what f lost, to first order
            float s0, c0;
            sincospif(f, &s0, &c0);
            sn = fmaf(d, c0, s0);
            c = fmaf(-d, s0, c0);
        }
        // pair p is the e-th of lane x
        const int x = P::lane(TURN != kTurnPairs ? p : 2 * p), e = TURN != kTurnPairs ? P::slot(p) : P::slot(2 * p) / 2;
        cs[t][(e >> 1) * LPR + x][e & 1] = c;
        cs[t][(e >> 1) * LPR + x][2 + (e & 1)] = sn;
    }
#pragma unroll
    for (int z = 0; z < 2; ++z) {
        const float *weight = z == 0 ? A.k_norm : A.q_norm;
        if (weight != nullptr) {
            const int e = threadIdx.x;
            nw[z][P::slot(e) / 4][P::lane(e)][P::slot(e) % 4] = weight[e];
        }
    }
    __syncthreads();
    // norm and rotation of a row
    auto prepare = [&](F2(&x)[8], bool norm, int z) {
        if (norm) {
            F2 ss = mul2(x[0], x[0]);
#pragma unroll
            for (int i = 1; i < 8; ++i) ss = fma2(x[i], x[i], ss);
            const float2 two = both(ss);
            const float ms = group_sum<LPR>(two.x + two.y) * (1.0f / D) + A.eps;
            float f1 = rsqrtf(ms);
            if (ms > 0.0f && f1 > 0.0f) f1 = fmaf(0.5f * f1, fmaf(-ms * f1, f1, 1.0f), f1);  // Newton: rsqrtf is off by 2 ulp
            const F2 f = pack2(f1, f1);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const ulonglong2 w = *reinterpret_cast<const ulonglong2 *>(nw[z][i][l]);
                x[2 * i] = mul2(mul2(x[2 * i], f), w.x);
                x[2 * i + 1] = mul2(mul2(x[2 * i + 1], f), w.y);
            }
        }
        if (half == 0) return;
        const float(*const turn)[4] = cs[on ? tok : 0];
        if constexpr (TURN == kTurnPart) {
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 v = both(x[i]);
                const int e = P::at(l, i >> 2, 2 * (i & 3));
                line[gid][e] = v.x;
                line[gid][e + 1] = v.y;
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float v[2] = {both(x[i]).x, both(x[i]).y};
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const int e = P::at(l, i >> 2, 2 * (i & 3)) + y;
                    if (e < A.rot) {
                        const int p = e < half ? e : e - half;
                        const float *const r = turn[P::slot(p) / 2 * LPR + P::lane(p)] + (p & 1);
                        v[y] = e < half ? v[y] * r[0] - line[gid][e + half] * r[2] : v[y] * r[0] + line[gid][e - half] * r[2];
                    }
                }
                x[i] = pack2(v[0], v[1]);
            }
        } else if constexpr (TURN == kTurnHalves) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const ulonglong2 r = *reinterpret_cast<const ulonglong2 *>(turn[i * LPR + l]);  // cosines, sines
                const F2 a = x[i], b = x[i + 4];
                x[i] = fma2(a, r.x, mul2(b, r.y ^ 0x8000000080000000ull));
                x[i + 4] = fma2(b, r.x, mul2(a, r.y));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 r = *reinterpret_cast<const float4 *>(turn[i * LPR + l]);
                const float2 a = both(x[2 * i]), b = both(x[2 * i + 1]);
                x[2 * i] = pack2(a.x * r.x - a.y * r.z, a.y * r.x + a.x * r.z);
                x[2 * i + 1] = pack2(b.x * r.y - b.y * r.w, b.y * r.y + b.x * r.w);
            }
        }
    };

    auto put_codes = [&](uint8_t *to, const uint2 (&c)[2]) {
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            if constexpr (P::WIDE) {
                *reinterpret_cast<uint32_t *>(to + P::at(l, z, 0)) = c[z].x;
                *reinterpret_cast<uint32_t *>(to + P::at(l, z, 4)) = c[z].y;
            } else {
                *reinterpret_cast<uint2 *>(to + P::at(l, z, 0)) = c[z];
            }
        }
    };
    if (kvp > 0) {
        constexpr float top = FMT == Q4RDNA_KV_INT8 ? 127.0f : 448.0f, rtop = 1.0f / top;
        for (int z = 0; z < kvp; ++z) {
            const int par = z & 1, h = h0 + z * step;
            const bool here = h < A.c.hk;  // this group's head
            // (the page, and so whether it lies in the cache, is the same for every head)
            if (z > 0) enter(h);
            F2 k[8], v[8];
            ring.take(here && on, k);
            issue();
            ring.take(here && on, v);
            issue();
            if (tile == nullptr) continue;
            prepare(k, A.k_norm != nullptr, 0);
            float mk = 0.0f, mv = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 a = both(k[i]), b = both(v[i]);
                mk = max_nan(max_nan(mk, fabsf(a.x)), fabsf(a.y));
                mv = max_nan(max_nan(mv, fabsf(b.x)), fabsf(b.y));
            }
            mk = group_max<LPR>(mk);
            mv = group_max<LPR>(mv);
#pragma unroll
            for (int o = LPR; o < 32; o <<= 1)
                if (o < LPR << tpl) {  // this warp's other tokens of the head
                    mk = max_nan(mk, __shfl_xor_sync(0xffffffffu, mk, o));
                    mv = max_nan(mv, __shfl_xor_sync(0xffffffffu, mv, o));
                }
            if (l == 0) {
                part[par][0][gid] = mk;
                part[par][1][gid] = mv;
            }
            __syncthreads();
            // keys, then values: one copy of the code, for a single token runs each line once
            float was = old.x;
#pragma unroll 1
            for (int y = 0; y < 2; ++y) {
                float m = 0.0f;
                for (int i = 0; i < (1 << tpl); i += 32 / LPR) m = max_nan(m, part[par][y][(gid >> tpl << tpl) + i]);
                const float now = m / top;
                float x = fmaxf(was, now);
                if (x < kTinyScale) x = 0.0f;
                if (!(m < INFINITY) || isnan(was)) x = __int_as_float(0x7fffffff);
                // 1 / x in two parts; where this call sets the scale, of m / top before its rounding
                const float hi = x > 0.0f ? 1.0f / x : 0.0f;
                const float lost = now > was ? fmaf(-x, top, m) * rtop : 0.0f;
                const float low = (fmaf(-hi, x, 1.0f) - lost * hi) * hi;
                uint8_t *codes = tile + kHeader + y * kBlock * D;
                uint2 c[2];
                if (here && x > was)  // the scale grew: the older rows follow
#pragma unroll 1
                    for (int r = tok; r < r0; r += 1 << tpl) {
                        F2 u[8];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float t[4];
                            load_codes<4>(codes + r * D + P::at(l, i >> 1, 4 * (i & 1)), FMT, t);
                            u[2 * i] = pack2(t[0] * was, t[1] * was);
                            u[2 * i + 1] = pack2(t[2] * was, t[3] * was);
                        }
                        codes_of<FMT>(u, hi, low, c);
                        put_codes(codes + r * D, c);
                    }
                if (here && on) {
                    codes_of<FMT>(k, hi, low, c);
                    // the scale marks the tile; a NaN code would reach rows that do not see it, as 0 * NaN
                    if (isnan(x)) c[0] = c[1] = make_uint2(0, 0);
                    put_codes(codes + (r0 + tok) * D, c);
                }
                if (here && tok == 0 && l == 0) reinterpret_cast<float *>(tile)[y] = x;
                was = old.y;
#pragma unroll
                for (int i = 0; i < 8; ++i) k[i] = v[i];
            }
        }
    }
    uint8_t *to = reinterpret_cast<uint8_t *>(A.q_out) + row * A.qos * E + col;
    for (int z = 0; z < qp; ++z) {
        const bool here = h0 + z * step < A.heads && on;
        F2 x[8];
        ring.take(here, x);
        issue();
        prepare(x, A.q_norm != nullptr, 1);
        if (here) {
            constexpr int W = P::WIDE ? 4 : 8;  // elements of a 16-byte piece
#pragma unroll
            for (int i = 0; i < 16 / W; ++i) {
                float a[W];
#pragma unroll
                for (int t = 0; t < W / 2; ++t) {
                    const float2 u = both(x[i * (W / 2) + t]);
                    a[2 * t] = u.x;
                    a[2 * t + 1] = u.y;
                }
                store_row<W>(to, i * (D * W / 16), TYPE, a);
            }
        }
        to += over;
    }
}

// One CTA per tile of the listed pages; a page outside the cache reads as zeros.
template <int D>
__global__ void __launch_bounds__(128) kv_dequant_kernel(Cache c, const int32_t *list, int type, void *k, void *v) {
    constexpr int EPL = D / 32;
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per = c.hk << c.nbl;
    const size_t i = blockIdx.x / per;
    const int in = blockIdx.x % per;  // head, then tile of the page
    const int page = list[i];
    const bool ok = (unsigned)page < (unsigned)c.pages;
    if (!ok) atomicOr(&g_kv_fault, kFaultBatch);
    const uint8_t *tile = c.tiles + ((size_t)(ok ? page : 0) * per + in) * c.tile_bytes;
    const float2 sc = *reinterpret_cast<const float2 *>(tile);
#pragma unroll
    for (int r = w; r < kBlock; r += 4) {
        const size_t at = (((size_t)blockIdx.x * kBlock) + r) * D + (size_t)lane * EPL;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            float x[EPL];
            load_codes<EPL>(tile + kHeader + (z * kBlock + r) * D + lane * EPL, c.format, x);
#pragma unroll
            for (int t = 0; t < EPL; ++t) x[t] = ok ? x[t] * (z == 0 ? sc.x : sc.y) : 0.0f;
            store_row<EPL>(z == 0 ? k : v, at, type, x);
        }
    }
}

}  // namespace q4kv
