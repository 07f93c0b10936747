// Append of keys and values to the 8-bit cache: per-head RMSNorm, rotation,
// block scales and codes in one pass (q4rdna_kv_append).
//
// One CTA (4 warps) owns one 16-token block of one sequence, and of its heads
// the slice blockIdx.y, + gridDim.y, ...  It first makes the block's cosines and
// sines in shared memory, shared by all its heads: position * inv_freq and the
// reduction by multiples of 2 pi in f64 (an f32 product is off by 0.06 rad at
// position 10^6), then sincosf of a reduced f32 angle.  A warp holds a row of
// head_dim elements, head_dim / 32 consecutive ones per lane; the partner of an
// element in the rotation is a lane shuffle away.  Keys and values of the whole
// block stay in registers between the maximum and the codes, so each is read
// once.
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
    int type, heads, rot, neox;
    float eps;
};

constexpr int kAppendWarps = 4;
constexpr int kAppendThreads = 32 * kAppendWarps;
constexpr int kAppendRows = kBlock / kAppendWarps;  // rows of a block per warp

// First unit of sequence s: sequences take at most (n + 15) / 16 + 1 blocks, and
// floor((a + n) / 16) - floor(a / 16) + 2 is never less.
__device__ __forceinline__ int append_unit(const Batch &b, int s) {
    return b.q_start == nullptr ? s : (b.q_start[s] >> 4) + 2 * s;
}

template <int EPL>
__device__ __forceinline__ void norm_row(float (&x)[EPL], const float (&w)[EPL], float eps) {
    float ss = 0.0f;
#pragma unroll
    for (int t = 0; t < EPL; ++t) ss = fmaf(x[t], x[t], ss);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float f = rsqrtf(ss * (1.0f / (32 * EPL)) + eps);
#pragma unroll
    for (int t = 0; t < EPL; ++t) x[t] = x[t] * f * w[t];
}

template <int EPL>
__device__ __forceinline__ void rotate_row(float (&x)[EPL], const float2 *cs, int rot, bool neox, int lane) {
    const int half = rot >> 1;
    if (neox) {
        const int e0 = lane * EPL;  // half is a multiple of EPL: a lane lies in one half
        const bool low = e0 < half, in = e0 < rot;
        const int src = in ? (low ? lane + half / EPL : lane - half / EPL) : lane;
        const float2 *p = cs + (in ? (low ? e0 : e0 - half) : 0);
#pragma unroll
        for (int t = 0; t < EPL; ++t) {
            const float y = __shfl_sync(0xffffffffu, x[t], src);
            if (in) {
                const float2 r = p[t];
                x[t] = low ? x[t] * r.x - y * r.y : x[t] * r.x + y * r.y;
            }
        }
    } else if (lane * EPL < rot) {
#pragma unroll
        for (int t = 0; t < EPL; t += 2) {
            const float2 r = cs[(lane * EPL + t) >> 1];
            const float a = x[t], y = x[t + 1];
            x[t] = a * r.x - y * r.y;
            x[t + 1] = y * r.x + a * r.y;
        }
    }
}

template <int D>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const __grid_constant__ AppendArgs A) {
    constexpr int EPL = D / 32;
    __shared__ float2 cs[kBlock][D / 2];
    __shared__ uint32_t wmax[2][kAppendWarps][2];
    const Batch &B = A.b;
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
    const int first = q.L - q.n;  // may be negative: padded rows, not stored
    const int blk = (first >> 4) + j;  // rounds down
    const int lo = max(first, blk * kBlock), cnt = min(q.L, (blk + 1) * kBlock) - lo;
    if (j < 0 || cnt <= 0) return;
    const int r0 = lo - blk * kBlock;        // the tile's first new row
    const int row0 = q.a + (lo - first);     // its row of q, k, v
    const int half = A.rot >> 1;
    for (int i = threadIdx.x; i < cnt * half; i += kAppendThreads) {
        const int t = i / half, p = i - t * half;
        const int pos = A.positions != nullptr ? A.positions[row0 + t] : lo + t;
        const double a = (double)pos * (double)A.inv_freq[p];
        const double r = fma(-rint(a * 0.15915494309189535), 6.283185307179586, a);
        float sn, c;
        sincosf((float)r, &sn, &c);
        cs[t][p] = make_float2(c, sn);
    }
    __syncthreads();

    const size_t col = (size_t)lane * EPL;
    float nw[EPL];
    if (A.k_norm != nullptr) load_row<EPL>(A.k_norm, col, Q4RDNA_F32, nw);
    if (blk >= 0) {
        const float top = code_top(A.c.format);
        int par = 0;
        for (int h = blockIdx.y; h < A.c.hk; h += gridDim.y, par ^= 1) {
            uint8_t *tile = tile_of(A.c, B, s, h, blk);
            if (tile == nullptr) break;  // the same page for every head
            float k[kAppendRows][EPL], v[kAppendRows][EPL];
            uint32_t mk = 0, mv = 0;  // the largest |x| as bits: NaN above infinity above the numbers
#pragma unroll
            for (int u = 0; u < kAppendRows; ++u) {
                const int i = w + u * kAppendWarps;
                if (i < cnt) {
                    load_row<EPL>(A.k, (size_t)(row0 + i) * A.ks + (size_t)h * D + col, A.type, k[u]);
                    load_row<EPL>(A.v, (size_t)(row0 + i) * A.vs + (size_t)h * D + col, A.type, v[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < kAppendRows; ++u) {
                const int i = w + u * kAppendWarps;
                if (i < cnt) {
                    if (A.k_norm != nullptr) norm_row<EPL>(k[u], nw, A.eps);
                    if (half > 0) rotate_row<EPL>(k[u], cs[i], A.rot, A.neox, lane);
#pragma unroll
                    for (int t = 0; t < EPL; ++t) {
                        mk = max(mk, __float_as_uint(k[u][t]) & 0x7fffffffu);
                        mv = max(mv, __float_as_uint(v[u][t]) & 0x7fffffffu);
                    }
                }
            }
            mk = __reduce_max_sync(0xffffffffu, mk);
            mv = __reduce_max_sync(0xffffffffu, mv);
            if (lane == 0) {
                wmax[par][w][0] = mk;
                wmax[par][w][1] = mv;
            }
            float2 old = make_float2(0.0f, 0.0f);  // a tile begun by this call: what it held does not count
            if (r0 > 0) old = *reinterpret_cast<const float2 *>(tile);
            __syncthreads();
            const float s_old[2] = {old.x, old.y};
            float sc[2], low[2], inv[2];
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                uint32_t m = 0;
#pragma unroll
                for (int i = 0; i < kAppendWarps; ++i) m = max(m, wmax[par][i][z]);
                const float now = __uint_as_float(m) / top;
                float x = fmaxf(s_old[z], now);
                if (x < kTinyScale) x = 0.0f;
                if (m >= 0x7f800000u || isnan(s_old[z])) x = __int_as_float(0x7fffffff);
                sc[z] = x;
                inv[z] = x > 0.0f ? 1.0f / x : 0.0f;
                // what the rounding of max / top left out: 16-bit inputs give many exact halves of a step
                low[z] = x > s_old[z] && x > 0.0f ? fmaf(-now, top, __uint_as_float(m)) / top : 0.0f;
            }
            if (threadIdx.x == 0) *reinterpret_cast<float2 *>(tile) = make_float2(sc[0], sc[1]);
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                uint8_t *codes = tile + kHeader + z * kBlock * D + col;
                if (sc[z] > s_old[z])  // the scale grew: the older rows follow
                    for (int r = w; r < r0; r += kAppendWarps) {
                        float x[EPL];
                        load_codes<EPL>(codes + r * D, A.c.format, x);
                        #pragma unroll
                        for (int t = 0; t < EPL; ++t) x[t] *= s_old[z];
                        store_codes<EPL>(codes + r * D, A.c.format, x, sc[z], low[z], inv[z]);
                    }
#pragma unroll
                for (int u = 0; u < kAppendRows; ++u) {
                    const int i = w + u * kAppendWarps;
                    if (i < cnt) store_codes<EPL>(codes + (r0 + i) * D, A.c.format, z == 0 ? k[u] : v[u], sc[z], low[z], inv[z]);
                }
            }
        }
    }
    if (A.q_norm != nullptr) load_row<EPL>(A.q_norm, col, Q4RDNA_F32, nw);
    const int nq = A.heads > (int)blockIdx.y ? (A.heads - (int)blockIdx.y + (int)gridDim.y - 1) / (int)gridDim.y : 0;
    for (int i = w; i < cnt * nq; i += kAppendWarps) {
        const int t = i / nq, h = (int)blockIdx.y + (i - t * nq) * (int)gridDim.y;
        float x[EPL];
        load_row<EPL>(A.q, (size_t)(row0 + t) * A.qs + (size_t)h * D + col, A.type, x);
        if (A.q_norm != nullptr) norm_row<EPL>(x, nw, A.eps);
        if (half > 0) rotate_row<EPL>(x, cs[t], A.rot, A.neox, lane);
        store_row<EPL>(A.q_out, (size_t)(row0 + t) * A.qos + (size_t)h * D + col, A.type, x);
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
