// Attention over the 8-bit cache (q4rdna_kv_attention).
#pragma once

#include "q4rdna_kv.cuh"

namespace q4kv {

struct AttnArgs {
    Cache c;
    Batch b;
    const void *q;
    void *out;
    int64_t qs, os;
    int type, heads, group;
    float scale;   // of q . k, times log2(e)
    int window;    // 0: none
};

// One warp per row (token, query head), one cached token at a time: softmax with
// a running maximum and sum.
template <int D>
__global__ void __launch_bounds__(128) kv_attention_row_kernel(const __grid_constant__ AttnArgs A) {
    constexpr int EPL = D / 32;
    const Batch &B = A.b;
    const int lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (item >= (long long)B.T * A.heads) return;
    const int row = (int)(item / A.heads), hq = (int)(item % A.heads);
    int s = row;
    if (B.q_start != nullptr) {
        int lo = 0, hi = B.S - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (B.q_start[mid] <= row) lo = mid; else hi = mid - 1;
        }
        s = lo;
    }
    const Seq sq = load_seq(B, s);
    if (row < sq.a || row >= sq.a + sq.n) return;
    const int p = sq.L - sq.n + (row - sq.a);
    const int lo = A.window > 0 ? max(0, p - A.window + 1) : 0;
    float x[EPL], o[EPL], m = -INFINITY, l = 0.0f;
    load_row<EPL>(A.q, (size_t)row * A.qs + (size_t)hq * D + lane * EPL, A.type, x);
#pragma unroll
    for (int t = 0; t < EPL; ++t) {
        x[t] *= A.scale;
        o[t] = 0.0f;
    }
    for (int j = lo; j <= p; ++j) {
        const uint8_t *tile = tile_of(A.c, B, s, hq / A.group, j >> 4);
        if (tile == nullptr) continue;
        const float2 sc = *reinterpret_cast<const float2 *>(tile);
        float k[EPL], v[EPL], d = 0.0f;
        load_codes<EPL>(tile + kHeader + (j & 15) * D + lane * EPL, A.c.format, k);
        load_codes<EPL>(tile + kHeader + (kBlock + (j & 15)) * D + lane * EPL, A.c.format, v);
#pragma unroll
        for (int t = 0; t < EPL; ++t) d = fmaf(x[t], k[t], d);
#pragma unroll
        for (int i = 16; i > 0; i >>= 1) d += __shfl_xor_sync(0xffffffffu, d, i);
        d *= sc.x;
        const float m1 = fmaxf(m, d), f = exp2f(m - m1), e = exp2f(d - m1);
        l = fmaf(l, f, e);
#pragma unroll
        for (int t = 0; t < EPL; ++t) o[t] = fmaf(o[t], f, e * sc.y * v[t]);
        m = m1;
    }
#pragma unroll
    for (int t = 0; t < EPL; ++t) o[t] = l == 0.0f ? 0.0f : o[t] / l;
    store_row<EPL>(A.out, (size_t)row * A.os + (size_t)hq * D + lane * EPL, A.type, o);
}

}  // namespace q4kv
