// What the attention's kernels share: arguments, the cut of all tasks' work into
// equal shares, the decoding of two codes to f16, and the join of partial results.
//
// A column is one query row (token, head); the columns of a kv head are all the
// query heads of its group for all the sequence's new tokens.  A task is (sequence,
// kv head, group of nc columns); its work is the pieces of 2^shift tokens that any of
// its columns sees.  All tasks' work in a row is cut into equal shares, one per CTA
// (as many CTAs as the GPU holds at once), so a batch of uneven lengths and a single
// long sequence fill the GPU alike.  A task that lies in several shares leaves one
// partial result (maximum, sum, nc x D sums) per share, and kv_join_kernel, launched
// behind as a programmatic dependent, adds them in share order: no atomics, no order
// that changes a result.
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
    float scale;    // of q . k, times log2(e)
    int window;     // 0: none
    int min_share;  // pieces per CTA at least
    int few, many;  // only sequences of few <= columns < many
    float *part;    // partial results: two slots per CTA
    int4 *rec;      // per CTA: the task that begins in its share and goes on
};

// Floats of one partial result
__host__ __device__ constexpr int part_floats(int D, int NC) { return NC * (D + 2); }

// The columns col0 .. col0 + nc - 1 of a sequence: pieces [lo, hi) that any of them sees
struct Span {
    int lo, hi;
};
__device__ __forceinline__ Span span_of(const Seq &q, int col0, int nc, int group, int window, int shift) {
    const int i0 = col0 / group, i1 = min(q.n - 1, (col0 + nc - 1) / group);
    const int p0 = q.L - q.n + i0, p1 = q.L - q.n + i1;
    Span s;
    s.hi = p1 < 0 ? 0 : (p1 >> shift) + 1;
    s.lo = window > 0 ? min(max(0, p0 - window + 1) >> shift, s.hi) : 0;
    return s;
}
// Work of a task: one piece at least, so that every task lies in a share and its rows are written
__device__ __forceinline__ int work_of(const Span &s) { return max(1, s.hi - s.lo); }

// Work of one kv head of a sequence; 0 for a sequence that is not this kernel's.  The
// lanes of a warp call it together, each with a sequence of its own or all with the
// same one; a sequence of many tasks is summed by the whole warp.
__device__ __forceinline__ long long head_work(const AttnArgs &A, const Seq &q, int nc, int shift) {
    const int lane = threadIdx.x & 31;
    const int cols = q.n * A.group;
    const bool ours = cols >= A.few && cols < A.many && cols > 0;
    long long mine = ours && cols <= nc ? work_of(span_of(q, 0, nc, A.group, A.window, shift)) : 0;
    unsigned todo = __ballot_sync(0xffffffffu, ours && cols > nc);
    while (todo != 0) {
        const int who = __ffs(todo) - 1;
        Seq x;
        x.a = 0;
        x.n = __shfl_sync(0xffffffffu, q.n, who);
        x.L = __shfl_sync(0xffffffffu, q.L, who);
        // (lanes with the same sequence are served at once)
        const bool same = x.n == q.n && x.L == q.L && ours && cols > nc;
        long long w = 0;
        for (int c = lane * nc; c < x.n * A.group; c += 32 * nc) w += work_of(span_of(x, c, nc, A.group, A.window, shift));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
        if (same) mine = w;
        todo &= ~__ballot_sync(0xffffffffu, same);
    }
    return mine;
}

// a / b; 64-bit divisions take a few hundred cycles
__device__ __forceinline__ long long quotient(long long a, long long b) {
    if (((a | b) >> 31) == 0) return (long long)((uint32_t)a / (uint32_t)b);
    return a / b;
}

// A CTA's share
struct Share {
    long long left;   // its length; 0: nothing
    long long share;  // the length of every CTA's but the last
    long long rest;   // offset of its begin in sequence `seq`
    long long head;   // that sequence's work per kv head
    int seq;
    Seq q;
};
template <int WARPS>
struct ShareSmem {
    long long sum[WARPS];
    Share found;
};

// The CTA's share; all of its threads take part
template <int WARPS>
__device__ __forceinline__ Share find_share(const AttnArgs &A, int nc, int shift, ShareSmem<WARPS> &sm) {
    constexpr int THREADS = 32 * WARPS;
    const Batch &B = A.b;
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (B.S <= 32) {  // every warp by itself: no barrier
        Seq q{0, 0, 0};
        if (lane < B.S) q = load_seq(B, lane);
        const long long head = head_work(A, q, nc, shift), mine = head * A.c.hk;
        long long x = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        const long long total = __shfl_sync(0xffffffffu, x, 31);
        Share out{};
        out.share = max((long long)A.min_share, quotient(total + gridDim.x - 1, gridDim.x));
        const long long begin = out.share * blockIdx.x;
        out.left = max(0LL, min(out.share, total - begin));
        const unsigned behind = __ballot_sync(0xffffffffu, x > begin);
        if (behind == 0) return out;
        out.seq = __ffs(behind) - 1;
        out.rest = begin - __shfl_sync(0xffffffffu, x - mine, out.seq);
        out.head = __shfl_sync(0xffffffffu, head, out.seq);
        out.q.a = __shfl_sync(0xffffffffu, q.a, out.seq);
        out.q.n = __shfl_sync(0xffffffffu, q.n, out.seq);
        out.q.L = __shfl_sync(0xffffffffu, q.L, out.seq);
        return out;
    }
    Seq q{0, 0, 0};
    auto work = [&](int s) -> long long {
        q = Seq{0, 0, 0};
        if (s < B.S) q = load_seq(B, s);
        return head_work(A, q, nc, shift) * A.c.hk;
    };
    const long long first = work(threadIdx.x);  // of a chunk of THREADS sequences; most batches are one
    long long total = 0;
    for (int base = 0; base < B.S; base += THREADS) {
        long long x = base == 0 ? first : work(base + threadIdx.x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        if (lane == 0) sm.sum[w] = x;
        __syncthreads();
        x = lane < WARPS ? sm.sum[lane] : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        total += x;
        __syncthreads();
    }
    const long long share = max((long long)A.min_share, quotient(total + gridDim.x - 1, gridDim.x));
    const long long begin = share * blockIdx.x;
    if (begin >= total) return Share{};
    long long before = 0;
    for (int base = 0; base < B.S && before <= begin; base += THREADS) {
        const long long mine = base == 0 && B.S <= THREADS ? first : work(base + threadIdx.x);  // (and q)
        long long x = mine;  // inclusive prefix
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) sm.sum[w] = x;
        __syncthreads();
        long long ahead = lane < w ? sm.sum[lane] : 0, all = lane < WARPS ? sm.sum[lane] : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
            all += __shfl_xor_sync(0xffffffffu, all, o);
        }
        x += ahead;
        const long long at = begin - before - (x - mine);
        if (at >= 0 && at < mine) {
            sm.found = {min(share, total - begin), share, at, quotient(mine, A.c.hk), base + (int)threadIdx.x, q};
        }
        before += all;
        __syncthreads();
    }
    return sm.found;
}

// The tasks of a share, one after the other (the same in all threads; the lanes of a
// warp call next() together)
struct Walk {
    const AttnArgs &A;
    int nc, shift;
    long long left, rest, share;
    int s;
    Seq q{};
    int cols = 0, h = 0, col0 = 0;
    // the piece of the current task that is this share's
    Span span{};
    int begin = 0, end = 0, all = 0, cnt = 0;
    bool begins = false, ends = false;

    __device__ __forceinline__ Walk(const AttnArgs &a, int nc_, int shift_, const Share &f)
        : A(a), nc(nc_), shift(shift_), left(f.left), rest(f.rest), share(f.share), s(f.seq), q(f.q) {
        cols = q.n * A.group;
        h = (int)quotient(rest, f.head);
        rest -= h * f.head;
        col0 = -nc;
    }

    __device__ __forceinline__ bool next() {
        if (left <= 0) return false;
        col0 += nc;
        while (true) {
            if (col0 >= cols) {  // the next head, or the next sequence with work
                col0 = 0;
                if (++h >= A.c.hk) {
                    long long hw;
                    do {
                        if (++s >= A.b.S) return false;
                        q = load_seq(A.b, s);
                        hw = head_work(A, q, nc, shift);
                    } while (hw == 0);
                    cols = q.n * A.group;
                    h = (int)quotient(rest, hw);
                    rest -= h * hw;
                }
            }
            // the task with `rest` in it: the warp looks at 32 tasks at a time
            const int lane = threadIdx.x & 31;
            const int c = col0 + lane * nc;
            const int mine = c < cols ? work_of(span_of(q, c, nc, A.group, A.window, shift)) : 0;
            uint32_t upto = mine;
            constexpr long long kMost = 32ll * (kMaxTokens / kBlock);
            static_assert((decltype(upto))kMost == kMost, "the work of 32 tasks");
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
            const unsigned behind = __ballot_sync(0xffffffffu, upto > rest);
            if (behind != 0) {
                const int hit = __ffs(behind) - 1;
                all = __shfl_sync(0xffffffffu, mine, hit);
                rest -= __shfl_sync(0xffffffffu, upto, hit) - all;
                col0 += hit * nc;
                span = span_of(q, col0, nc, A.group, A.window, shift);
                break;
            }
            rest -= __shfl_sync(0xffffffffu, upto, 31);
            col0 += 32 * nc;
        }
        begin = span.lo + (int)rest;
        cnt = (int)min((long long)(all - (int)rest), left);
        end = min(begin + cnt, span.hi);
        begins = rest == 0;
        ends = (int)rest + cnt == all;
        rest = 0;
        left -= cnt;
        return true;
    }
    __device__ __forceinline__ bool whole() const { return begins && ends; }
    // this piece's partial result
    __device__ __forceinline__ float *part(int D) const {
        return A.part + (size_t)(2 * blockIdx.x + (begins ? 1 : 0)) * part_floats(D, nc);
    }
    // the share ends inside a task that began in it: what the join needs
    __device__ __forceinline__ void note() const {
        A.rec[2 * blockIdx.x] = make_int4(1, q.a, cols, col0);
        A.rec[2 * blockIdx.x + 1] = make_int4(h, (int)blockIdx.x + (int)quotient(all - cnt + share - 1, share), 0, 0);
    }
    __device__ __forceinline__ bool open() const { return begins && !ends; }
};

// ------------------------------------------------------------ codes to f16

__device__ __forceinline__ uint32_t sub_1152(uint32_t x) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0x64806480u));
    return r;
}

// The two e4m3 numbers in the low (high) half of a word as f16, exact.  2 cycles a warp
// and scheduler; the same by shifts and masks takes 8.
template <bool HIGH>
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t w) {
    uint32_t r;
    if constexpr (HIGH) asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %1;\n cvt.rn.f16x2.e4m3x2 %0, h;\n}" : "=r"(r) : "r"(w));
    else asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %1;\n cvt.rn.f16x2.e4m3x2 %0, l;\n}" : "=r"(r) : "r"(w));
    return r;
}

// Two codes to two f16 numbers, exact.  int8: `w` holds code ^ 0x80; byte b under the
// exponent byte 0x64 is 1024 + b, less 1152 the code.
// (a, b): codes number LO and LO + 1 of one word
template <int FMT, int LO>
__device__ __forceinline__ uint32_t pair_of(uint32_t w) {
    if constexpr (FMT == Q4RDNA_KV_INT8) return sub_1152(__byte_perm(w, 0x64646464u, LO == 0 ? 0x4140 : 0x4342));
    else return e4m3_pair<LO != 0>(w);
}

// A row's q is scaled by 2^e, its largest |q| to [2^13, 2^14): e from -114 (2^127) up to here, where 2^e and 2^-e are
// still normal numbers; below 2^-113 the row lies lower in f16's range (the last bit of a denormal f32 at 2^-23)
constexpr int kMostExponent = 126;

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// l * 2^d, d <= 0, in two steps: a sum of weights over tiny values' scales is large, and 2^d alone may be no f32 number
__device__ __forceinline__ float shrunk(float l, float d) {
    const float h = ex2(0.5f * d);
    return l * h * h;
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Joins the pieces of the task that began in CTA blockIdx.x's share and went on in the
// next ones: bound by the latency of a few dependent loads (about 3.6 us behind the
// attention), so as many as can be are on their way together.  One CTA per share and
// column: a grid of as many CTAs as there can be tasks, each looking for its record
// among all shares', took 1.8 us more for 8 tasks in 296 shares.

constexpr int kJoinWarps = 8;

// Where the pieces of a record lie
struct Pieces {
    const float *part;
    int nc, n;  // columns of a task; pieces
    size_t floats;
    // piece 0: this CTA's second slot; then the first slots of the CTAs up to the task's last
    __device__ __forceinline__ const float *operator()(int i) const {
        return part + (size_t)(i == 0 ? 2 * blockIdx.x + 1 : 2 * (blockIdx.x + i)) * floats;
    }
};
template <int D>
__device__ __forceinline__ Pieces pieces_of(const AttnArgs &A, int nc, int last) {
    return {A.part, nc, min(last, (int)gridDim.x - 1) - (int)blockIdx.x + 1, (size_t)part_floats(D, nc)};
}
template <int EPL>
__device__ __forceinline__ void store_column(const AttnArgs &A, const int4 &r0, int h, int col, float L, float (&x)[EPL]) {
    const float r = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
    for (int t = 0; t < EPL; ++t) x[t] *= r;
    const int i = col / A.group, lane = threadIdx.x & 31;
    store_row<EPL>(A.out,
                   (size_t)(r0.y + i) * A.os + ((size_t)h * A.group + (col - i * A.group)) * (32 * EPL) + lane * EPL, A.type, x);
}

// Few columns: one CTA per column, blockIdx.y, whose warps take every eighth piece each
// (a long sequence's few columns lie in tens of pieces)
template <int D>
__global__ void __launch_bounds__(32 * kJoinWarps) kv_join_kernel(const __grid_constant__ AttnArgs A, int nc) {
    constexpr int EPL = D / 32, AHEAD = 4;
    __shared__ float sum[kJoinWarps][D + 1];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 r0 = A.rec[2 * blockIdx.x], r1 = A.rec[2 * blockIdx.x + 1];
    if (r0.x == 0) return;
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int j = blockIdx.y, col = r0.w + j;
    if (col >= r0.z) return;
    const Pieces piece = pieces_of<D>(A, nc, r1.y);
    const int n = piece.n;
    // lane i holds the maximum and sum of piece i (of 32 at a time)
    float M = -INFINITY;
    for (int i = lane; i < n; i += 32) M = fmaxf(M, piece(i)[nc * D + j]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    float x[EPL], L = 0.0f;
#pragma unroll
    for (int t = 0; t < EPL; ++t) x[t] = 0.0f;
    for (int base = 0; base < n; base += 32) {
        float m = -INFINITY, l = 0.0f;
        if (base + lane < n) {
            m = piece(base + lane)[nc * D + j];
            l = piece(base + lane)[nc * D + nc + j];
        }
        const float f = m == -INFINITY ? 1.0f : ex2(m - M);
        L += m == -INFINITY ? l : shrunk(l, m - M);
        const int cnt = min(32, n - base);
        for (int i = w; i < cnt; i += AHEAD * kJoinWarps) {
            float y[AHEAD][EPL];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
                if (i + u * kJoinWarps < cnt)
                    load_row<EPL>(piece(base + i + u * kJoinWarps), (size_t)j * D + lane * EPL, Q4RDNA_F32, y[u]);
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const float fu = __shfl_sync(0xffffffffu, f, (i + u * kJoinWarps) & 31);
                if (i + u * kJoinWarps < cnt)
#pragma unroll
                    for (int t = 0; t < EPL; ++t) x[t] = fmaf(fu, y[u][t], x[t]);
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
#pragma unroll
    for (int t = 0; t < EPL; ++t) sum[w][lane * EPL + t] = x[t];
    __syncthreads();
    if (w > 0) return;
#pragma unroll
    for (int t = 0; t < EPL; ++t) x[t] = 0.0f;
#pragma unroll
    for (int i = 0; i < kJoinWarps; ++i)
#pragma unroll
        for (int t = 0; t < EPL; ++t) x[t] += sum[i][lane * EPL + t];
    store_column<EPL>(A, r0, r1.x, col, L, x);
}

// Many columns: a warp takes four of them together, all pieces; blockIdx.y the 32 columns
constexpr int kJoinCols = 4;
template <int D>
__global__ void __launch_bounds__(32 * kJoinWarps) kv_join_wide_kernel(const __grid_constant__ AttnArgs A, int nc) {
    constexpr int EPL = D / 32, AHEAD = 4;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 r0 = A.rec[2 * blockIdx.x], r1 = A.rec[2 * blockIdx.x + 1];
    if (r0.x == 0) return;
    const int lane = threadIdx.x & 31;
    const int j0 = (blockIdx.y * kJoinWarps + (threadIdx.x >> 5)) * kJoinCols;
    if (r0.w + j0 >= r0.z) return;
    const Pieces piece = pieces_of<D>(A, nc, r1.y);
    const int n = piece.n, cols = min(kJoinCols, r0.z - r0.w - j0);
    // lane 8 k + i holds the maximum and sum of piece i (of 8 at a time) of column k
    const int k = lane >> 3, i = lane & 7;
    const bool there = k < cols;
    float M = -INFINITY;
    for (int b = i; b < n && there; b += 8) M = fmaxf(M, piece(b)[nc * D + j0 + k]);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    float x[kJoinCols][EPL], L = 0.0f;
#pragma unroll
    for (int c = 0; c < kJoinCols; ++c)
#pragma unroll
        for (int t = 0; t < EPL; ++t) x[c][t] = 0.0f;
    for (int base = 0; base < n; base += 8) {
        float m = -INFINITY, l = 0.0f;
        if (base + i < n && there) {
            m = piece(base + i)[nc * D + j0 + k];
            l = piece(base + i)[nc * D + nc + j0 + k];
        }
        const float f = m == -INFINITY ? 1.0f : ex2(m - M);
        L += m == -INFINITY ? l : shrunk(l, m - M);
#pragma unroll
        for (int u0 = 0; u0 < 8; u0 += AHEAD) {
            if (base + u0 >= n) break;
            float y[AHEAD][kJoinCols][EPL];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                for (int c = 0; c < kJoinCols; ++c)
                    if (base + u0 + u < n && c < cols)
                        load_row<EPL>(piece(base + u0 + u), (size_t)(j0 + c) * D + lane * EPL, Q4RDNA_F32, y[u][c]);
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                for (int c = 0; c < kJoinCols; ++c) {
                    const float fu = __shfl_sync(0xffffffffu, f, 8 * c + u0 + u);
                    if (base + u0 + u < n && c < cols)
#pragma unroll
                        for (int t = 0; t < EPL; ++t) x[c][t] = fmaf(fu, y[u][c][t], x[c][t]);
                }
        }
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
#pragma unroll
    for (int c = 0; c < kJoinCols; ++c) {
        const float Lc = __shfl_sync(0xffffffffu, L, 8 * c);
        if (c < cols) store_column<EPL>(A, r0, r1.x, r0.w + j0 + c, Lc, x[c]);
    }
}

}  // namespace q4kv
