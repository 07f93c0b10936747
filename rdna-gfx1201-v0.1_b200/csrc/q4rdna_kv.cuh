// Key/value cache in 8 bits: what the append, the attention and the dequant
// kernels share.  Layout (include/q4rdna.h): a tile is 16 tokens of one kv head,
// f32 key scale, f32 value scale, 8 unused bytes, key codes [16][D], value codes
// [16][D]; a page is [kv_heads][page_tokens / 16] tiles.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "q4rdna.h"

namespace q4kv {

constexpr int kBlock = Q4RDNA_KV_BLOCK;
constexpr int kMaxTokens = 1 << 30;        // of a sequence
constexpr int kHeader = 16;                // bytes of a tile before its codes
constexpr float kTinyScale = 0x1p-100f;    // smaller scales are stored as 0
constexpr unsigned kFaultBatch = 8u;       // q4rdna_take_fault bit 3

__device__ unsigned int g_kv_fault;

struct Cache {
    uint8_t *tiles;
    int pages, hk;
    int nbl;      // log2 of the tiles of a page and head
    int format;
    int tile_bytes;
};

struct Batch {
    const int32_t *table, *lengths, *q_start;
    int S, stride;
    int max_len;  // bound of every length: table_stride * page_tokens or less
    int T;        // rows
};

// One sequence of a batch: rows a .. a + n - 1 are its tokens L - n .. L - 1.
struct Seq {
    int a, n, L;
};

__device__ __forceinline__ Seq load_seq(const Batch &b, int s) {
    Seq q;
    q.a = s;
    q.n = 1;
    if (b.q_start != nullptr) {
        q.a = b.q_start[s];
        const int e = b.q_start[s + 1];
        q.n = e - q.a;
        if (q.a < 0 || e < q.a || e > b.T) {
            atomicOr(&g_kv_fault, kFaultBatch);
            q.a = q.n = 0;
        }
    }
    q.L = b.lengths[s];
    if (q.L < 0 || q.L > b.max_len) {
        atomicOr(&g_kv_fault, kFaultBatch);
        q.L = 0;
    }
    return q;
}

// Tile of block `blk` (tokens 16 blk .. 16 blk + 15) of sequence s, head h; null
// for a page outside the cache.  blk must lie below max_len / 16 rounded up.
__device__ __forceinline__ uint8_t *tile_of(const Cache &c, const Batch &b, int s, int h, int blk) {
    const int page = b.table[(size_t)s * b.stride + (blk >> c.nbl)];
    if ((unsigned)page >= (unsigned)c.pages) {
        atomicOr(&g_kv_fault, kFaultBatch);
        return nullptr;
    }
    const size_t tile = ((((size_t)page * c.hk + h) << c.nbl)) + (blk & ((1 << c.nbl) - 1));
    return c.tiles + tile * c.tile_bytes;
}

// ------------------------------------------------------------ numbers

__device__ __forceinline__ float code_top(int format) { return format == Q4RDNA_KV_INT8 ? 127.0f : 448.0f; }

__device__ __forceinline__ float from_code(uint32_t code, int format) {
    if (format == Q4RDNA_KV_INT8) return (float)(int8_t)code;
    return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)code, __NV_E4M3)));
}

// N consecutive elements (2, 4 or 8; aligned to their size) of a row of the given type
template <int N>
__device__ __forceinline__ void load_row(const void *p, size_t at, int type, float (&x)[N]) {
    if (type == Q4RDNA_F32) {
        const float *f = reinterpret_cast<const float *>(p) + at;
        if constexpr (N == 2) {
            const float2 v = *reinterpret_cast<const float2 *>(f);
            x[0] = v.x; x[1] = v.y;
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const float4 v = *reinterpret_cast<const float4 *>(f + i);
                x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
            }
        }
        return;
    }
    uint32_t w[N / 2];
    const uint16_t *h = reinterpret_cast<const uint16_t *>(p) + at;
    if constexpr (N == 2) w[0] = *reinterpret_cast<const uint32_t *>(h);
    else if constexpr (N == 4) {
        const uint2 v = *reinterpret_cast<const uint2 *>(h);
        w[0] = v.x; w[1] = v.y;
    } else {
        const uint4 v = *reinterpret_cast<const uint4 *>(h);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        if (type == Q4RDNA_BF16) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
}

template <int N>
__device__ __forceinline__ void store_row(void *p, size_t at, int type, const float (&x)[N]) {
    if (type == Q4RDNA_F32) {
        float *f = reinterpret_cast<float *>(p) + at;
        if constexpr (N == 2) *reinterpret_cast<float2 *>(f) = make_float2(x[0], x[1]);
        else {
#pragma unroll
            for (int i = 0; i < N; i += 4)
                *reinterpret_cast<float4 *>(f + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
        }
        return;
    }
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        if (type == Q4RDNA_BF16) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&b);
        } else {
            const __half2 b = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&b);
        }
    }
    uint16_t *h = reinterpret_cast<uint16_t *>(p) + at;
    if constexpr (N == 2) *reinterpret_cast<uint32_t *>(h) = w[0];
    else if constexpr (N == 4) *reinterpret_cast<uint2 *>(h) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint4 *>(h) = make_uint4(w[0], w[1], w[2], w[3]);
}

// N codes (2, 4 or 8, aligned to N bytes)
template <int N>
__device__ __forceinline__ void load_codes(const uint8_t *p, int format, float (&x)[N]) {
    uint64_t w;
    if constexpr (N == 2) w = *reinterpret_cast<const uint16_t *>(p);
    else if constexpr (N == 4) w = *reinterpret_cast<const uint32_t *>(p);
    else w = *reinterpret_cast<const uint64_t *>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = from_code((uint32_t)(w >> (8 * i)) & 0xffu, format);
}
// Two f32 numbers in one register pair: one instruction for both
typedef unsigned long long F2;
__device__ __forceinline__ F2 pack2(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 both(F2 x) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// ------------------------------------------------------------ asynchronous copies

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

}  // namespace q4kv
