// Key/value cache operators for sm_100a, host side: argument checks and
// launches of q4rdna_kv_append.cuh and q4rdna_kv_attention.cuh.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>

#include "q4rdna_kv.h"
#include "q4rdna_kv_append.cuh"
#include "q4rdna_kv_attention.cuh"

namespace q4 {
extern std::atomic<uint64_t> g_launches;  // q4rdna_gemv.cu: kernels launched by the library
}

namespace q4kv {

bool aligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int type_bytes(int type) { return type == Q4RDNA_F32 ? 4 : 2; }

q4rdna_status check_cache(const q4rdna_kv_cache *c, Cache &out) {
    if (c == nullptr || c->tiles == nullptr) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (c->pages <= 0 || c->kv_heads <= 0) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (c->format != Q4RDNA_KV_INT8 && c->format != Q4RDNA_KV_E4M3) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (q4rdna_kv_cache_bytes(c) == 0) return Q4RDNA_ERR_SHAPE;
    if (!aligned(c->tiles)) return Q4RDNA_ERR_ALIGNMENT;
    out.tiles = c->tiles;
    out.pages = c->pages;
    out.hk = c->kv_heads;
    out.nbl = 0;
    while ((kBlock << out.nbl) < c->page_tokens) ++out.nbl;
    out.format = c->format;
    out.tile_bytes = (int)q4rdna_kv_tile_bytes(c->head_dim);
    return Q4RDNA_OK;
}

q4rdna_status check_batch(const q4rdna_kv_cache *c, const q4rdna_kv_batch *b, int tokens, Batch &out) {
    if (b == nullptr || b->page_table == nullptr || b->lengths == nullptr) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (b->sequences < 0 || b->table_stride <= 0 || b->max_length < 0 || tokens < 0) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (b->q_start == nullptr && tokens != b->sequences) return Q4RDNA_ERR_SHAPE;
    const long long room = std::min<long long>((long long)b->table_stride * c->page_tokens, INT_MAX - 256);
    if (b->max_length > room) return Q4RDNA_ERR_SHAPE;
    // the append's units and the attention's 32-bit row arithmetic
    if (b->sequences > (1 << 28) || tokens > (1 << 28)) return Q4RDNA_ERR_TOO_LARGE;
    out.table = b->page_table;
    out.lengths = b->lengths;
    out.q_start = b->q_start;
    out.S = b->sequences;
    out.stride = b->table_stride;
    out.max_len = b->max_length > 0 ? b->max_length : (int)room;
    out.T = tokens;
    return Q4RDNA_OK;
}

// A row operand: [rows][heads][D] with `stride` elements from row to row
q4rdna_status check_rows(const void *p, int64_t stride, int type, int heads, int D) {
    if (p == nullptr) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (stride < (int64_t)heads * D) return Q4RDNA_ERR_SHAPE;
    if (!aligned(p) || stride * type_bytes(type) % 16 != 0) return Q4RDNA_ERR_ALIGNMENT;
    return Q4RDNA_OK;
}

bool known_type(int t) { return t == Q4RDNA_F32 || t == Q4RDNA_F16 || t == Q4RDNA_BF16; }

q4rdna_status launched() {
    if (cudaGetLastError() != cudaSuccess) return Q4RDNA_ERR_CUDA;
    q4::g_launches.fetch_add(1, std::memory_order_relaxed);
    return Q4RDNA_OK;
}

q4rdna_status check_attention(const q4rdna_kv_cache *cache, const q4rdna_kv_batch *batch,
                              const q4rdna_kv_attention_args *args, AttnArgs &A) {
    q4rdna_status st = check_cache(cache, A.c);
    if (st != Q4RDNA_OK) return st;
    if (args == nullptr || !known_type(args->type) || args->window < 0) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (!std::isfinite(args->scale) || args->scale < 0.0f) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if ((st = check_batch(cache, batch, args->tokens, A.b)) != Q4RDNA_OK) return st;
    if (args->heads <= 0) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (args->heads % cache->kv_heads != 0) return Q4RDNA_ERR_SHAPE;
    const int D = cache->head_dim;
    if (args->tokens > 0) {
        if ((st = check_rows(args->q, args->q_stride, args->type, args->heads, D)) != Q4RDNA_OK) return st;
        if ((st = check_rows(args->out, args->out_stride, args->type, args->heads, D)) != Q4RDNA_OK) return st;
    }
    A.q = args->q;
    A.out = args->out;
    A.qs = args->q_stride;
    A.os = args->out_stride;
    A.type = args->type;
    A.heads = args->heads;
    A.group = args->heads / cache->kv_heads;
    const float scale = args->scale > 0.0f ? args->scale : 1.0f / std::sqrt((float)D);
    A.scale = scale * 1.44269504088896340736f;
    A.window = args->window;
    return Q4RDNA_OK;
}

}  // namespace q4kv

uint32_t q4kv_take_fault() {
    unsigned v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, q4kv::g_kv_fault, sizeof(v)) != cudaSuccess) return 0xffffffffu;
    if (v != 0) cudaMemcpyToSymbol(q4kv::g_kv_fault, &zero, sizeof(zero));
    return v;
}

extern "C" {

size_t q4rdna_kv_tile_bytes(int head_dim) {
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return 0;
    return q4kv::kHeader + 2 * (size_t)q4kv::kBlock * head_dim;
}

size_t q4rdna_kv_cache_bytes(const q4rdna_kv_cache *c) {
    if (c == nullptr || c->pages <= 0 || c->kv_heads <= 0) return 0;
    const int p = c->page_tokens;
    if (p < 16 || p > 256 || (p & (p - 1)) != 0) return 0;
    return (size_t)c->pages * c->kv_heads * (p / q4kv::kBlock) * q4rdna_kv_tile_bytes(c->head_dim);
}

q4rdna_status q4rdna_kv_append(const q4rdna_kv_cache *cache, const q4rdna_kv_batch *batch,
                               const q4rdna_kv_append_args *args, q4rdna_stream_t stream) {
    using namespace q4kv;
    AppendArgs A{};
    q4rdna_status st = check_cache(cache, A.c);
    if (st != Q4RDNA_OK) return st;
    if (args == nullptr || !known_type(args->type) || args->heads < 0) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if ((args->q_norm != nullptr || args->k_norm != nullptr) && (!std::isfinite(args->norm_eps) || args->norm_eps < 0.0f))
        return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (args->rope != Q4RDNA_ROPE_NEOX && args->rope != Q4RDNA_ROPE_NORM) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if ((st = check_batch(cache, batch, args->tokens, A.b)) != Q4RDNA_OK) return st;
    const int D = cache->head_dim;
    const int rot = args->inv_freq == nullptr ? 0 : args->rotary_dim == 0 ? D : args->rotary_dim;
    if (rot < 0 || rot > D || rot % 16 != 0) return Q4RDNA_ERR_SHAPE;
    if (args->heads % cache->kv_heads != 0) return Q4RDNA_ERR_SHAPE;
    if (!aligned(args->q_norm) || !aligned(args->k_norm)) return Q4RDNA_ERR_ALIGNMENT;
    if (args->tokens > 0) {
        if ((st = check_rows(args->k, args->k_stride, args->type, cache->kv_heads, D)) != Q4RDNA_OK) return st;
        if ((st = check_rows(args->v, args->v_stride, args->type, cache->kv_heads, D)) != Q4RDNA_OK) return st;
        if (args->heads > 0) {
            if ((st = check_rows(args->q, args->q_stride, args->type, args->heads, D)) != Q4RDNA_OK) return st;
            if ((st = check_rows(args->q_out, args->q_out_stride, args->type, args->heads, D)) != Q4RDNA_OK) return st;
        }
    }
    if (args->tokens == 0 || batch->sequences == 0) return Q4RDNA_OK;
    A.k = args->k; A.v = args->v; A.q = args->q; A.q_out = args->q_out;
    A.ks = args->k_stride; A.vs = args->v_stride; A.qs = args->q_stride; A.qos = args->q_out_stride;
    A.inv_freq = args->inv_freq; A.q_norm = args->q_norm; A.k_norm = args->k_norm; A.positions = args->positions;
    A.type = args->type; A.heads = args->heads; A.rot = rot; A.neox = args->rope == Q4RDNA_ROPE_NEOX;
    A.eps = args->norm_eps;
    const int units = batch->q_start == nullptr ? batch->sequences : args->tokens / kBlock + 2 * batch->sequences;
    const dim3 grid((unsigned)units, (unsigned)std::min(cache->kv_heads, 65535));
    const cudaStream_t cs = (cudaStream_t)stream;
    if (D == 64) kv_append_kernel<64><<<grid, kAppendThreads, 0, cs>>>(A);
    else if (D == 128) kv_append_kernel<128><<<grid, kAppendThreads, 0, cs>>>(A);
    else kv_append_kernel<256><<<grid, kAppendThreads, 0, cs>>>(A);
    return launched();
}

q4rdna_status q4rdna_kv_dequant(const q4rdna_kv_cache *cache, const int32_t *page_list, int count, int type, void *k,
                                void *v, q4rdna_stream_t stream) {
    using namespace q4kv;
    Cache c{};
    const q4rdna_status st = check_cache(cache, c);
    if (st != Q4RDNA_OK) return st;
    if (count < 0 || !known_type(type)) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (count == 0) return Q4RDNA_OK;
    if (page_list == nullptr || k == nullptr || v == nullptr) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (!aligned(k) || !aligned(v)) return Q4RDNA_ERR_ALIGNMENT;
    const long long n = ((long long)count * c.hk) << c.nbl;
    if (n > 0x7fffffffLL) return Q4RDNA_ERR_TOO_LARGE;
    const cudaStream_t cs = (cudaStream_t)stream;
    if (cache->head_dim == 64) kv_dequant_kernel<64><<<(unsigned)n, 128, 0, cs>>>(c, page_list, type, k, v);
    else if (cache->head_dim == 128) kv_dequant_kernel<128><<<(unsigned)n, 128, 0, cs>>>(c, page_list, type, k, v);
    else kv_dequant_kernel<256><<<(unsigned)n, 128, 0, cs>>>(c, page_list, type, k, v);
    return launched();
}

size_t q4rdna_kv_attention_workspace_bytes(const q4rdna_kv_cache *cache, const q4rdna_kv_batch *batch,
                                           const q4rdna_kv_attention_args *args) {
    q4kv::AttnArgs A{};
    if (q4kv::check_attention(cache, batch, args, A) != Q4RDNA_OK) return 0;
    return 0;
}

q4rdna_status q4rdna_kv_attention(const q4rdna_kv_cache *cache, const q4rdna_kv_batch *batch,
                                  const q4rdna_kv_attention_args *args, void *workspace, size_t workspace_bytes,
                                  q4rdna_stream_t stream) {
    using namespace q4kv;
    AttnArgs A{};
    const q4rdna_status st = check_attention(cache, batch, args, A);
    if (st != Q4RDNA_OK) return st;
    (void)workspace;
    (void)workspace_bytes;
    if (args->tokens == 0 || batch->sequences == 0) return Q4RDNA_OK;
    const long long n = ((long long)args->tokens * args->heads + 3) / 4;
    if (n > 0x7fffffffLL) return Q4RDNA_ERR_TOO_LARGE;
    const cudaStream_t cs = (cudaStream_t)stream;
    if (cache->head_dim == 64) kv_attention_row_kernel<64><<<(unsigned)n, 128, 0, cs>>>(A);
    else if (cache->head_dim == 128) kv_attention_row_kernel<128><<<(unsigned)n, 128, 0, cs>>>(A);
    else kv_attention_row_kernel<256><<<(unsigned)n, 128, 0, cs>>>(A);
    return launched();
}

}  // extern "C"
